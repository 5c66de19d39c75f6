"""Prints the compiler flags of an extension of the torch that this interpreter
has: its headers, Python's and CUDA's, and torch's libraries.  With --which, prints
which interpreter and torch these are instead, without importing it, and nothing
where there is none or it was built without CUDA."""
import sys

if sys.argv[1:] == ["--which"]:
    import importlib.metadata
    import importlib.util
    import os
    spec = importlib.util.find_spec("torch")
    if spec is not None and spec.origin and os.path.exists(
            os.path.join(os.path.dirname(spec.origin), "lib", "libc10_cuda.so")):
        try:
            version = importlib.metadata.version("torch")
        except importlib.metadata.PackageNotFoundError:
            version = "unknown"
        print(sys.implementation.cache_tag, spec.origin, version)
    sys.exit(0)

import sysconfig

from torch.utils import cpp_extension

flags = ["-I" + d for d in cpp_extension.include_paths("cuda")]
flags.append("-I" + sysconfig.get_paths()["include"])
flags += ["-L" + d for d in cpp_extension.library_paths()]
flags += ["-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
print(" ".join(flags))
