"""Prints the compiler flags of an extension of the torch that this interpreter
has: its headers, Python's and CUDA's, and torch's libraries."""
import sysconfig

from torch.utils import cpp_extension

flags = ["-I" + d for d in cpp_extension.include_paths("cuda")]
flags.append("-I" + sysconfig.get_paths()["include"])
flags += ["-L" + d for d in cpp_extension.library_paths()]
flags += ["-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
print(" ".join(flags))
