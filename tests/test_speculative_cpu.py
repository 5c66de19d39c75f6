"""The Python entry points of the serving operators on a machine without a GPU:
they refuse host tensors and mismatched shapes before anything reaches the
library, and the host-only queries of the C ABI answer."""
import pytest
import torch

from nelisp_cuda import _lib as L
from nelisp_cuda import dev
from serving_structs import PACKED


def test_host_tensors_are_refused():
    x, g = torch.zeros(2, 256), torch.ones(64)
    t, p = torch.zeros(4, 32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        dev.qk_norm_rope(x, g, g, t, t, p, x[:, :128], x[:, 128:192])
    with pytest.raises(ValueError, match="CUDA"):
        dev.qk_norm_rope_bwd(x, g, g, t, t, p, x[:, :128], x[:, 128:192], x, g, g)
    cache = dev.kv_cache(2, 16, 1, 64, 8, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        dev.kv_append(x[:, :64], x[:, :64], p, *cache)
    with pytest.raises(ValueError, match="CUDA"):
        dev.kv_read(p, *cache, x[:, :64], x[:, :64])
    with pytest.raises(ValueError, match="CUDA"):
        dev.kv_move(p.view(1, 2), p.view(1, 2), *cache, 64)
    with pytest.raises(ValueError, match="CUDA"):
        dev.tree_attn(x[:, :64], *cache, p.view(2, 1), p, torch.ones(2, 1, dtype=torch.int64),
                      x[:, :64], 64)


def test_types_are_refused():
    x = torch.zeros(2, 256, dtype=torch.float16)
    g, p = torch.ones(64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="f32 or bf16"):
        dev.qk_norm_rope(x, g, g, g, g, p, x, x)
    with pytest.raises(ValueError, match="bits"):
        dev.kv_cache(2, 16, 1, 64, 6, device="cpu")


def test_cache_arrays():
    for bits, row in ((8, 128), (4, 64)):
        kc, kp, vc, vp = dev.kv_cache(3, 16, 2, 128, bits, device="cpu")
        assert kc.shape == vc.shape == (3, 2, 16, row) and kc.dtype == torch.uint8
        assert kp.shape == vp.shape == (3, 2, 16) and kp.dtype == torch.int32


def test_workspace_queries():
    lib = L.load()
    for d in (64, 128, 256):
        assert lib.nl_qk_norm_rope_bwd_workspace_bytes(d) % 16 == 0
        last = 0
        for nodes in (1, 2, 8, 33, 64):
            n = lib.nl_tree_attn_workspace_bytes(nodes, 32, 8, d)
            assert n % 16 == 0 and n >= last
            last = n
    assert lib.nl_tree_attn_workspace_bytes(0, 0, 0, 128) >= 0


def test_packed_structures_match_the_header(tmp_path):
    """The Python packing and the C compiler agree on every structure's size
    and on where its last field is."""
    import os
    import subprocess

    from conftest import ROOT
    names = {"nl_qk_norm_rope_args": ("nl_qk_norm_rope_dev", "eps"),
             "nl_qk_norm_rope_bwd_args": ("nl_qk_norm_rope_bwd_dev", "ws_bytes"),
             "nl_kv_rows_args": ("nl_kv_rows", "v_stride"),
             "nl_kv_move_args": ("nl_kv_move_dev", "count"),
             "nl_tree_attn_args": ("nl_tree_attn_dev", "ws_bytes")}
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "nelisp_cuda.h"\n'
                   "int main(void) {\n" +
                   "".join(f'printf("%zu %zu\\n", offsetof({n}, {last}) + '
                           f"sizeof((({n} *)0)->{last}), sizeof({n}));\n"
                           for n, (_, last) in names.items()) + "}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    for line, (packed, _) in zip(out, names.values()):
        end, size = map(int, line.split())
        assert PACKED[packed].size == end <= size < end + 8, packed
