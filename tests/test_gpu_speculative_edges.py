"""The operators of speculative serving where one value, one slot or one row
could spoil another.  Formulas and bounds are those of test_gpu_speculative.py
unless a test derives its own.
"""
import numpy as np
import pytest

import test_gpu_speculative as S
from test_gpu_speculative import dev, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


# ---- a value that a row does not see costs it nothing -----------------------------------
#
# The bounds go by the largest value that a row sees; a node's value may be any
# times larger than the others'.

def put(kv, table, t, vec, bits):
    """VEC as the value of token T of sequence 0."""
    code, word = S.quantise(np.asarray(vec, np.float32), bits)
    bs = kv[3].shape[2]
    kv[2][table[0, t // bs], 0, t % bs] = S.pack(code, bits)
    kv[3][table[0, t // bs], 0, t % bs] = word


# Up to four rows, a tile, several tiles a warp, the tcgen05 form with 32 and 64
# rows at a time; heads of 64 and 256.
FORMS = [("f32", 5, 1, 128), ("f32", 5, 2, 128), ("f32", 20, 4, 128), ("f32", 9, 2, 64),
         ("f32", 9, 3, 256), ("bf16", 5, 1, 128), ("bf16", 5, 3, 128), ("bf16", 20, 1, 128),
         ("bf16", 20, 4, 128), ("bf16", 20, 4, 64), ("bf16", 20, 2, 256)]


@pytest.mark.parametrize("name,M,H,d", FORMS)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("big", [1e4, 1e8, 1e20, 1e30])
@pytest.mark.parametrize("L", [0, 70, 300])
def test_a_large_value_of_another_node(dev, torch, name, M, H, d, bits, big, L):  # noqa: F811
    rng = np.random.default_rng(M + H + d + bits)
    mask = [1 | 1 << i for i in range(M)]               # all see node 0, else themselves
    q, kv, table, lens, mask = S.attn_inputs(torch, rng, 1, M, H, 1, d, bits, 16, [L], [mask], name)
    put(kv, table, L + 3, rng.standard_normal(d) * big, bits)
    S.check_tree(dev, torch, q, kv, table, lens, mask, bits, H, d)


@pytest.mark.parametrize("name,M,H,d", [("f32", 60, 1, 128), ("bf16", 60, 1, 128),
                                        ("bf16", 60, 2, 64), ("bf16", 60, 1, 256)])
@pytest.mark.parametrize("bits", [8, 4])
def test_large_and_small_values_across_node_tiles(dev, torch, name, M, H, d, bits):  # noqa: F811
    """Nodes over several tiles, their values growing and shrinking by turns, in
    chains that do not see each other."""
    rng = np.random.default_rng(5)
    mask = [sum(1 << j for j in range(i % 4, i + 1, 4)) for i in range(M)]      # four chains
    for L in (0, 100, 127):
        q, kv, table, lens, m = S.attn_inputs(torch, rng, 1, M, H, 1, d, bits, 16, [L], [mask], name)
        for i in range(M):
            size = (1.0, 1e12, 1e-9, 1e25)[i % 4] * 8.0 ** (i // 4 % 5)
            put(kv, table, L + i, rng.standard_normal(d) * size, bits)
        S.check_tree(dev, torch, q, kv, table, lens, m, bits, H, d)


@pytest.mark.parametrize("name,M,H,d", FORMS)
@pytest.mark.parametrize("bits", [8, 4])
def test_whatever_an_unused_node_holds(dev, torch, name, M, H, d, bits):  # noqa: F811
    """The slots of unused nodes hold any bits: the largest finite scale, an
    infinity, NaN."""
    rng = np.random.default_rng(M + H)
    L = 90
    mask = [0 if i in (2, 4) else 1 | 1 << i for i in range(M)]
    q, kv, table, lens, mask = S.attn_inputs(torch, rng, 1, M, H, 1, d, bits, 16, [L], [mask], name)
    want = None
    for key, value in ((0, 0), (0x7f7fffff, 0x7f7fffff), (0x7f7f7f7f, 0x7f7f7f7f),
                       (0x7f807f80, 0x7f807f80), (0x7fc07fc0, 0x7fc07fc0), (0xff80ff80, 0x00010001)):
        for t in (L + 2, L + 4):
            at = table[0, t // 16], 0, t % 16
            kv[1][at], kv[3][at] = key, value
            kv[0][at], kv[2][at] = 255, 255
        got, lse = S.check_tree(dev, torch, q, kv, table, lens, mask, bits, H, d)
        assert not got[0, [2, 4]].any() and (lse[0, [2, 4]] == -np.inf).all()
        if want is None:
            want = got
        assert np.array_equal(got, want)                # to the bit what it is without them
