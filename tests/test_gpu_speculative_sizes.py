"""The operators of speculative serving at the sizes where their kernels take
other forms than at the small ones: bulk calls of the cache and of the norm,
several steps a job with a partial last one; tree attention with every number of
rows a kernel is made for, in every head size, and more rows than an item holds.
Formulas and bounds are those of test_gpu_speculative.py, except:
* the gains' gradients: a lane sums up to 80 terms here, so 128 u of the
  magnitudes' sum;
* the log of the softmax sums: weights are summed in float32 whatever the
  output's type, and bfloat16 queries are exact in the products, so both types
  are held to the float32 bound, eps + 2^-20 |lse|.
"""
import numpy as np
import pytest

import test_gpu_speculative as S
from test_gpu_speculative import dev, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
U = S.U


# ---- the cache in bulk ----------------------------------------------------------

# Tokens enough that a warp takes several vectors a group at a time; the last
# also several such steps a job, for float32.  3 and 5 key heads leave the last
# step partly empty.
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n,kvh,d,bs", [(1300, 3, 64, 16), (1300, 5, 128, 48), (1201, 20, 128, 64),
                                        (1300, 3, 256, 7), (4000, 20, 256, 64)])
def test_kv_append_and_read_in_bulk(dev, torch, n, kvh, d, bs, bits, name):  # noqa: F811
    rng = np.random.default_rng(n + d + bits)
    t = S.dtype_of(torch, name)
    x = rng.standard_normal((2, n, kvh, d), dtype=np.float32)
    for j in range(2):                          # awkward vectors at many rows and heads
        i, h = rng.integers(0, n, (6, n // 20)), rng.integers(0, kvh, (6, n // 20))
        x[j, i[0], h[0]] = 0
        x[j, i[1], h[1]] *= 1e-36
        x[j, i[2], h[2]] = 100 + 1e-3 * x[j, i[2], h[2]]
        x[j, i[3], h[3]] *= 1e30
        x[j, i[4], h[4], rng.integers(0, d, n // 20)] = np.nan
        x[j, i[5], h[5], rng.integers(0, d, n // 20)] = np.inf
    rows = torch.from_numpy(np.concatenate([x[0].reshape(n, -1), x[1].reshape(n, -1)], 1))
    rows = rows.to("cuda", t)
    K, V = rows[:, :kvh * d], rows[:, kvh * d:]
    blocks = -(-n // bs) + 2
    slot = rng.permutation(blocks * bs)[:n].astype(np.int32)
    slot[n // 2], slot[n // 3] = -1, blocks * bs            # outside: skipped
    inside = (slot >= 0) & (slot < blocks * bs)
    at = slot[inside]
    cache = dev.kv_cache(blocks, bs, kvh, d, bits)
    dev.kv_append(K, V, torch.from_numpy(slot).cuda(), *cache)
    ko, vo = torch.full((2, n, kvh * d), 7.0, dtype=t, device="cuda").unbind()
    dev.kv_read(torch.from_numpy(slot).cuda(), *cache, ko, vo)
    torch.cuda.synchronize()
    for j, (X, have) in enumerate(((K, ko), (V, vo))):
        code, word = S.quantise(X.float().cpu().numpy().reshape(n, kvh, d), bits)
        codes = np.zeros(tuple(cache[2 * j].shape), np.uint8)
        words = np.zeros(tuple(cache[2 * j + 1].shape), np.uint32)
        codes[at // bs, :, at % bs] = S.pack(code, bits)[inside]
        words[at // bs, :, at % bs] = word[inside]
        assert np.array_equal(cache[2 * j].cpu().numpy(), codes)
        assert np.array_equal(cache[2 * j + 1].cpu().numpy().view(np.uint32), words)
        want = np.where(inside[:, None, None], S.values(code, word, bits), np.float32(0))
        want = torch.from_numpy(want.reshape(n, -1)).to(t)
        assert torch.equal(have.cpu().nan_to_num(nan=123.0), want.nan_to_num(nan=123.0))


# ---- norm + rotation in bulk ------------------------------------------------------

# Rows enough that a warp takes all heads of one: several steps a row, the last
# of them partly empty.
BULK = [(3000, 7, 3, 128, 128), (2600, 20, 6, 64, 32), (2500, 9, 2, 256, 128), (4000, 7, 3, 80, 48)]


def gains64(gq, gk, h, k):
    return np.concatenate([np.tile(gq.cpu().numpy(), (h, 1)),
                           np.tile(gk.cpu().numpy(), (k, 1))]).astype(float)


@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shape", BULK)
def test_norm_rope_in_bulk(dev, torch, shape, name, pairs):  # noqa: F811
    n, h, k, d, rot = shape
    rng = np.random.default_rng(n + d)
    x, gq, gk, co, si, pos = S.norm_inputs(torch, rng, shape, name)
    q = torch.full((n, h * d), 7.0, device="cuda", dtype=x.dtype)
    kk = torch.full((n, k * d), 7.0, device="cuda", dtype=x.dtype)
    dev.qk_norm_rope(x, gq, gk, co, si, pos, q, kk, eps=1e-5, pairs=pairs)
    tabs = co.cpu().numpy().astype(float), si.cpu().numpy().astype(float), pos.cpu().numpy()
    want, mag = S.norm_rope64(S.heads64(x, n, h + k, d), gains64(gq, gk, h, k), *tabs,
                              float(np.float32(1e-5)), pairs)
    got = np.concatenate([S.heads64(q, n, h, d), S.heads64(kk, n, k, d)], 1)
    assert S.within(torch, got, want, 32 * U * mag + 1e-30, name).all()
    assert not got[1:3].any()

    dq = torch.from_numpy(rng.standard_normal((n, h * d))).to("cuda", x.dtype)
    dk = torch.from_numpy(rng.standard_normal((n, k * d))).to("cuda", x.dtype)
    dx = torch.full_like(x, 7.0)
    dgq, dgk = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    dev.qk_norm_rope_bwd(x, gq, gk, co, si, pos, dq, dk, dx, dgq, dgk, eps=1e-5, pairs=pairs)
    dy = np.concatenate([S.heads64(dq, n, h, d), S.heads64(dk, n, k, d)], 1)
    want, mag, dg, dgm = S.norm_rope_grad64(S.heads64(x, n, h + k, d), gains64(gq, gk, h, k), *tabs,
                                            dy, float(np.float32(1e-5)), pairs)
    assert S.within(torch, S.heads64(dx, n, h + k, d), want, 128 * U * mag + 1e-30, name).all()
    for have, part in ((dgq, slice(0, h)), (dgk, slice(h, h + k))):
        assert (np.abs(have.cpu().numpy() - dg[:, part].sum((0, 1)))
                <= 128 * U * dgm[:, part].sum((0, 1)) + 1e-30).all()
    assert (dx[:, (h + k) * d:].float() == 7).all()


# ---- tree attention: rows a key head --------------------------------------------------

def check_tree(dev, torch, q, kv, table, lens, mask, bits, H, d):  # noqa: F811
    B, M = mask.shape
    cache, (tt, tl, tm) = S.device(torch, kv, table, lens, mask)
    Q = q[:, 16:16 + H * d]
    o = torch.full((B * M, H * d + 8), 7.0, device="cuda", dtype=q.dtype)
    lse = torch.full((B * M, H), 7.0, device="cuda")
    dev.tree_attn(Q, *cache, tt, tl, tm, o[:, :H * d], d, lse=lse)
    want, wl, eps, vmax = S.tree64(Q.float().cpu().numpy().astype(float).reshape(B, M, H, d), kv,
                                   table, lens, mask, bits, d ** -0.5)
    got = o[:, :H * d].float().cpu().numpy().astype(float).reshape(B, M, H, d)
    name = "bf16" if q.dtype == torch.bfloat16 else "f32"
    tol = ((eps + (2 ** -11 if name == "bf16" else 0)) * vmax)[..., None]
    bad = ~S.within(torch, got, want, np.broadcast_to(tol, want.shape), name)
    assert not bad.any(), (np.abs(got - want)[bad].max(), tol.min())
    gl, fin = lse.cpu().numpy().reshape(B, M, H), np.isfinite(wl)
    assert (gl[~fin] == -np.inf).all()
    off = np.abs(gl[fin] - wl[fin]) - (eps[fin] + 2 ** -20 * np.abs(wl[fin]))
    assert (off <= 0).all(), off.max()
    assert (o[:, H * d:].float() == 7).all()


# nodes, heads, key heads: 1, 2 x 4, 16, 32, 64, 100 and 256 rows a key head
ROWS = [(1, 2, 2), (2, 4, 1), (4, 8, 2), (8, 4, 1), (16, 4, 1), (25, 4, 1), (64, 4, 1)]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("M,H,kvh", ROWS)
def test_tree_attn_rows(dev, torch, M, H, kvh, d, bits, name):  # noqa: F811
    rng = np.random.default_rng(M * H + d + bits)
    masks = [S.tree(rng, M), S.chain(M), S.tree(rng, M)]
    masks[2][M // 2:] = [0] * (M - M // 2)
    args = S.attn_inputs(torch, rng, 3, M, H, kvh, d, bits, 16, [170, 0, 31], masks, name)
    check_tree(dev, torch, *args, bits, H, d)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("d,M,H", [(64, 50, 4), (128, 32, 4), (128, 40, 4), (256, 3, 4), (256, 40, 2)])
def test_tree_attn_rows_over_many_parts(dev, torch, d, M, H, bits, name):  # noqa: F811
    """A context that several CTAs share, beside a short one."""
    rng = np.random.default_rng(d + M + bits)
    args = S.attn_inputs(torch, rng, 2, M, H, 1, d, bits, 64, [6001, 50],
                         [S.tree(rng, M), S.chain(M)], name)
    check_tree(dev, torch, *args, bits, H, d)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("M,H", [(3, 2), (20, 1)])
def test_tree_attn_long_bf16_log_sums(dev, torch, bits, M, H):  # noqa: F811
    """70,001 keys: a tile of 32 that is lost would move the log by 5e-4."""
    rng = np.random.default_rng(M)
    args = S.attn_inputs(torch, rng, 1, M, H, 1, 128, bits, 64, [70001], [S.tree(rng, M)], "bf16")
    check_tree(dev, torch, *args, bits, H, 128)
