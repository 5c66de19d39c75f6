"""The operators of speculative serving on the GPU against their formulas in 64
bits: per-head Q/K norm with the rotation and its gradient, the quantised paged
KV cache (append, read, move), and draft-tree attention over it.

Tolerances.  u = 2^-24 is the rounding of float32.
* norm + rotation: the sum of at most 256 squares carries at most 16 u of
  rounding (8 lane sums of 16, 5 group steps), its inverse root 8 u + 4 u, the
  products 3 u and the rotation 2 u, so |error| <= 32 u (|a| + |b|) of the pair.
* a bfloat16 output is the rounding of a float32 result within the bound, and
  rounding is monotonic: it lies between the roundings of the interval's ends.
* gradient of x: three such chains enter a sum of three terms that the result
  may cancel, so 128 u of the sum of the terms' magnitudes; of the gains: the
  sums over rows and heads are at most 64 deep, 96 u of the magnitudes' sum.
* codes and parameter words: equal bits; values read back: equal bits.
* attention: products are exact, scores err by at most 2^-21 scale sum |q k|
  (16-step sums, cut), weights by that and 2^-20, and the output is a mean of v:
  |error| <= (2^-20 scale max_t sum |q k_t| + 2^-19) max |v|; where the output
  is bfloat16 the weights' float16 rounding adds 2^-11 max |v|.
"""
import math

import numpy as np
import pytest

from serving_structs import PACKED

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    from nelisp_cuda import dev as d
    return d


@pytest.fixture(scope="module")
def torch():
    import torch as t
    return t


def dtype_of(torch, name):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def within(torch, got, want, tol, name):
    """Where GOT (float64 of the output) is a result within TOL of WANT."""
    if name == "f32":
        return np.abs(got - want) <= tol
    lo, hi = (torch.from_numpy(np.ascontiguousarray(x)).bfloat16().double().numpy()
              for x in (want - tol, want + tol))
    return (lo <= got) & (got <= hi)


# ---- formulas ---------------------------------------------------------------

def pairs_of(rot, pairs):
    h = np.arange(rot // 2)
    return (h, h + rot // 2) if pairs == "half" else (2 * h, 2 * h + 1)


def norm_rope64(x, g, co, si, pos, eps, pairs):
    """x [n, heads, d], g [heads, d] -> y, and the magnitudes its error goes by."""
    d, rot = x.shape[-1], 2 * co.shape[1]
    xn = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = xn * g
    mag = np.abs(y)
    real = (pos >= 0) & (pos < co.shape[0])
    at = np.where(real, pos, 0)
    c, s = co[at][:, None], si[at][:, None]
    a, b = pairs_of(rot, pairs)
    out, m = y.copy(), mag.copy()
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
    m[..., a] = m[..., b] = mag[..., a] + mag[..., b]
    out[~real] = 0
    return out, m


def norm_rope_grad64(x, g, co, si, pos, dy, eps, pairs):
    d, rot = x.shape[-1], 2 * co.shape[1]
    real = ((pos >= 0) & (pos < co.shape[0]))[:, None, None]
    at = np.where(real[:, 0, 0], pos, 0)
    c, s = co[at][:, None], si[at][:, None]
    a, b = pairs_of(rot, pairs)
    u, um = dy.copy(), np.abs(dy)
    u[..., a], u[..., b] = dy[..., a] * c + dy[..., b] * s, dy[..., b] * c - dy[..., a] * s
    um[..., a] = um[..., b] = np.abs(dy[..., a]) + np.abs(dy[..., b])
    u, um = np.where(real, u, 0), np.where(real, um, 0)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xn, w = x * r, u * g
    dx = r * (w - xn * (w * xn).mean(-1, keepdims=True))
    mag = r * (um * np.abs(g) + np.abs(xn) * (um * np.abs(g) * np.abs(xn)).mean(-1, keepdims=True))
    return dx, mag, u * xn, um * np.abs(xn)


def rope_tables(rows, rot):
    ang = np.arange(rows)[:, None] * 10000.0 ** (-2 * np.arange(rot // 2) / rot)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def bf16_round(x, mode):
    """float32 x rounded to bfloat16 down or up, as float32."""
    w = np.asarray(x, np.float32).view(np.int32)
    cut = (w & -65536).astype(np.int32)
    away = (cut + 65536).astype(np.int32)
    inexact = cut != w
    grow = inexact & ((np.asarray(x) < 0) if mode == "down" else (np.asarray(x) > 0))
    return np.where(grow, away, cut).astype(np.int32).view(np.float32)


def quantise(x, bits):
    """Codes (unpacked) and parameter words of float32 head vectors [..., d]."""
    x = x.astype(np.float32)
    tiny = np.float32(2.0 ** -112)
    with np.errstate(all="ignore"):
        if bits == 8:
            most = np.abs(x).max(-1)
            bad = ~np.isfinite(x).all(-1)
            some = most >= np.float32(127) * tiny
            s = np.where(some, most / np.float32(127), np.float32(0))
            inv = np.where(some, np.float32(127) / most, np.float32(0))
            code = 128 + np.rint(x * inv[..., None])
            code = np.where(bad[..., None], 128, code)
            word = np.where(bad, np.float32(np.nan), s).astype(np.float32).view(np.uint32)
            return code.astype(np.uint8), np.where(bad, np.uint32(0x7fc00000), word)
        lo = bf16_round(x.min(-1), "down")
        span = (x.max(-1) - lo).astype(np.float32)
        bad = ~np.isfinite(x).all(-1) | ~np.isfinite(span)
        s = bf16_round(span / np.float32(15), "up")
        s = np.where(s >= tiny, s, np.float32(0)).astype(np.float32)
        inv = np.where(s > 0, np.float32(1) / s, np.float32(0)).astype(np.float32)
        code = np.minimum(np.rint((x - lo[..., None]) * inv[..., None]), 15)
        code = np.where(bad[..., None], 0, code)
        word = (s.view(np.uint32) >> 16) | (lo.view(np.uint32) & np.uint32(0xffff0000))
        return code.astype(np.uint8), np.where(bad, np.uint32(0x7fc0), word)


def values(code, word, bits):
    """float32 values of unpacked codes."""
    with np.errstate(all="ignore"):
        if bits == 8:
            return word.view(np.float32)[..., None] * (code.astype(np.float32) - 128)
        s = (word << np.uint32(16)).view(np.float32)
        lo = (word & np.uint32(0xffff0000)).view(np.float32)
        return (s[..., None] * code.astype(np.float32) + lo[..., None]).astype(np.float32)


def pack(code, bits):
    return code if bits == 8 else (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8)


def unpack(byte, bits):
    return byte if bits == 8 else np.stack((byte & 15, byte >> 4), -1).reshape(
        *byte.shape[:-1], -1)


def tree64(q, kv, table, lens, mask, bits, scale):
    """q [b, m, h, d] -> o, lse, the bound of a score's and weight's error, max |v|."""
    kc, kp, vc, vp = kv
    B, M, H, D = q.shape
    nb, kvh, bs = kp.shape
    o = np.zeros((B, M, H, D))
    lse = np.full((B, M, H), -np.inf)
    tol = np.zeros((B, M, H))
    vmax = np.zeros((B, M, H))
    for b in range(B):
        pre = max(int(lens[b]), 0)
        toks = [t for t in range(pre + M) if t // bs < table.shape[1]
                and 0 <= table[b, t // bs] < nb]
        for i in range(M):
            w = int(mask[b, i]) & ((1 << M) - 1)
            see = [t for t in toks if w and (t < pre or w >> (t - pre) & 1)]
            if not see:
                continue
            blk = np.array([table[b, t // bs] for t in see])
            off = np.array([t % bs for t in see])
            for h in range(H):
                g = h // (H // kvh)
                K = values(unpack(kc[blk, g, off], bits), kp[blk, g, off], bits).astype(float)
                V = values(unpack(vc[blk, g, off], bits), vp[blk, g, off], bits).astype(float)
                s = scale * (K @ q[b, i, h])
                with np.errstate(all="ignore"):
                    top = s.max()
                    e = np.exp(s - top)
                    z = e.sum()
                    o[b, i, h] = e / z @ V
                    lse[b, i, h] = top + np.log(z)
                    vmax[b, i, h] = np.abs(V).max()
                    tol[b, i, h] = (2 ** -20 * scale * (np.abs(K) @ np.abs(q[b, i, h])).max()
                                    + 2 ** -19)
    return o, lse, tol, vmax


# ---- norm + rotation ------------------------------------------------------------

SHAPES = [  # n, heads, kv_heads, dim, rot
    (1, 20, 20, 128, 128), (3, 5, 1, 64, 64), (37, 6, 2, 256, 128), (130, 4, 4, 80, 48),
    (2, 1, 1, 16, 16), (9, 3, 3, 96, 32), (700, 8, 2, 128, 128),
]


def norm_inputs(torch, rng, shape, name, extra=0):
    n, h, k, d, rot = shape
    t = dtype_of(torch, name)
    x = rng.standard_normal((n, (h + 2 * k) * d + extra)) * rng.uniform(0.1, 3, (n, 1))
    x = torch.from_numpy(x).to("cuda", t)
    g = torch.from_numpy(rng.uniform(0.5, 1.5, (2, d)).astype(np.float32)).cuda()
    co, si = rope_tables(50, rot)
    pos = rng.integers(0, 50, n).astype(np.int32)
    if n > 2:
        pos[1], pos[2] = -1, 50           # padding: below and past the tables
    return (x, g[0].contiguous(), g[1].contiguous(), torch.from_numpy(co).cuda(),
            torch.from_numpy(si).cuda(), torch.from_numpy(pos).cuda())


def heads64(t, n, heads, d):
    return t.float().cpu().numpy().astype(float)[:, :heads * d].reshape(n, heads, d)


@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_rope(dev, torch, shape, name, pairs):
    n, h, k, d, rot = shape
    rng = np.random.default_rng(n + d)
    x, gq, gk, co, si, pos = norm_inputs(torch, rng, shape, name)
    q = torch.full((n, h * d + 16), 7.0, device="cuda", dtype=x.dtype)   # strided outputs
    kk = torch.full((n, k * d), 7.0, device="cuda", dtype=x.dtype)
    dev.qk_norm_rope(x, gq, gk, co, si, pos, q[:, :h * d], kk, eps=1e-5, pairs=pairs)
    torch.cuda.synchronize()
    g = np.concatenate([np.tile(gq.cpu().numpy(), (h, 1)), np.tile(gk.cpu().numpy(), (k, 1))])
    want, mag = norm_rope64(heads64(x, n, h + k, d), g.astype(float), co.cpu().numpy().astype(float),
                            si.cpu().numpy().astype(float), pos.cpu().numpy(), float(np.float32(1e-5)),
                            pairs)
    got = np.concatenate([heads64(q, n, h, d), heads64(kk, n, k, d)], 1)
    assert within(torch, got, want, 32 * U * mag + 1e-30, name).all()
    assert (q[:, h * d:].float() == 7).all()                # nothing past the rows
    if n > 2:
        assert not got[1:3].any()


def test_norm_rope_in_place_and_on_another_stream(dev, torch):
    shape = (65, 8, 2, 128, 64)
    n, h, k, d, _ = shape
    x, *rest = norm_inputs(torch, np.random.default_rng(5), shape, "f32")
    q, kk = torch.empty(n, h * d, device="cuda"), torch.empty(n, k * d, device="cuda")
    dev.qk_norm_rope(x, *rest, q, kk)
    y = x.clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    dev.qk_norm_rope(y, *rest, y[:, :h * d], y[:, h * d:(h + k) * d], stream=s)
    s.synchronize()
    assert torch.equal(y[:, :h * d], q) and torch.equal(y[:, h * d:(h + k) * d], kk)
    assert torch.equal(y[:, (h + k) * d:], x[:, (h + k) * d:])


def test_norm_rope_of_zeros_nan_and_infinity(dev, torch):
    shape = (4, 2, 1, 64, 64)
    x, gq, gk, co, si, pos = norm_inputs(torch, np.random.default_rng(6), shape, "f32")
    pos.fill_(3)
    x[0, :64] = 0
    x[1, 5] = float("nan")
    x[2, 64] = float("inf")
    q, kk = torch.empty(4, 128, device="cuda"), torch.empty(4, 64, device="cuda")
    dev.qk_norm_rope(x, gq, gk, co, si, pos, q, kk)
    assert not q[0, :64].any()
    assert q[1, :64].isnan().all() and q[1, 64:].isfinite().all()
    assert q[2, :64].isfinite().all() and q[2, 64:].isnan().any()
    assert q[3].isfinite().all() and kk.isfinite().all()


@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_rope_gradient(dev, torch, shape, name, pairs):
    n, h, k, d, rot = shape
    rng = np.random.default_rng(n * 3 + d)
    x, gq, gk, co, si, pos = norm_inputs(torch, rng, shape, name)
    dq = torch.from_numpy(rng.standard_normal((n, h * d))).to("cuda", x.dtype)
    dk = torch.from_numpy(rng.standard_normal((n, k * d))).to("cuda", x.dtype)
    dx = torch.full_like(x, 7.0)
    dgq, dgk = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    dev.qk_norm_rope_bwd(x, gq, gk, co, si, pos, dq, dk, dx, dgq, dgk, eps=1e-5, pairs=pairs)
    torch.cuda.synchronize()
    g = np.concatenate([np.tile(gq.cpu().numpy(), (h, 1)), np.tile(gk.cpu().numpy(), (k, 1))])
    dy = np.concatenate([heads64(dq, n, h, d), heads64(dk, n, k, d)], 1)
    want, mag, dg, dgm = norm_rope_grad64(
        heads64(x, n, h + k, d), g.astype(float), co.cpu().numpy().astype(float),
        si.cpu().numpy().astype(float), pos.cpu().numpy(), dy, float(np.float32(1e-5)), pairs)
    got = heads64(dx, n, h + k, d)
    assert within(torch, got, want, 128 * U * mag + 1e-30, name).all()
    for have, part in ((dgq, slice(0, h)), (dgk, slice(h, h + k))):
        assert (np.abs(have.cpu().numpy() - dg[:, part].sum((0, 1)))
                <= 96 * U * dgm[:, part].sum((0, 1)) + 1e-30).all()
    assert (dx[:, (h + k) * d:].float() == 7).all()         # the values' part is not touched
    again = [t.clone() for t in (dx, dgq, dgk)]
    dev.qk_norm_rope_bwd(x, gq, gk, co, si, pos, dq, dk, dx, dgq, dgk, eps=1e-5, pairs=pairs)
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dgq, dgk)))   # a fixed order


@pytest.mark.parametrize("pairs", ["half", "adjacent"])
def test_norm_rope_gradient_against_differences(dev, torch, pairs):
    """The kernel's gradients against central differences of the 64-bit
    forward: step e = 1e-4 of values around 1 leaves an error of about e^2."""
    n, h, k, d, rot = shape = (3, 2, 1, 16, 16)
    rng = np.random.default_rng(8)
    x, gq, gk, co, si, pos = norm_inputs(torch, rng, shape, "f32")
    pos.copy_(torch.tensor([3, -1, 49], dtype=torch.int32))
    dq, dk = torch.randn(n, h * d, device="cuda"), torch.randn(n, k * d, device="cuda")
    dx, dgq, dgk = torch.zeros_like(x), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    dev.qk_norm_rope_bwd(x, gq, gk, co, si, pos, dq, dk, dx, dgq, dgk, pairs=pairs)
    x0 = heads64(x, n, h + k, d)
    dy = np.concatenate([heads64(dq, n, h, d), heads64(dk, n, k, d)], 1)
    gains = [gq.cpu().numpy().astype(float), gk.cpu().numpy().astype(float)]
    tabs = co.cpu().numpy().astype(float), si.cpu().numpy().astype(float), pos.cpu().numpy()

    def loss(x, gains):
        g = np.concatenate([np.tile(gains[0], (h, 1)), np.tile(gains[1], (k, 1))])
        return (norm_rope64(x, g, *tabs, 1e-5, pairs)[0] * dy).sum()

    e = 1e-4
    got = heads64(dx, n, h + k, d)
    for at in [(0, 0, 0), (0, 1, 7), (0, 2, 15), (1, 0, 3), (2, 2, 8), (2, 1, 12)]:
        up, down = x0.copy(), x0.copy()
        up[at] += e
        down[at] -= e
        assert abs((loss(up, gains) - loss(down, gains)) / (2 * e) - got[at]) < 1e-4
    for part, have in enumerate((dgq, dgk)):
        for i in (0, 5, 15):
            up, down = [g.copy() for g in gains], [g.copy() for g in gains]
            up[part][i] += e
            down[part][i] -= e
            assert abs((loss(x0, up) - loss(x0, down)) / (2 * e) - have[i].item()) < 1e-4


def test_norm_rope_no_rows(dev, torch):
    x, gq, gk, co, si, pos = norm_inputs(torch, np.random.default_rng(1), (2, 2, 1, 64, 64), "f32")
    e = x[:0]
    dev.qk_norm_rope(e, gq, gk, co, si, pos[:0], e[:, :128], e[:, 128:192])
    dgq, dgk = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    dev.qk_norm_rope_bwd(e, gq, gk, co, si, pos[:0], e[:, :128], e[:, 128:192], e, dgq, dgk)
    assert not dgq.any() and not dgk.any()


# ---- the cache ---------------------------------------------------------------------

def awkward(rng, n, kvh, d):
    """Rows with the ranges a cache meets and some that it must survive."""
    x = rng.standard_normal((n, kvh, d)).astype(np.float32)
    x[0, 0] = 0
    if n > 1:
        x[1, 0] *= 1e-36
        x[1, -1] = 3.25
    if n > 2:
        x[2, 0] = 100 + x[2, 0] * 1e-3    # a small range far from zero
        x[2, -1] = -np.abs(x[2, -1]) * 1e30
    if n > 4:
        x[3, 0, 5] = np.nan
        x[4, 0, d - 1] = -np.inf
    return x


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n,kvh,d,bs", [(1, 1, 128, 16), (8, 20, 128, 64), (37, 3, 64, 5),
                                        (19, 2, 256, 1), (301, 4, 128, 48)])
def test_kv_append_and_read(dev, torch, n, kvh, d, bs, bits, name):
    rng = np.random.default_rng(n + d + bits)
    t = dtype_of(torch, name)
    kx, vx = awkward(rng, n, kvh, d), awkward(rng, n, kvh, d)[:, ::-1].copy()
    rows = torch.zeros(n, 2 * kvh * d + 8, dtype=t, device="cuda")      # K|V rows, strided
    rows[:, :kvh * d] = torch.from_numpy(kx.reshape(n, -1)).to("cuda", t)
    rows[:, kvh * d:2 * kvh * d] = torch.from_numpy(vx.reshape(n, -1)).to("cuda", t)
    K, V = rows[:, :kvh * d], rows[:, kvh * d:2 * kvh * d]
    blocks = -(-n // bs) + 2
    slot = rng.permutation(blocks * bs)[:n].astype(np.int32)
    if n > 8:
        slot[6], slot[7] = -1, blocks * bs        # outside: skipped
    cache = dev.kv_cache(blocks, bs, kvh, d, bits)
    dev.kv_append(K, V, torch.from_numpy(slot).cuda(), *cache)
    torch.cuda.synchronize()
    want = [np.zeros(tuple(c.shape), np.uint8 if i % 2 == 0 else np.uint32)
            for i, c in enumerate(cache)]
    for j, X in enumerate((K, V)):
        code, word = quantise(X.float().cpu().numpy().reshape(n, kvh, d), bits)
        for i in range(n):
            if 0 <= slot[i] < blocks * bs:
                want[2 * j][slot[i] // bs, :, slot[i] % bs] = pack(code[i], bits)
                want[2 * j + 1][slot[i] // bs, :, slot[i] % bs] = word[i]
    for have, need in zip(cache, want):
        have = have.cpu().numpy()
        assert np.array_equal(have.view(need.dtype), need)
    ko = torch.full((n, kvh * d + 8), 7.0, dtype=t, device="cuda")
    vo = torch.full((n, kvh * d), 7.0, dtype=t, device="cuda")
    dev.kv_read(torch.from_numpy(slot).cuda(), *cache, ko[:, :kvh * d], vo)
    torch.cuda.synchronize()
    for have, j in ((ko[:, :kvh * d], 0), (vo, 1)):
        inside = (slot >= 0) & (slot < blocks * bs)
        at = np.where(inside, slot, 0)
        y = values(unpack(want[2 * j][at // bs, :, at % bs], bits),
                   want[2 * j + 1][at // bs, :, at % bs], bits)
        y = np.where(inside[:, None, None], y, 0).reshape(n, -1)
        y = torch.from_numpy(np.ascontiguousarray(y)).to(t)
        assert torch.equal(have.cpu().nan_to_num(nan=123.0), y.nan_to_num(nan=123.0))
        if n > 4:
            assert have[3 if j == 0 else 4].isnan().any()
    assert (ko[:, kvh * d:].float() == 7).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_kv_values_are_near(dev, torch, bits):
    """Half a step of the code: |x - value| <= s / 2 and the roundings."""
    n, kvh, d = 50, 2, 128
    x = torch.randn(n, kvh * d, device="cuda")
    cache = dev.kv_cache(4, 16, kvh, d, bits)
    slot = torch.arange(n, dtype=torch.int32, device="cuda")
    dev.kv_append(x, x, slot, *cache)
    k, v = torch.empty_like(x), torch.empty_like(x)
    dev.kv_read(slot, *cache, k, v)
    r = x.view(n, kvh, d)
    s = r.abs().amax(-1) / 127 if bits == 8 else (r.amax(-1) - r.amin(-1)) / 15 * 1.03
    assert ((k - x).view(n, kvh, d).abs() <= s[..., None] * 0.501 + 1e-6).all()
    assert torch.equal(k, v)


@pytest.mark.parametrize("bits", [8, 4])
def test_kv_move(dev, torch, bits):
    B, kvh, d, bs, nb = 3, 2, 64, 7, 12
    rng = np.random.default_rng(bits)
    cache = dev.kv_cache(nb, bs, kvh, d, bits)
    for c in cache:
        c.copy_(torch.from_numpy(rng.integers(0, 200, tuple(c.shape))).to(c.dtype))
    perm = rng.permutation(nb * bs)
    src = np.stack([perm[20 * b:20 * b + 5] for b in range(B)]).astype(np.int32)
    # paths whose destinations are sources of later pairs, a self move, skips
    dst = np.stack([np.roll(src[0], 1), [src[1][0], src[1][0], 0, 0, 0], src[2]]).astype(np.int32)
    dst[1, 1:] = perm[80:84]
    dst[1, 3], src[1, 4] = nb * bs, -1
    want = [c.cpu().numpy().copy() for c in cache]
    old = [w.copy() for w in want]
    for w, o in zip(want, old):
        for b in range(B):
            for a, z in zip(src[b], dst[b]):
                if 0 <= a < nb * bs and 0 <= z < nb * bs:
                    w[z // bs, :, z % bs] = o[a // bs, :, a % bs]
    dev.kv_move(torch.from_numpy(src).cuda(), torch.from_numpy(dst).cuda(), *cache, d)
    for c, w in zip(cache, want):
        assert np.array_equal(c.cpu().numpy(), w)


# ---- attention -----------------------------------------------------------------------

def chain(m):
    return [(1 << (i + 1)) - 1 for i in range(m)]


def tree(rng, m):
    rows = []
    for i in range(m):
        up = 0 if i == 0 else rows[rng.integers(max(0, i - 5), i)]
        rows.append(up | 1 << i)
    return rows


def attn_inputs(torch, rng, B, M, H, kvh, d, bits, bs, lens, masks, name, extra_blocks=2,
                blocks=None):
    per = -(-(max(max(lens), 0) + M) // bs)
    nb = B * per + extra_blocks
    x = rng.standard_normal((2, nb, kvh, bs, d)).astype(np.float32)
    x[0] *= np.where(rng.random(d) < 0.1, 4, 1)
    kv = []
    for part in x:
        code, word = quantise(part, bits)
        kv += [pack(code, bits), word]
    table = rng.permutation(nb)[:B * per].reshape(B, per).astype(np.int32)
    mask = np.array([[w - (1 << 64) if w >> 63 else w for w in row] for row in masks], np.int64)
    t = dtype_of(torch, name)
    q = torch.from_numpy(rng.standard_normal((B * M, H * d + 32))).to("cuda", t)
    return q, kv, table, np.array(lens, np.int32), mask


def device(torch, kv, table, lens, mask):
    c = [torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda() for a in kv]
    return c, [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (table, lens, mask)]


def check_tree(dev, torch, q, kv, table, lens, mask, bits, H, d, scale=None, stream=None,
               workspace=None):
    B, M = mask.shape
    cache, (tt, tl, tm) = device(torch, kv, table, lens, mask)
    Q = q[:, 16:16 + H * d]                       # a strided view into wider rows
    o = torch.full((B * M, H * d + 8), 7.0, device="cuda", dtype=q.dtype)
    lse = torch.full((B * M, H), 7.0, device="cuda")
    torch.cuda.synchronize()
    dev.tree_attn(Q, *cache, tt, tl, tm, o[:, :H * d], d, scale=scale, lse=lse, stream=stream,
                  workspace=workspace)
    torch.cuda.synchronize()
    want, wl, eps, vmax = tree64(Q.float().cpu().numpy().astype(float).reshape(B, M, H, d), kv,
                                 table, lens, mask, bits, d ** -0.5 if scale is None else scale)
    got = o[:, :H * d].float().cpu().numpy().astype(float).reshape(B, M, H, d)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    tol = np.broadcast_to((eps * vmax)[..., None], want.shape).copy()
    name = "f32"
    if q.dtype == torch.bfloat16:
        name = "bf16"
        tol += 2 ** -11 * vmax[..., None]
    with np.errstate(all="ignore"):
        bad = ~within(torch, got, want, tol, name) & ~nan
    assert not bad.any(), (np.abs(got - want)[bad].max(), tol[bad].min())
    gl = lse.cpu().numpy().reshape(B, M, H)
    fin = np.isfinite(wl)
    assert np.array_equal(np.isfinite(gl), fin) and (gl[~fin & ~np.isnan(wl)] == -np.inf).all()
    lt = (eps[fin] if name == "f32" else 2 ** -9) + 2 ** -20 * np.abs(wl[fin])
    assert (np.abs(gl[fin] - wl[fin]) <= lt).all()
    assert (o[:, H * d:].float() == 7).all()
    return got, gl


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("B,M,H,kvh,d,bs,lens", [
    (1, 1, 1, 1, 128, 16, [0]),                     # a token that sees itself only
    (1, 1, 4, 4, 128, 16, [1]),
    (2, 1, 8, 2, 64, 16, [127, 128]),               # a tile that ends with the keys, and one past
    (3, 5, 6, 2, 128, 7, [0, 33, 200]),             # pages that end inside a tile
    (2, 7, 4, 1, 256, 48, [31, 300]),
    (1, 16, 8, 1, 64, 1, [65]),                     # pages of one token, 128 rows of a head
    (2, 64, 3, 3, 128, 64, [0, 150]),               # every bit of the masks
    (1, 33, 8, 2, 128, 32, [95]),
    (5, 2, 2, 1, 128, 256, [4, 700, -3, 1, 64]),    # a negative length is none
])
def test_tree_attn(dev, torch, B, M, H, kvh, d, bs, lens, bits, name):
    rng = np.random.default_rng(B * 100 + M + d + bits)
    masks = [chain(M) if b % 2 else tree(rng, M) for b in range(B)]
    args = attn_inputs(torch, rng, B, M, H, kvh, d, bits, bs, lens, masks, name)
    check_tree(dev, torch, *args, bits, H, d)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
def test_tree_attn_over_many_parts(dev, torch, bits, name):
    """One key head and a long context: every CTA has a part of the same item."""
    rng = np.random.default_rng(3)
    args = attn_inputs(torch, rng, 1, 3, 2, 1, 128, bits, 64, [70001], [tree(rng, 3)], name)
    check_tree(dev, torch, *args, bits, 2, 128)


@pytest.mark.parametrize("bits", [8, 4])
def test_tree_attn_unused_nodes_and_foreign_bits(dev, torch, bits):
    rng = np.random.default_rng(11)
    M = 6
    m = tree(rng, M)
    m[1] = m[4] = 0                                 # unused
    m[5] |= 0xff << 50                              # bits past the nodes are not read
    m[3] = 1 << 2                                   # a node that does not see itself
    args = attn_inputs(torch, rng, 2, M, 4, 2, 128, bits, 16, [0, 90], [m, m], "f32")
    got, lse = check_tree(dev, torch, *args, bits, 4, 128)
    assert not got[:, [1, 4]].any() and (lse[:, [1, 4]] == -np.inf).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("bad", [-1, 1 << 20])
def test_tree_attn_blocks_outside_the_pool_hold_no_keys(dev, torch, bits, bad):
    rng = np.random.default_rng(12)
    q, kv, table, lens, mask = attn_inputs(torch, rng, 2, 2, 2, 1, 64, bits, 16, [100, 40],
                                           [chain(2), chain(2)], "f32")
    table[0, 2] = bad
    table[1, :] = bad                               # no key at all
    got, lse = check_tree(dev, torch, q, kv, table, lens, mask, bits, 2, 64)
    assert not got[1].any() and (lse[1] == -np.inf).all()
    short = table[:, :3].copy()                     # a table that ends before the keys do
    check_tree(dev, torch, q, kv, short, lens, mask, bits, 2, 64)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("which", [1, 3])           # the keys' or the values' words
def test_tree_attn_nan_reaches_only_rows_that_see_it(dev, torch, bits, which):
    rng = np.random.default_rng(13)
    M, L = 5, 40
    m = [1, 3, 5, 9, 17]                            # all see node 0, else themselves
    q, kv, table, lens, mask = attn_inputs(torch, rng, 1, M, 2, 1, 128, bits, 16, [L], [m], "f32")
    t = L + 3                                       # node 3 alone sees it
    kv[which][table[0, t // 16], 0, t % 16] = 0x7fc00000 if bits == 8 else 0x7fc0
    got, _ = check_tree(dev, torch, q, kv, table, lens, mask, bits, 2, 128)
    assert np.isnan(got[0, 3]).all() and np.isfinite(got[0, [0, 1, 2, 4]]).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_tree_attn_scales_far_apart(dev, torch, bits, name):
    """Value scales from 2^-100 to 2^60 with the largest last, query rows from
    tiny to large, scores in the hundreds, and a scale argument."""
    rng = np.random.default_rng(14)
    q, kv, table, lens, mask = attn_inputs(torch, rng, 1, 4, 2, 1, 128, bits, 32, [300],
                                           [chain(4)], name)
    nb, kvh, bs, _ = kv[0].shape
    flat = np.empty(kv[3].shape, np.float32)
    order = np.argsort(np.argsort(table[0]))
    flat[...] = 1.0
    for j, blk in enumerate(table[0]):
        flat[blk] = 2.0 ** (-100 + 160 * j / (len(table[0]) - 1))
    x = rng.standard_normal(kv[2].shape[:3] + (128,)).astype(np.float32) * flat[..., None]
    code, word = quantise(x, bits)
    kv[2], kv[3] = pack(code, bits), word
    q *= torch.tensor([1e-30, 1.0, 40.0, 1e-3], device="cuda", dtype=q.dtype)[:, None]
    check_tree(dev, torch, q, kv, table, lens, mask, bits, 2, 128, scale=0.25)


# More than 16 rows a key head of 128 values, or 32 of 64, in bfloat16 take the
# tcgen05 form where the pages are whole 16-key runs: 32 rows at a time up to
# 32, else 64.
WIDE = [(8, 8, 2), (33, 2, 1), (64, 4, 1), (17, 3, 1)]      # nodes, heads, kv_heads


@pytest.mark.parametrize("M,H,kvh", WIDE)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("bs,lens", [(16, [0, 300, 1, 126]), (48, [129, 0]), (256, [700]),
                                     (5, [40, 130])])
def test_wide_tree_attn(dev, torch, M, H, kvh, d, bits, bs, lens):
    rng = np.random.default_rng(M + d + bits + bs)
    masks = [chain(M) if b % 2 else tree(rng, M) for b in range(len(lens))]
    masks[-1][M // 2:] = [0] * (M - M // 2)             # a sequence with unused nodes
    masks[0][1] = 0
    args = attn_inputs(torch, rng, len(lens), M, H, kvh, d, bits, bs, lens, masks, "bf16")
    got, lse = check_tree(dev, torch, *args, bits, H, d)
    assert not got[0, 1].any() and (lse[0, 1] == -np.inf).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("M,H", [(5, 4), (9, 8)])
def test_wide_tree_attn_over_many_parts(dev, torch, bits, M, H):
    rng = np.random.default_rng(30)
    args = attn_inputs(torch, rng, 1, M, H, 1, 128, bits, 64, [40001], [tree(rng, M)], "bf16")
    check_tree(dev, torch, *args, bits, H, 128)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("bad", [-1, 1 << 20])
def test_wide_tree_attn_blocks_outside_the_pool(dev, torch, bits, bad):
    rng = np.random.default_rng(31)
    M = 20
    q, kv, table, lens, mask = attn_inputs(torch, rng, 2, M, 2, 1, 64, bits, 16, [300, 40],
                                           [chain(M)] * 2, "bf16")
    table[0, [2, 9, 10]] = bad
    table[1, :] = bad
    got, lse = check_tree(dev, torch, q, kv, table, lens, mask, bits, 2, 64)
    assert not got[1].any() and (lse[1] == -np.inf).all()
    check_tree(dev, torch, q, kv, table[:, :3].copy(), lens, mask, bits, 2, 64)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("which", [1, 3])
@pytest.mark.parametrize("M,H", [(20, 1), (20, 2)])
def test_wide_tree_attn_nan_reaches_only_rows_that_see_it(dev, torch, bits, which, M, H):
    rng = np.random.default_rng(32)
    L = 140
    m = [1 | 1 << i for i in range(M)]                  # all see node 0, else themselves
    q, kv, table, lens, mask = attn_inputs(torch, rng, 1, M, H, 1, 128, bits, 16, [L], [m], "bf16")
    t = L + 3
    kv[which][table[0, t // 16], 0, t % 16] = 0x7fc00000 if bits == 8 else 0x7fc0
    got, _ = check_tree(dev, torch, q, kv, table, lens, mask, bits, H, 128)
    others = [i for i in range(M) if i != 3]
    assert np.isnan(got[0, 3]).all() and np.isfinite(got[0, others]).all()
    kv[which][table[0, 1], 0, 2] = 0x7fc00000 if bits == 8 else 0x7fc0    # a prefix key: all see it
    got, _ = check_tree(dev, torch, q, kv, table, lens, mask, bits, H, 128)
    assert np.isnan(got).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_wide_tree_attn_scales_far_apart(dev, torch, bits):
    """Scores that keep rising from key to key, value scales from 2^-100 to
    2^60, query rows from tiny to large: every way to move a reference."""
    rng = np.random.default_rng(33)
    M = 24
    q, kv, table, lens, mask = attn_inputs(torch, rng, 1, M, 1, 1, 128, bits, 32, [900],
                                           [chain(M)], "bf16")
    flat = np.ones(kv[3].shape, np.float32)
    for j, blk in enumerate(table[0]):
        flat[blk] = 2.0 ** (-100 + 160 * j / (len(table[0]) - 1))
    x = rng.standard_normal(kv[2].shape[:3] + (128,)).astype(np.float32) * flat[..., None]
    code, word = quantise(x, bits)
    kv[2], kv[3] = pack(code, bits), word
    y = values(unpack(kv[0], bits), kv[1], bits)
    for j, blk in enumerate(table[0]):                  # keys along one direction, longer and longer
        y[blk] = y[blk] * 0.1 + np.float32(0.1 * j)
    code, word = quantise(y, bits)
    kv[0], kv[1] = pack(code, bits), word
    rows = torch.logspace(-30, 1, M, device="cuda")
    q.copy_((q.float().abs() * rows[:, None]).to(q.dtype))
    check_tree(dev, torch, q, kv, table, lens, mask, bits, 1, 128, scale=0.25)


def test_wide_tree_attn_rows_of_nan_and_infinity(dev, torch):
    rng = np.random.default_rng(34)
    M = 20
    q, kv, table, lens, mask = attn_inputs(torch, rng, 1, M, 1, 1, 128, 8, 16, [200], [chain(M)],
                                           "bf16")
    q[1, 16 + 3] = float("nan")
    q[2, 16 + 100] = float("inf")
    cache, (tt, tl, tm) = device(torch, kv, table, lens, mask)
    o = torch.empty(M, 128, device="cuda", dtype=q.dtype)
    dev.tree_attn(q[:, 16:16 + 128], *cache, tt, tl, tm, o, 128)
    assert o[1].isnan().all() and o[2].isnan().any()
    assert o[0].isfinite().all() and o[3:].isfinite().all()
    from nelisp_cuda import _lib as L
    assert L.load().nl_wait_status() == L.NL_OK


def test_wide_tree_attn_streams_and_graph(dev, torch):
    rng = np.random.default_rng(35)
    q, kv, table, lens, mask = attn_inputs(torch, rng, 3, 16, 8, 2, 128, 8, 16, [3000, 17, 900],
                                           [chain(16)] * 3, "bf16")
    cache, (tt, tl, tm) = device(torch, kv, table, lens, mask)
    Q = q[:, :1024]
    want = torch.empty(48, 1024, device="cuda", dtype=q.dtype)
    dev.tree_attn(Q, *cache, tt, tl, tm, want, 128)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(want) for _ in range(8)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        dev.tree_attn(Q, *cache, tt, tl, tm, o, 128, stream=streams[i % 2])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    g, o = torch.cuda.CUDAGraph(), torch.zeros_like(want)
    with torch.cuda.graph(g):
        for _ in range(4):
            dev.tree_attn(Q, *cache, tt, tl, tm, o, 128)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want)
    # the workspace that the query asks for is enough, to the byte
    from nelisp_cuda import _lib as L
    n = L.load().nl_tree_attn_workspace_bytes(16, 8, 2, 128)
    ws = torch.full((n + 4096,), 7, dtype=torch.uint8, device="cuda")
    o.zero_()
    dev.tree_attn(Q, *cache, tt, tl, tm, o, 128, workspace=ws[:n])
    assert torch.equal(o, want) and (ws[n:] == 7).all()


def test_tree_attn_rows_of_nan_and_infinity(dev, torch):
    rng = np.random.default_rng(15)
    q, kv, table, lens, mask = attn_inputs(torch, rng, 1, 3, 2, 1, 128, 8, 16, [50], [chain(3)],
                                           "f32")
    q[1, 16 + 3] = float("nan")
    q[2, 16 + 128] = float("inf")
    cache, (tt, tl, tm) = device(torch, kv, table, lens, mask)
    o = torch.empty(3, 256, device="cuda")
    dev.tree_attn(q[:, 16:16 + 256], *cache, tt, tl, tm, o, 128)
    o = o.view(3, 2, 128)
    assert o[1, 0].isnan().all() and o[2, 1].isnan().any()
    assert o[0].isfinite().all() and o[1, 1].isfinite().all() and o[2, 0].isfinite().all()


def test_tree_attn_streams_and_workspaces(dev, torch):
    """Calls on two streams at once, each with a workspace of its own, and one
    captured into a graph, give the bits of a call alone."""
    rng = np.random.default_rng(16)
    q, kv, table, lens, mask = attn_inputs(torch, rng, 3, 4, 8, 2, 128, 8, 16, [3000, 17, 900],
                                           [chain(4)] * 3, "bf16")
    cache, (tt, tl, tm) = device(torch, kv, table, lens, mask)
    Q = q[:, :1024]
    want = torch.empty(12, 1024, device="cuda", dtype=q.dtype)
    dev.tree_attn(Q, *cache, tt, tl, tm, want, 128)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(want) for _ in range(8)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        dev.tree_attn(Q, *cache, tt, tl, tm, o, 128, stream=streams[i % 2])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    g, o = torch.cuda.CUDAGraph(), torch.zeros_like(want)
    with torch.cuda.graph(g):
        dev.tree_attn(Q, *cache, tt, tl, tm, o, 128)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want)


@pytest.mark.parametrize("bits,d", [(8, 256), (4, 256)])
def test_offsets_past_32_bits(dev, torch, bits, d):
    """A pool whose code arrays pass 2^32 bytes: rows written, read, moved and
    attended at its far end."""
    bs = 64
    nb = (1 << 32) // (d * bits // 8 * bs) + 8
    cache = (torch.empty(nb, 1, bs, d * bits // 8, dtype=torch.uint8, device="cuda"),
             torch.empty(nb, 1, bs, dtype=torch.int32, device="cuda"),
             torch.empty(nb, 1, bs, d * bits // 8, dtype=torch.uint8, device="cuda"),
             torch.empty(nb, 1, bs, dtype=torch.int32, device="cuda"))
    n = 100
    x = torch.randn(2, n, d, device="cuda")
    table = torch.tensor([[nb - 1, nb - 4]], dtype=torch.int32, device="cuda")
    at = torch.arange(n, device="cuda")
    slot = (table[0][at // bs] * bs + at % bs).int()
    dev.kv_append(x[0], x[1], slot, *cache)
    k, v = torch.empty(n, d, device="cuda"), torch.empty(n, d, device="cuda")
    dev.kv_read(slot, *cache, k, v)
    assert (k - x[0]).abs().max() < 0.5
    q = torch.randn(1, d, device="cuda")
    o = torch.empty_like(q)
    ln = torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    one = torch.ones(1, 1, dtype=torch.int64, device="cuda")
    dev.tree_attn(q, *cache, table, ln, one, o, d)
    p = torch.softmax((q.double() @ k.double().T) * d ** -0.5, -1)
    assert (o - (p @ v.double())).abs().max() < 1e-5 * v.abs().max()
    to = torch.tensor([[(nb - 7) * bs + 3]], dtype=torch.int32, device="cuda")
    dev.kv_move(slot[5:6].view(1, 1), to, *cache, d)
    k2, v2 = torch.empty(1, d, device="cuda"), torch.empty(1, d, device="cuda")
    dev.kv_read(to[0], *cache, k2, v2)
    assert torch.equal(k2[0], k[5]) and torch.equal(v2[0], v[5])


def test_empty_calls(dev, torch):
    cache = dev.kv_cache(2, 16, 1, 64, 8)
    e, s = torch.empty(0, 64, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    dev.kv_append(e, e, s, *cache)
    dev.kv_read(s, *cache, e, e)
    dev.kv_move(s.view(0, 1), s.view(0, 1), *cache, 64)
    dev.tree_attn(e, *cache, s.view(0, 1), s, torch.empty(0, 1, dtype=torch.int64, device="cuda"),
                  e, 64)
    # an empty pool: every read is of nothing
    none = dev.kv_cache(0, 16, 1, 64, 8)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.ones(1, 64, device="cuda")
    dev.kv_append(x, x, one, *none)
    k, v = torch.ones(1, 64, device="cuda"), torch.ones(1, 64, device="cuda")
    dev.kv_read(one, *none, k, v)
    assert not k.any() and not v.any()
    o = torch.ones(1, 64, device="cuda")
    dev.tree_attn(x, *none, one.view(1, 1), one, torch.ones(1, 1, dtype=torch.int64, device="cuda"),
                  o, 64)
    assert not o.any()


# ---- refusals ---------------------------------------------------------------------------

def test_python_refusals(dev, torch):
    x, gq, gk, co, si, pos = norm_inputs(torch, np.random.default_rng(1), (4, 2, 1, 64, 64), "f32")
    q, k = torch.empty(4, 128, device="cuda"), torch.empty(4, 64, device="cuda")
    with pytest.raises(ValueError):
        dev.qk_norm_rope(x, gq, gk, co, si, pos, q.bfloat16(), k)
    with pytest.raises(ValueError):
        dev.qk_norm_rope(x, gq, gk, co, si, pos.long(), q, k)
    with pytest.raises(ValueError):
        dev.qk_norm_rope(x, gq, gk, co, si, pos, q, k, pairs="third")
    with pytest.raises(ValueError):
        dev.qk_norm_rope(x.half(), gq, gk, co, si, pos, q.half(), k.half())
    with pytest.raises(ValueError):
        dev.qk_norm_rope(x[:3], gq, gk, co, si, pos, q, k)
    cache = dev.kv_cache(2, 16, 1, 64, 8)
    s = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        dev.kv_append(k, k[:, :32], s, *cache)
    with pytest.raises(ValueError):
        dev.kv_append(k, k, s[:3], *cache)
    with pytest.raises(ValueError):
        dev.kv_cache(2, 16, 1, 64, 5)
    with pytest.raises(ValueError):
        dev.kv_move(s.view(2, 2), s.view(2, 2), *cache, 96)
    with pytest.raises(ValueError):
        dev.tree_attn(k, *cache, s.view(4, 1), s, torch.ones(4, 1, dtype=torch.int32,
                                                             device="cuda"), k, 64)


def test_library_refusals(dev, torch):
    """Each is a status with a message, and nothing is launched."""
    from nelisp_cuda import _lib as L
    x, gq, gk, co, si, pos = norm_inputs(torch, np.random.default_rng(1), (4, 2, 1, 64, 64), "f32")
    q, k = torch.empty(4, 128, device="cuda"), torch.empty(4, 64, device="cuda")
    before = dev.launch_count()
    with pytest.raises(L.NlError, match="head size"):
        g = torch.ones(20, device="cuda")
        dev.qk_norm_rope(x[:, :60], g, g, co[:, :8].contiguous(), si[:, :8].contiguous(), pos,
                         q[:, :40], k[:, :20])
    with pytest.raises(L.NlError, match="rotated part"):
        dev.qk_norm_rope(x, gq, gk, co[:, :3].contiguous(), si[:, :3].contiguous(), pos, q, k)
    with pytest.raises(L.NlError, match="aligned"):
        flat = torch.empty(4 * 192 + 1, device="cuda")
        dev.qk_norm_rope(flat[1:].view(4, 192), gq, gk, co, si, pos, q, k)
    with pytest.raises(L.NlError, match="workspace"):
        dev.qk_norm_rope_bwd(x, gq, gk, co, si, pos, q, k, x.clone(), gq.clone(), gk.clone(),
                             workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    s = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(L.NlError, match="head size"):
        dev.kv_append(k[:, :32], k[:, :32], s, *dev.kv_cache(2, 16, 1, 32, 8))
    lib, p = L.load(), 16

    def cache(fmt=8, kvh=1, hd=64, bs=16, nb=1, kc=p, kp=p, vc=p, vp=p):
        return fmt, kvh, hd, bs, nb, kc, kp, vc, vp

    def rows(pool, dtype=0, n=1, slot=p, k=p, ks=64, v=p, vs=64):
        return PACKED["nl_kv_rows"].pack(*pool, dtype, n, slot, k, ks, v, vs)

    def tree(pool, dtype=0, batch=1, nodes=1, heads=1, mb=1, scale=0.1, q=p, qs=64, table=p, ln=p,
             mask=p, o=p, os=64, lse=0, ws=p, wsb=1 << 30):
        return PACKED["nl_tree_attn_dev"].pack(*pool, dtype, batch, nodes, heads, mb, scale, q,
                                                 qs, table, ln, mask, o, os, lse, ws, wsb)
    move = PACKED["nl_kv_move_dev"].pack
    cases = [("nl_kv_append_dev", rows(cache(fmt=5)), "format"),
             ("nl_kv_append_dev", rows(cache(), dtype=2), "type"),
             ("nl_kv_append_dev", rows(cache(bs=1 << 16, nb=1 << 15)), "slots"),
             ("nl_kv_append_dev", rows(cache(kvh=4, bs=1 << 16, nb=1 << 14), ks=256, vs=256),
              "rows"),
             ("nl_kv_append_dev", rows(cache(), ks=32), "stride"),
             ("nl_kv_append_dev", rows(cache(hd=32)), "head size"),
             ("nl_kv_read_dev", rows(cache(), slot=0), "slots"),
             ("nl_kv_read_dev", rows(cache(), v=8), "aligned"),
             ("nl_kv_move_dev", move(*cache(), p, p, 1, 65), "count"),
             ("nl_kv_move_dev", move(*cache(), 0, p, 1, 1), "null"),
             ("nl_tree_attn_dev", tree(cache(), nodes=65), "nodes"),
             ("nl_tree_attn_dev", tree(cache(kvh=2), heads=3), "heads"),
             ("nl_tree_attn_dev", tree(cache(hd=96), qs=96, os=96), "head size"),
             ("nl_tree_attn_dev", tree(cache(), scale=0.0), "scale"),
             ("nl_tree_attn_dev", tree(cache(), scale=math.inf), "scale"),
             ("nl_tree_attn_dev", tree(cache(), scale=math.nan), "scale"),
             ("nl_tree_attn_dev", tree(cache(), qs=63), "strides"),
             ("nl_tree_attn_dev", tree(cache(), o=8), "aligned"),
             ("nl_tree_attn_dev", tree(cache(), mask=0), "null"),
             ("nl_tree_attn_dev", tree(cache(), wsb=100), "workspace"),
             ("nl_tree_attn_dev", tree(cache(bs=1 << 16), batch=64, mb=1 << 16), "too much"),
             ("nl_tree_attn_dev", tree(cache(fmt=6)), "format"),
             ("nl_tree_attn_dev", tree(cache(kc=4)), "unaligned")]
    cases += [(name, None, "null") for name in
              ("nl_qk_norm_rope_dev", "nl_qk_norm_rope_bwd_dev", "nl_kv_append_dev",
               "nl_kv_read_dev", "nl_kv_move_dev", "nl_tree_attn_dev")]
    for name, args, word in cases:
        assert getattr(lib, name)(args, None) == L.NL_ERROR, (name, word)
        assert word in lib.nl_last_error().decode(), (name, word, lib.nl_last_error())
    assert dev.launch_count() == before
