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


@pytest.mark.parametrize("name,M,H,d", [("f32", 60, 1, 128), ("bf16", 60, 1, 128),
                                        ("bf16", 20, 1, 64), ("bf16", 60, 2, 64)])
@pytest.mark.parametrize("bits", [8, 4])
def test_rows_that_meet_their_first_value_late(dev, torch, name, M, H, d, bits):  # noqa: F811
    """No prefix key (its pages are outside the pool), and nodes over several
    tiles: the first ones, of ordinary size, are seen by themselves alone, and the
    last by themselves and small."""
    rng = np.random.default_rng(6)
    mask = [1 << i for i in range(M)]
    for L in (112, 96):
        q, kv, table, lens, m = S.attn_inputs(torch, rng, 1, M, H, 1, d, bits, 16, [L], [mask], name)
        table[0, :L // 16] = -1
        for i in range(M):
            put(kv, table, L + i, rng.standard_normal(d) * (1.0 if i < M // 2 else 1e-12), bits)
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


# ---- long contexts in one part ---------------------------------------------------------
#
# 160 sequences over the same pages give every CTA items of its own, so a part is
# as long as the context.

def long_case(torch, name, M, H, d, bits, bs, n, B, shape):  # noqa: F811
    """Q, cache, table, lengths, masks, and keys and values as float64: scores
    gamma_row a_t that are flat, or rise or fall along the keys, and positive values
    whose mean goes with the score."""
    g = torch.Generator(device="cuda").manual_seed(n + d + M)
    nb = -(-(n + M) // bs)
    N = nb * bs
    u = torch.randn(d, device="cuda", generator=g)
    u /= u.norm()
    a = torch.randn(N, device="cuda", generator=g)
    along = torch.arange(N, device="cuda") / N
    trend = {"flat": 0 * along, "rising": 8 * along, "falling": -8 * along}[shape]
    V = 1.5 + torch.rand(d, device="cuda", generator=g) * torch.tanh(a)[:, None] \
        + 0.3 * torch.rand(N, d, device="cuda", generator=g)
    if shape != "flat":
        V = V * torch.exp2(2 * along)[:, None]
    parts = []
    for x in ((a + trend)[:, None] * u * d ** 0.5, V):
        code, word = S.quantise(x.cpu().numpy(), bits)
        y = torch.from_numpy(S.values(code, word, bits)).double().cuda()
        parts.append((torch.from_numpy(S.pack(code, bits)).cuda().view(nb, 1, bs, -1).contiguous(),
                      torch.from_numpy(word.view(np.int32)).cuda().view(nb, 1, bs).contiguous(), y))
    (kc, kp, k), (vc, vp, v) = parts
    rows = B * M * H
    gamma = torch.linspace(-1, 1, rows, device="cuda")
    gamma = gamma[torch.randperm(rows, device="cuda", generator=g)]
    if shape != "flat":
        gamma = 0.75 + gamma / 4
    q = (gamma[:, None] * u).view(B * M, H * d).to(S.dtype_of(torch, name))
    table = torch.arange(nb, dtype=torch.int32, device="cuda").expand(B, nb).contiguous()
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    mask = torch.tensor(S.chain(M), dtype=torch.int64, device="cuda").expand(B, M).contiguous()
    return q, (kc, kp, vc, vp), table, lens, mask, k, v


def long_check(dev, torch, name, M, H, d, bits, bs, n, shape, B=160):  # noqa: F811
    """The relative error of the outputs of four sequences."""
    q, cache, table, lens, mask, k, v = long_case(torch, name, M, H, d, bits, bs, n, B, shape)
    o, lse = torch.empty_like(q), torch.empty(B * M, H, device="cuda")
    dev.tree_attn(q, *cache, table, lens, mask, o, d, lse=lse)
    off = []
    for b in range(0, B, B // 4):
        for i in range(M):
            row, see = b * M + i, n + i + 1
            x = q[row].view(H, d).double()
            s = x @ k[:see].T * d ** -0.5
            want = torch.softmax(s, -1) @ v[:see]
            far = (x.abs() @ k[:see].abs().T).amax(-1) * d ** -0.5
            ls = torch.logsumexp(s, -1)
            assert ((lse[row].double() - ls).abs() <=
                    2 ** -20 * far + 2 ** -19 + 2 ** -20 * ls.abs()).all()
            vmax = v[:see].abs().max()
            tol = (2 ** -20 * far + 2 ** -19)[:, None] * vmax
            if name == "bf16":                  # the weights' rounding, and the output's
                tol = tol + 2 ** -11 * vmax + 2 ** -8 * want.abs()
            got = o[row].view(H, d).double()
            assert ((got - want).abs() <= tol).all()
            off.append(((got - want) / want).flatten())
    from nelisp_cuda import _lib as L
    assert L.load().nl_wait_status() == L.NL_OK
    return torch.cat(off)


# One node of 8 and 16 heads, 128 rows with pages that the tcgen05 form does not
# take, heads of 256; the tcgen05 form with 20, 64 and 128 rows, heads of 64 and 128.
@pytest.mark.parametrize("M,H,d,bits,bs,n", [
    (1, 8, 128, 8, 64, 300000), (1, 16, 128, 4, 64, 150000), (32, 4, 128, 8, 40, 200000),
    (16, 4, 256, 8, 64, 200000), (20, 1, 128, 8, 64, 100000), (16, 4, 128, 8, 64, 100000),
    (16, 4, 128, 8, 64, 300000), (16, 4, 64, 8, 64, 100000), (32, 4, 128, 4, 64, 100000),
])
def test_long_contexts_do_not_drift(dev, torch, M, H, d, bits, bs, n):  # noqa: F811
    """The tensor core cuts what it adds to an accumulator: positive values lose
    a little at every addition, 1e-7 at most.  The sums are taken out of it after
    2,048 additions, 2^-12; the mean of at least 4,096 roundings to bfloat16 (2^-9 /
    sqrt 3 each) stays within 2^-14."""
    B = 600 if M == 1 else 160                  # for parts as long as the context
    off = long_check(dev, torch, "bf16", M, H, d, bits, bs, n, "flat", B)
    assert off.numel() >= 4096 and off.mean().abs() <= 2 ** -12 + 2 ** -14, off.mean()


@pytest.mark.parametrize("shape", ["rising", "falling"])
@pytest.mark.parametrize("name,M,H,d,bs", [
    ("bf16", 1, 8, 128, 64), ("bf16", 32, 4, 128, 40), ("bf16", 4, 2, 256, 64),
    ("bf16", 20, 1, 128, 64), ("bf16", 16, 4, 64, 64), ("f32", 2, 2, 128, 64)])
@pytest.mark.parametrize("bits", [8, 4])
def test_long_contexts_with_a_trend(dev, torch, name, M, H, d, bits, bs, shape):  # noqa: F811
    """Maxima and value scales that move after sums were taken out, and that do
    not."""
    long_check(dev, torch, name, M, H, d, bits, bs, 100000, shape, 600 if M == 1 else 160)


# ---- the gradient of large and of small rows ----------------------------------------------

@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("size,eps", [(1e14, 1e-5), (1e17, 1e-5), (1e18, 1e-5), (1e-14, 0.0),
                                      (1e-17, 0.0), (1e-3, 0.0)])
@pytest.mark.parametrize("grad", [1e-8, 1.0, 1e6])
def test_norm_rope_gradient_of_any_size(dev, torch, name, pairs, size, eps, grad):  # noqa: F811
    """Wherever the sum of squares is a float32, so is the gradient, to the bound
    that it has for rows of ordinary size (relative: nothing is added to it).  Some
    vectors of size 1e18 are past that: their 1 / rms is 0, and so is what they give."""
    n, h, k, d, _ = shape = (7, 3, 2, 128, 64)
    rng = np.random.default_rng(4)
    x, gq, gk, co, si, pos = S.norm_inputs(torch, rng, shape, name)
    x *= size
    dq = torch.from_numpy(rng.standard_normal((n, h * d)) * grad).to("cuda", x.dtype)
    dk = torch.from_numpy(rng.standard_normal((n, k * d)) * grad).to("cuda", x.dtype)
    dx = torch.full_like(x, 7.0)
    dgq, dgk = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    dev.qk_norm_rope_bwd(x, gq, gk, co, si, pos, dq, dk, dx, dgq, dgk, eps=eps, pairs=pairs)
    g = np.concatenate([np.tile(gq.cpu().numpy(), (h, 1)), np.tile(gk.cpu().numpy(), (k, 1))])
    want, mag, dg, dgm = S.norm_rope_grad64(
        S.heads64(x, n, h + k, d), g.astype(float), co.cpu().numpy().astype(float),
        si.cpu().numpy().astype(float), pos.cpu().numpy(),
        np.concatenate([S.heads64(dq, n, h, d), S.heads64(dk, n, k, d)], 1), float(np.float32(eps)),
        pairs)
    over = ((S.heads64(x, n, h + k, d) ** 2).sum(-1) > np.finfo(np.float32).max)[..., None]
    assert over.any() == (size == 1e18)
    want, mag, dg, dgm = (np.where(over, 0, t) for t in (want, mag, dg, dgm))
    assert S.within(torch, S.heads64(dx, n, h + k, d), want, 128 * S.U * mag, name).all()
    for have, part in ((dgq, slice(0, h)), (dgk, slice(h, h + k))):
        assert (np.abs(have.cpu().numpy() - dg[:, part].sum((0, 1)))
                <= 96 * S.U * dgm[:, part].sum((0, 1))).all()


# ---- equal slots ---------------------------------------------------------------------------

@pytest.mark.parametrize("bits,d", [(8, 128), (4, 256), (8, 64)])
def test_kv_move_to_equal_destinations(dev, torch, bits, d):  # noqa: F811
    """Of pairs with one destination the last that is inside the pool is kept,
    whole: codes and word."""
    kvh, bs, nb, count = 2, 7, 40, 64
    for seed in range(8):
        rng = np.random.default_rng(seed)
        cache = dev.kv_cache(nb, bs, kvh, d, bits)
        for c in cache:
            c.copy_(torch.from_numpy(rng.integers(0, 256, tuple(c.shape))).to(c.dtype))
        perm = rng.permutation(nb * bs).astype(np.int32)
        src = np.stack([perm[:count], perm[100:100 + count]])
        dst = np.stack([rng.choice(src[0][:3], count), rng.choice(perm[200:205], count)])
        src[0, -1], dst[1, -1], src[1, -2] = -1, nb * bs, 1 << 30      # skipped, though last
        want = [c.cpu().numpy().copy() for c in cache]
        old = [w.copy() for w in want]
        for w, o in zip(want, old):
            for b in range(2):
                for a, z in zip(src[b], dst[b]):
                    if 0 <= a < nb * bs and 0 <= z < nb * bs:
                        w[z // bs, :, z % bs] = o[a // bs, :, a % bs]
        dev.kv_move(torch.from_numpy(src).cuda(), torch.from_numpy(dst).cuda(), *cache, d)
        for c, w in zip(cache, want):
            assert np.array_equal(c.cpu().numpy(), w)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
def test_kv_append_to_a_slot_given_twice(dev, torch, bits, name):  # noqa: F811
    """What such a slot holds is not defined; all others hold what they would."""
    n, kvh, d, bs = 1500, 3, 128, 16
    rng = np.random.default_rng(bits)
    x = torch.from_numpy(rng.standard_normal((2, n, kvh * d))).to("cuda", S.dtype_of(torch, name))
    nb = n // bs + 3
    slot = rng.permutation(nb * bs)[:n].astype(np.int32)
    alone = dev.kv_cache(nb, bs, kvh, d, bits)
    dev.kv_append(x[0], x[1], torch.from_numpy(slot).cuda(), *alone)
    twice = slot.copy()
    twice[100:200] = slot[300:400]                  # and 100 slots get none
    twice[7] = twice[8] = twice[9] = -1
    cache = dev.kv_cache(nb, bs, kvh, d, bits)
    dev.kv_append(x[0], x[1], torch.from_numpy(twice).cuda(), *cache)
    other = np.setdiff1d(slot, np.concatenate([slot[300:400], slot[100:200], slot[7:10]]))
    none = np.setdiff1d(np.arange(nb * bs), twice)
    for c, a in zip(cache, alone):
        c, a = c.cpu().numpy(), a.cpu().numpy()
        assert np.array_equal(c[other // bs, :, other % bs], a[other // bs, :, other % bs])
        assert not c[none // bs, :, none % bs].any()


# ---- tensors and streams of another device -------------------------------------------------

def test_tensors_of_another_device_are_refused(dev, torch):  # noqa: F811
    """The mismatch is made on the host: the module is told that the library is
    on the next device, so that these tensors are the foreign ones.  Nothing is
    launched."""
    x, gq, gk, co, si, pos = S.norm_inputs(torch, np.random.default_rng(1), (4, 2, 1, 64, 64), "f32")
    q, k = torch.empty(4, 128, device="cuda"), torch.empty(4, 64, device="cuda")
    cache = dev.kv_cache(2, 16, 1, 64, 8)
    slot = torch.arange(4, dtype=torch.int32, device="cuda")
    one = torch.ones(4, 1, dtype=torch.int64, device="cuda")
    calls = [lambda: dev.qk_norm_rope(x, gq, gk, co, si, pos, q, k),
             lambda: dev.qk_norm_rope_bwd(x, gq, gk, co, si, pos, q, k, x.clone(), gq.clone(),
                                          gk.clone()),
             lambda: dev.kv_append(k, k, slot, *cache),
             lambda: dev.kv_read(slot, *cache, k, k.clone()),
             lambda: dev.kv_move(slot.view(2, 2), slot.view(2, 2), *cache, 64),
             lambda: dev.tree_attn(k, *cache, slot.view(4, 1) % 2, slot, one, k.clone(), 64)]
    for call in calls:
        call()
    device = dev._device
    try:
        dev._device = device + 1
        dev._bind()
        before = dev.launch_count()
        for call in calls:
            with pytest.raises(ValueError, match="device"):
                call()
        with pytest.raises(ValueError, match="stream"):
            dev.kv_append(k, k, slot, *cache, stream=torch.cuda.current_stream())
        assert dev.launch_count() == before
    finally:
        dev._device = device
        dev._bind()
    for call in calls:
        call()
    torch.cuda.synchronize()


# ---- one row, whatever its stride -------------------------------------------------------------

@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_one_row_of_any_stride(dev, torch, name):  # noqa: F811
    """A single row has no stride that matters: that of a transposed column is 1,
    of an expanded vector 0."""
    t = S.dtype_of(torch, name)
    h, k, d = 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)

    def odd(x, stride):
        return x.clone().as_strided((1, x.numel()), (stride, 1))

    def rows(stride):
        g.manual_seed(1)
        x = odd(torch.randn(1, (h + 2 * k) * d, device="cuda", generator=g).to(t), stride)
        gq, gk = torch.rand(2, d, device="cuda", generator=g).unbind()
        gq, gk = gq.contiguous(), gk.contiguous()
        co, si = torch.rand(2, 5, d // 2, device="cuda", generator=g).unbind()
        pos = torch.tensor([3], dtype=torch.int32, device="cuda")
        q, kk = (odd(torch.zeros(1, m * d, device="cuda", dtype=t), stride) for m in (h, k))
        dev.qk_norm_rope(x, gq, gk, co, si, pos, q, kk)
        dx = odd(torch.zeros_like(x), stride)
        dev.qk_norm_rope_bwd(x, gq, gk, co, si, pos, q, kk, dx, gq.clone(), gk.clone())
        cache = dev.kv_cache(2, 16, k, d, 8)
        slot = torch.tensor([5], dtype=torch.int32, device="cuda")
        v = odd(x[:, (h + k) * d:], stride)
        dev.kv_append(kk, v, slot, *cache)
        ko, vo = (odd(torch.zeros(1, k * d, device="cuda", dtype=t), stride) for _ in range(2))
        dev.kv_read(slot, *cache, ko, vo)
        o = odd(torch.zeros_like(q), stride)
        dev.tree_attn(q, *cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), slot,
                      torch.ones(1, 1, dtype=torch.int64, device="cuda"), o, d)
        return [x.clone() for x in (q, kk, dx, *cache, ko, vo, o)]

    want = rows(1 << 12)
    assert all(x.float().abs().sum() > 0 for x in want[-3:])
    for stride in (0, 1, 3):
        assert all(torch.equal(a, b) for a, b in zip(rows(stride), want))
