"""The cache operators of speculative serving, and the query / key norms
before them, as measured work.

Four operators, in the order in which a decoder layer meets them:

* ``norm_rope``       RMS norm of every query and key head with a gain, and the
                      position rotation, from rows of Q|K|V in one pass
* ``norm_rope_grad``  its backward pass: the gradient of the Q|K part of the
                      rows and of the two gains
* ``kv``              keys and values quantised to 8 or 4 bits as they are
                      written to a paged cache, and the same rows read back
* ``tree``            attention of a tree of drafted tokens (one token is the
                      ordinary decode step) over a prefix in that cache

``run`` computes them with elementary torch operations in 32 bits, or, where
``own`` is set, with the calls of ``nelisp_cuda.dev``.

The quantised form of a head vector x, exactly as both sides and ``exact``
form it (fl: one rounding to 32 bits):
  8 bits  s = fl(max|x| / 127), code = 128 + rint(fl(x * fl(127 / max|x|))),
          value s * (code - 128); the parameter word is s
  4 bits  lo = min x rounded down to bfloat16, s = fl(fl(max x - lo) / 15)
          rounded up to bfloat16, code = min(15, rint(fl(fl(x - lo) * fl(1 / s)))),
          value fl(s * code) + lo; the parameter word is s | lo << 16
A vector whose s is under 2^-112 has s = 0 and the codes of zero.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
TINY = 2.0 ** -112


# ---- cases ----------------------------------------------------------------

def listed():
    return [
        # one token of the decoder's own shape (20 heads of 128, f32): latency
        dict(name="norm_rope_token", op="norm_rope", type="f32", n=1, heads=20, kv_heads=20,
             dim=128, rot=128, pairs="half", padded=False),
        # the prompts of a serving batch, grouped heads, some rows of padding
        dict(name="norm_rope_prompt", op="norm_rope", type="bf16", n=8192, heads=32, kv_heads=8,
             dim=128, rot=128, pairs="half", padded=True),
        # one training sequence of the decoder's shape, an odd number of tokens
        dict(name="norm_rope_grad_seq", op="norm_rope_grad", type="f32", n=513, heads=20,
             kv_heads=20, dim=128, rot=128, pairs="half", padded=False),
        # a training batch with small heads, half of each rotated, adjacent pairs
        dict(name="norm_rope_grad_batch", op="norm_rope_grad", type="bf16", n=8191, heads=32,
             kv_heads=8, dim=64, rot=32, pairs="adjacent", padded=True),
        # the new tokens of one decode step of a batch of 8
        dict(name="kv_step_i8", op="kv", type="f32", n=8, kv_heads=20, dim=128, bits=8, block=64),
        # a batch of prompts of the decoder's shape into an 8-bit cache
        dict(name="kv_prompt_i8", op="kv", type="f32", n=4095, kv_heads=20, dim=128, bits=8,
             block=64),
        # a long prompt into a 4-bit cache with short pages
        dict(name="kv_prompt_i4", op="kv", type="bf16", n=16384, kv_heads=8, dim=128, bits=4,
             block=16),
        # a decode step of the decoder: one token, no drafts, short context
        dict(name="tree_token", op="tree", type="f32", batch=1, nodes=1, heads=20, kv_heads=20,
             dim=128, bits=8, block=64, length=640, ragged=False, chain=True),
        # a decode step of a batch at a long context, one head per key head
        dict(name="tree_batch", op="tree", type="f32", batch=8, nodes=1, heads=32, kv_heads=32,
             dim=128, bits=8, block=64, length=4096, ragged=False, chain=True),
        # small draft trees over ragged contexts in 4 bits, short pages
        dict(name="tree_draft_i4", op="tree", type="bf16", batch=16, nodes=8, heads=32,
             kv_heads=8, dim=128, bits=4, block=16, length=8192, ragged=True, chain=False),
        # one request with a very long context and a middling tree
        dict(name="tree_long", op="tree", type="bf16", batch=1, nodes=16, heads=32, kv_heads=8,
             dim=128, bits=8, block=64, length=131071, ragged=False, chain=False),
        # the widest trees over ragged contexts
        dict(name="tree_wide", op="tree", type="bf16", batch=4, nodes=64, heads=32, kv_heads=8,
             dim=128, bits=8, block=64, length=16384, ragged=True, chain=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope_grad", "kv", "tree", "tree"])
    kind = rng.choice(["f32", "bf16"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 16, 20])
    group = rng.choice([1, 1, 2, 3, 4, 8])
    heads = kv_heads * group
    if op in ("norm_rope", "norm_rope_grad"):
        n = _log_int(rng, 1, max(1, 8192 * 40 * 128 // ((heads + kv_heads) * dim)))
        return dict(op=op, type=kind, n=n, heads=heads, kv_heads=kv_heads, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2]), pairs=rng.choice(["half", "adjacent"]),
                    padded=rng.random() < 0.5)
    bits, block = rng.choice([8, 4]), rng.choice([16, 32, 48, 64, 256])
    if op == "kv":
        n = _log_int(rng, 1, max(1, 4096 * 20 * 128 // (kv_heads * dim)))
        return dict(op=op, type=kind, n=n, kv_heads=kv_heads, dim=dim, bits=bits, block=block)
    nodes = rng.choice([1, 1, 2, 4, 5, 7, 8, 16, 24, 33, 64])
    batch = rng.choice([1, 2, 3, 5, 8, 16])
    most = min(131072, (1 << 27) // (batch * kv_heads * dim),
               7_500_000_000 // (batch * nodes * heads * dim))
    return dict(op=op, type=kind, batch=batch, nodes=nodes, heads=heads, kv_heads=kv_heads,
                dim=dim, bits=bits, block=block, length=_log_int(rng, 1, max(1, most)),
                ragged=batch > 1 and rng.random() < 0.5, chain=rng.random() < 0.3)


def _lengths(c):
    """The prefix lengths of a case: all of them `length`, or spread over
    0..length, one of them empty where there are more than two."""
    if not c["ragged"]:
        return [c["length"]] * c["batch"]
    n = [max(1, int(c["length"] * ((0.618034 * b) % 1.0))) for b in range(c["batch"])]
    n[0] = c["length"]
    if c["batch"] > 2:
        n[-1] = 0
    return n


def work(c):
    es = 4 if c["type"] == "f32" else 2
    if c["op"] in ("norm_rope", "norm_rope_grad"):
        vectors = c["n"] * (c["heads"] + c["kv_heads"])
        streams = 2 if c["op"] == "norm_rope" else 3
        table = c["n"] * c["rot"] * 4 + c["n"] * 4
        return {"bytes": streams * vectors * c["dim"] * es + table + 16 * c["dim"],
                "flops": (8 if c["op"] == "norm_rope" else 20) * vectors * c["dim"]}
    held = c["dim"] * c["bits"] // 8 + 4
    if c["op"] == "kv":
        vectors = 2 * c["n"] * c["kv_heads"]
        return {"bytes": vectors * (2 * c["dim"] * es + 2 * held) + 8 * c["n"],
                "flops": 6 * vectors * c["dim"]}
    keys = sum(n + c["nodes"] for n in _lengths(c))
    rows = c["batch"] * c["nodes"] * c["heads"]
    return {"bytes": 2 * keys * c["kv_heads"] * held + 2 * rows * c["dim"] * es + 4 * rows,
            "flops": 4 * keys * c["nodes"] * c["heads"] * c["dim"]}


# ---- inputs -----------------------------------------------------------------

def _rope(rows, rot):
    half = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] \
        * 10000.0 ** (-2.0 * half / rot)
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def _store(x, bits):
    """Codes and parameter words of head vectors x [..., dim] in a cache."""
    code, s, lo = _quantise(x, bits)
    if bits == 8:
        return code, s.view(torch.int32)
    code = code[..., 0::2] | (code[..., 1::2] << 4)
    word = (s.view(torch.int32) >> 16 & 0xFFFF) | (lo.view(torch.int32) & -65536)
    return code.contiguous(), word


def _pool(c, blocks, g):
    """A paged cache whose every row holds a quantised random vector; the keys
    have a few channels several times the others, as trained ones do."""
    got = []
    for is_key in (True, False):
        x = torch.randn(blocks, c["kv_heads"], c["block"], c["dim"], device="cuda", generator=g)
        if is_key:
            x *= torch.where(torch.rand(c["dim"], device="cuda", generator=g) < 0.05, 4.0, 1.0)
        got += list(_store(x, c["bits"]))
        del x
    return got


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = random.Random(seed)
    t = TYPES[c["type"]]
    s = dict(c)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if c["op"] in ("norm_rope", "norm_rope_grad"):
        n, h, k, d = c["n"], c["heads"], c["kv_heads"], c["dim"]
        rows = max(1024, n)
        s["x"] = (normal(n, (h + 2 * k) * d) * (0.5 + 2 * torch.rand(n, 1, device="cuda",
                                                                    generator=g))).to(t)
        s["gq"], s["gk"] = (0.75 + 0.5 * torch.rand(2, d, device="cuda", generator=g)).unbind()
        s["co"], s["si"] = _rope(rows, c["rot"])
        pos = torch.randint(0, rows, (n,), device="cuda", generator=g, dtype=torch.int32)
        if c["padded"]:   # rows that hold no token
            pos[torch.rand(n, device="cuda", generator=g) < 0.05] = -1
        s["pos"] = pos
        if c["op"] == "norm_rope":
            s["q"] = torch.empty(n, h * d, device="cuda", dtype=t)
            s["k"] = torch.empty(n, k * d, device="cuda", dtype=t)
        else:
            s["dq"], s["dk"] = normal(n, h * d).to(t), normal(n, k * d).to(t)
            s["dx"] = torch.empty_like(s["x"])
            s["dgq"], s["dgk"] = torch.empty(2, d, device="cuda").unbind()
        return s
    if c["op"] == "kv":
        n, k, d = c["n"], c["kv_heads"], c["dim"]
        x = normal(n, 2 * k * d)   # the K|V part of the rows
        x[:, :k * d] *= torch.where(torch.rand(k * d, device="cuda", generator=g) < 0.05, 4.0, 1.0)
        x = x.to(t)
        s["x"], s["k"], s["v"] = x, x[:, :k * d], x[:, k * d:]
        blocks = -(-n // c["block"]) + 3
        order = torch.randperm(blocks, device="cuda", generator=g, dtype=torch.int32)
        at = torch.arange(n, device="cuda", dtype=torch.int32)
        s["slot"] = (order[(at // c["block"]).long()] * c["block"] + at % c["block"]).contiguous()
        held = d * c["bits"] // 8
        for name in ("kc", "vc"):
            s[name] = torch.zeros(blocks, k, c["block"], held, device="cuda", dtype=torch.uint8)
        for name in ("kp", "vp"):
            s[name] = torch.zeros(blocks, k, c["block"], device="cuda", dtype=torch.int32)
        s["ko"], s["vo"] = torch.empty(2, n, k * d, device="cuda", dtype=t).unbind()
        return s
    lengths = _lengths(c)
    r.shuffle(lengths)
    b, m = c["batch"], c["nodes"]
    per = -(-(max(lengths) + m) // c["block"])
    blocks = b * per + 2
    s["kc"], s["kp"], s["vc"], s["vp"] = _pool(c, blocks, g)
    order = torch.randperm(blocks, device="cuda", generator=g, dtype=torch.int32)
    s["table"] = order[:b * per].view(b, per).contiguous()
    s["len"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    words = []
    for i in range(b):
        used = m if not c["ragged"] or i == 0 else r.randint(1, m)
        row = []
        for j in range(m):
            up = 0 if j == 0 else row[j - 1 if c["chain"] else r.randrange(max(0, j - 8), j)]
            row.append(up | 1 << j)
        words.append([w - (1 << 64) if w >> 63 else w for w in row[:used]] + [0] * (m - used))
    s["mask"] = torch.tensor(words, device="cuda", dtype=torch.int64)
    width = c["heads"] * c["dim"]
    s["x"] = normal(b * m, width + 2 * c["kv_heads"] * c["dim"]).to(t)
    s["q"] = s["x"][:, :width]
    s["o"] = torch.empty(b * m, width, device="cuda", dtype=t)
    s["lse"] = torch.empty(b * m, c["heads"], device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------

def _bf16_down(x):
    """x rounded towards minus infinity to bfloat16, in 32 bits."""
    w = x.view(torch.int32)
    cut = w & -65536
    return torch.where((x < 0) & (cut != w), cut + 65536, cut).view(torch.float32)


def _quantise(x, bits):
    x = x.float()
    if bits == 8:
        most = x.abs().amax(-1)
        full = torch.full((), 127.0, device=x.device)
        some = most >= TINY * 127
        s = torch.where(some, most / full, 0.0)
        inverse = torch.where(some, torch.div(full, most), 0.0)
        return (torch.round(x * inverse[..., None]) + 128).to(torch.uint8), s, None
    low, high = _bf16_down(x.amin(-1)), x.amax(-1)
    s = -_bf16_down(-((high - low) / torch.full((), 15.0, device=x.device)))
    some = s >= TINY
    s = torch.where(some, s, 0.0)
    inverse = torch.where(some, torch.ones_like(s) / s, 0.0)
    code = torch.round((x - low[..., None]) * inverse[..., None]).clamp(max=15)
    return code.to(torch.uint8), s, low


def _value(code, word, bits):
    """The values that codes [..., bytes] with parameter words [...] stand for."""
    if bits == 8:
        return word.view(torch.float32)[..., None] * (code.float() - 128)
    code = torch.stack((code & 15, code >> 4), -1).flatten(-2).float()
    s, low = (word << 16).view(torch.float32), (word & -65536).view(torch.float32)
    return s[..., None] * code + low[..., None]


def _rotate(y, co, si, rot, pairs, back=False):
    a, b = (y[..., :rot // 2], y[..., rot // 2:rot]) if pairs == "half" \
        else (y[..., 0:rot:2], y[..., 1:rot:2])
    si = -si if back else si
    a, b = a * co - b * si, a * si + b * co
    turned = torch.cat((a, b), -1) if pairs == "half" else torch.stack((a, b), -1).flatten(-2)
    return torch.cat((turned, y[..., rot:]), -1)


def _plain_norm_rope(s):
    n, h, k, d = s["n"], s["heads"], s["kv_heads"], s["dim"]
    x = s["x"][:, :(h + k) * d].float().view(n, h + k, d)
    gain = torch.cat((s["gq"].expand(h, d), s["gk"].expand(k, d)))
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    real = (s["pos"] >= 0)[:, None, None]
    at = s["pos"].clamp(min=0).long()
    co, si = s["co"][at][:, None], s["si"][at][:, None]
    if s["op"] == "norm_rope":
        y = torch.where(real, _rotate(x * r * gain, co, si, s["rot"], s["pairs"]), 0.0)
        y = y.reshape(n, -1).to(TYPES[s["type"]])
        return y[:, :h * d], y[:, h * d:]
    dy = torch.cat((s["dq"], s["dk"]), 1).float().view(n, h + k, d)
    u = torch.where(real, _rotate(dy, co, si, s["rot"], s["pairs"], back=True), 0.0)
    xn, w = x * r, u * gain
    dx = r * (w - xn * (w * xn).mean(-1, keepdim=True))
    dg = u * xn
    return (dx.reshape(n, -1).to(TYPES[s["type"]]), dg[:, :h].sum((0, 1)), dg[:, h:].sum((0, 1)))


def _held(x, s):
    code, word = _store(x.reshape(s["n"], s["kv_heads"], s["dim"]), s["bits"])
    return _value(code, word, s["bits"]).reshape(s["n"], -1).to(TYPES[s["type"]])


def _plain_kv(s):
    return _held(s["k"], s), _held(s["v"], s)


def _plain_tree(s):
    b, m, h, k, d = s["batch"], s["nodes"], s["heads"], s["kv_heads"], s["dim"]
    n = s["table"].shape[1] * s["block"]
    at = torch.arange(n, device="cuda")
    page = s["table"].long()[:, at // s["block"]]
    off = (at % s["block"]).expand(b, n)
    keys, values = (_value(s[codes][page, :, off], s[words][page, :, off], s["bits"])
                    .transpose(1, 2) for codes, words in (("kc", "kp"), ("vc", "vp")))
    node = at[None, :] - s["len"][:, None]              # [b, n], below 0: the prefix
    bit = s["mask"][:, :, None] >> node.clamp(0, 63)[:, None, :] & 1
    seen = torch.where(node[:, None, :] < 0, s["mask"][:, :, None] != 0,
                       (node < m)[:, None, :] & (bit != 0))                     # [b, m, n]
    q = s["q"].float().reshape(b, m, k, h // k, d).permute(0, 2, 3, 1, 4).reshape(b, k, -1, d)
    score = (q @ keys.transpose(-1, -2) * d ** -0.5).view(b, k, h // k, m, n)
    score = torch.where(seen[:, None, None], score, -math.inf)
    most = score.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(score - most)
    z = e.sum(-1, keepdim=True)
    o = (e.view(b, k, -1, n) @ values).view(b, k, h // k, m, d) / torch.where(z > 0, z, 1.0)
    lse = torch.where(z > 0, most + torch.log(z), -math.inf)[..., 0]
    o = o.permute(0, 3, 1, 2, 4).reshape(b * m, h * d).to(TYPES[s["type"]])
    return o, lse.permute(0, 3, 1, 2).reshape(b * m, h)


# ---- the framework's calls -----------------------------------------------------

def _dev():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "nelisp-gpu_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    from nelisp_cuda import dev
    return dev


def _own_norm_rope(s, dev):
    args = (s["x"], s["gq"], s["gk"], s["co"], s["si"], s["pos"])
    if s["op"] == "norm_rope":
        dev.qk_norm_rope(*args, s["q"], s["k"], eps=1e-5, pairs=s["pairs"])
        return s["q"], s["k"]
    dev.qk_norm_rope_bwd(*args, s["dq"], s["dk"], s["dx"], s["dgq"], s["dgk"], eps=1e-5,
                         pairs=s["pairs"])
    return s["dx"][:, :(s["heads"] + s["kv_heads"]) * s["dim"]], s["dgq"], s["dgk"]


def _own_kv(s, dev):
    dev.kv_append(s["k"], s["v"], s["slot"], s["kc"], s["kp"], s["vc"], s["vp"])
    dev.kv_read(s["slot"], s["kc"], s["kp"], s["vc"], s["vp"], s["ko"], s["vo"])
    return s["ko"], s["vo"]


def _own_tree(s, dev):
    dev.tree_attn(s["q"], s["kc"], s["kp"], s["vc"], s["vp"], s["table"], s["len"], s["mask"],
                  s["o"], s["dim"], lse=s["lse"])
    return s["o"], s["lse"]


def run(s):
    if own:
        return {"kv": _own_kv, "tree": _own_tree}.get(s["op"], _own_norm_rope)(s, _dev())
    return {"kv": _plain_kv, "tree": _plain_tree}.get(s["op"], _plain_norm_rope)(s)


# ---- 64 bits ---------------------------------------------------------------------

def _exact_norm_rope(s):
    h, k, d, rot = s["heads"], s["kv_heads"], s["dim"], s["rot"]
    pos = s["pos"].long()
    real = torch.nonzero(pos >= 0)[:, 0]
    half = torch.arange(rot // 2, device="cuda")
    first, second = (half, half + rot // 2) if s["pairs"] == "half" else (2 * half, 2 * half + 1)
    co, si = s["co"].double()[pos[real]], s["si"].double()[pos[real]]
    rows, gains = [], []
    for head in range(h + k):
        g = (s["gq"] if head < h else s["gk"]).double()
        x = s["x"][real, head * d:(head + 1) * d].double()
        norm = 1.0 / torch.sqrt((x ** 2).sum(1, keepdim=True) / d + float(torch.tensor(1e-5)))
        out = torch.zeros(s["n"], d, device="cuda", dtype=torch.float64)
        if s["op"] == "norm_rope":
            y = x * norm * g
            z = y.clone()
            z[:, first] = y[:, first] * co - y[:, second] * si
            z[:, second] = y[:, first] * si + y[:, second] * co
            out[real] = z
        else:
            dz = (s["dq"][real, head * d:(head + 1) * d] if head < h else
                  s["dk"][real, (head - h) * d:(head - h + 1) * d]).double()
            dy = dz.clone()
            dy[:, first] = dz[:, first] * co + dz[:, second] * si
            dy[:, second] = dz[:, second] * co - dz[:, first] * si
            gains.append((dy * x * norm).sum(0))
            dot = (dy * g * x).sum(1, keepdim=True)
            out[real] = norm * dy * g - x * norm ** 3 * dot / d
        rows.append(out)
    if s["op"] == "norm_rope":
        return torch.cat(rows[:h], 1), torch.cat(rows[h:], 1)
    return torch.cat(rows, 1), torch.stack(gains[:h]).sum(0), torch.stack(gains[h:]).sum(0)


def _f32(x):
    return x.float().double()


def _bf16_toward(x, up):
    """The bfloat16 at or above (below) x, from the nearest one."""
    near = x.float().bfloat16()
    w = near.view(torch.int16).int()
    step = torch.where((w < 0) == up, -1, 1)   # to a larger, or a smaller magnitude
    other = (w + step).to(torch.int16).view(torch.bfloat16)
    wrong = near.double() < x if up else near.double() > x
    return torch.where(wrong & (near != 0), other, near).double()


def _exact_kv(s):
    got = []
    for x in (s["k"], s["v"]):
        x = x.reshape(-1, s["dim"]).double()
        if s["bits"] == 8:
            most = x.abs().max(1, keepdim=True).values
            full = torch.full_like(most, 127.0)
            y = _f32(most / full) * torch.round(_f32(x * _f32(full / most)))
        else:
            low = _bf16_toward(x.min(1, keepdim=True).values, False)
            span = _f32(x.max(1, keepdim=True).values - low)
            step = _bf16_toward(_f32(span / torch.full_like(span, 15.0)), True)
            code = torch.round(_f32(_f32(x - low) * _f32(torch.ones_like(step) / step)))
            y = _f32(step * torch.clamp(code, max=15.0) + low)
        got.append(y.view(s["n"], -1))
    return tuple(got)


def _exact_tree(s):
    m, h, k, d = s["nodes"], s["heads"], s["kv_heads"], s["dim"]
    group, block = h // k, s["block"]
    o = torch.zeros(s["batch"] * m, h, d, device="cuda", dtype=torch.float64)
    lse = torch.full((s["batch"] * m, h), -math.inf, device="cuda", dtype=torch.float64)

    def held(codes, words, page, off, head):
        c, w = s[codes][page, head, off], s[words][page, head, off]
        if s["bits"] == 8:
            return (c.double() - 128.0) * w.view(torch.float32).double()[:, None]
        pair = w.view(torch.bfloat16).view(-1, 2).double()
        x = torch.empty(c.shape[0], d, device="cuda", dtype=torch.float64)
        x[:, 0::2], x[:, 1::2] = (c % 16).double(), (c // 16).double()
        return x * pair[:, :1] + pair[:, 1:]

    for i, length in enumerate(s["len"].tolist()):
        at = torch.arange(length + m, device="cuda")
        page, off = s["table"][i].long()[at // block], at % block
        for head in range(k):
            key, value = held("kc", "kp", page, off, head), held("vc", "vp", page, off, head)
            for j, word in enumerate(s["mask"][i].tolist()):
                if not word:
                    continue
                sees = [t for t in range(m) if word >> t & 1]
                row, hs = i * m + j, slice(head * group, (head + 1) * group)
                q = s["q"][row].view(h, d)[hs].double()
                score = q @ key.T / math.sqrt(d)
                hide = torch.ones(length + m, device="cuda", dtype=torch.bool)
                hide[:length] = False
                hide[[length + t for t in sees]] = False
                score[:, hide] = -math.inf
                lse[row, hs] = torch.logsumexp(score, 1)
                o[row, hs] = torch.exp(score - lse[row, hs][:, None]) @ value
    return o.view(-1, h * d), lse


def exact(c, seed):
    s = prepare(c, seed)
    return {"kv": _exact_kv, "tree": _exact_tree}.get(s["op"], _exact_norm_rope)(s)
