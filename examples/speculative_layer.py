"""One ternary attention layer served with drafted-token trees over a quantised
paged cache: how the serving operators of nelisp_cuda.dev go together.

    python examples/speculative_layer.py [--bits 8|4] [--steps N]

Per step a tree of drafted tokens runs through the layer at once -- the fused
Q|K|V projection (ternary GEMV), the per-head norm of queries and keys with the
rotation, the append of the nodes' keys and values behind the prefix, the tree
attention, the output projection -- then one root-to-node path is accepted and
its rows move to the end of the prefix.  The prompt goes in the same way, 64
tokens at a time as a chain.  Every step is checked against the same rows of
Q|K|V decoded one by one on a cache of their own: accepted rows hold the same
bits, and the outputs agree to rounding.
"""
import argparse
import os
import random
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "nelisp-gpu_b200"))

import torch  # noqa: E402

from nelisp_cuda import dev  # noqa: E402


class Layer:
    """The weights of one attention layer: ternary Q|K|V and O, gains, tables."""

    def __init__(self, hidden=512, heads=8, kv_heads=2, head_dim=64, max_seq=1024, seed=1):
        g = torch.Generator().manual_seed(seed)
        self.hidden, self.heads, self.kv_heads, self.head_dim = hidden, heads, kv_heads, head_dim
        self.q, self.kv = heads * head_dim, kv_heads * head_dim
        self.width = self.q + 2 * self.kv

        def ternary(out, cols):
            code = torch.tensor([0, 1, 3])[torch.randint(0, 3, (out, cols), generator=g)]
            word = sum(code[:, f::16] << (2 * f) for f in range(16))
            word = torch.where(word >= 1 << 31, word - (1 << 32), word)
            scale = (0.5 + torch.rand(out, generator=g)) / (2 * cols / 3) ** 0.5
            return word.int().cuda().contiguous(), scale.cuda()

        self.wqkv, self.sqkv = ternary(self.width, hidden)
        self.wo, self.so = ternary(hidden, self.q)
        self.gq, self.gk = (0.75 + torch.rand(2, head_dim, generator=g) / 2).cuda().unbind()
        angle = torch.arange(max_seq)[:, None] * \
            10000.0 ** (-2.0 * torch.arange(head_dim // 2, dtype=torch.float64) / head_dim)
        self.co, self.si = angle.cos().float().cuda(), angle.sin().float().cuda()

    def project(self, x):
        """Rows of Q|K|V."""
        y = torch.empty(len(x), self.width, device="cuda")
        dev.ternary_gemv(x, self.wqkv, self.sqkv, y, len(x), self.width, self.hidden)
        return y

    def output(self, ctx):
        y = torch.empty(len(ctx), self.hidden, device="cuda")
        dev.ternary_gemv(ctx, self.wo, self.so, y, len(ctx), self.hidden, self.q)
        return y


class Sequence:
    """One sequence's pages in a cache of its own, and how far they are filled."""

    def __init__(self, layer, bits, block=16, blocks=64, seed=2):
        self.layer, self.block = layer, block
        self.cache = dev.kv_cache(blocks, block, layer.kv_heads, layer.head_dim, bits)
        order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))
        self.table = order.int().cuda().view(1, -1)
        self.length = 0

    def slots(self, tokens):
        t = torch.as_tensor(tokens, device="cuda")
        return self.table[0][t // self.block] * self.block + (t % self.block).int()

    def run(self, qkv, parents):
        """The layer's outputs for the nodes of a tree (their rows of Q|K|V,
        overwritten; parents[i] < i, or -1) behind the prefix; the nodes' keys
        and values stay in the cache after it until accept()."""
        a, n = self.layer, qkv.shape[0]
        depth, mask = [], []
        for i, p in enumerate(parents):
            depth.append(depth[p] + 1 if p >= 0 else 0)
            mask.append((mask[p] if p >= 0 else 0) | 1 << i)
        pos = torch.tensor([self.length + d for d in depth], dtype=torch.int32, device="cuda")
        signed = [m - (1 << 64) if m >> 63 else m for m in mask]
        mask = torch.tensor([signed], dtype=torch.int64, device="cuda")
        length = torch.tensor([self.length], dtype=torch.int32, device="cuda")
        q, k, v = qkv[:, :a.q], qkv[:, a.q:a.q + a.kv], qkv[:, a.q + a.kv:]
        dev.qk_norm_rope(qkv, a.gq, a.gk, a.co, a.si, pos, q, k)          # in place
        dev.kv_append(k, v, self.slots(range(self.length, self.length + n)), *self.cache)
        ctx = torch.empty(n, a.q, device="cuda")
        dev.tree_attn(q, *self.cache, self.table, length, mask, ctx, a.head_dim)
        return a.output(ctx)

    def accept(self, path):
        """Keep the nodes of PATH (ascending) as the next tokens of the prefix."""
        src = self.slots([self.length + i for i in path]).view(1, -1)
        dst = self.slots([self.length + i for i in range(len(path))]).view(1, -1)
        dev.kv_move(src.contiguous(), dst.contiguous(), *self.cache, self.layer.head_dim)
        self.length += len(path)

    def rows(self):
        k, v = torch.empty(2, self.length, self.layer.kv, device="cuda").unbind()
        dev.kv_read(self.slots(range(self.length)), *self.cache, k, v)
        return k, v


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--bits", type=int, default=8, choices=(4, 8))
    ap.add_argument("--steps", type=int, default=6)
    a = ap.parse_args(argv)
    r, g = random.Random(3), torch.Generator(device="cuda").manual_seed(4)
    layer = Layer()
    drafted, plain = Sequence(layer, a.bits, seed=2), Sequence(layer, a.bits, seed=5)
    prompt = torch.randn(150, layer.hidden, device="cuda", generator=g)
    for s in (drafted, plain):
        for i in range(0, len(prompt), 64):
            part = prompt[i:i + 64]
            s.run(layer.project(part), [j - 1 for j in range(len(part))])
            s.accept(list(range(len(part))))
    worst = 0.0
    for step in range(a.steps):
        nodes = r.randint(2, 24)
        parents = [-1] + [r.randrange(max(0, i - 6), i) for i in range(1, nodes)]
        x = torch.randn(nodes, layer.hidden, device="cuda", generator=g)
        qkv = layer.project(x)
        y = drafted.run(qkv.clone(), parents)
        node, path = r.randrange(nodes), []
        while node >= 0:
            path.insert(0, node)
            node = parents[node]
        drafted.accept(path)
        for i in path:                                   # the same tokens, one by one
            one = plain.run(qkv[i:i + 1].clone(), [-1])
            plain.accept([0])
            worst = max(worst, ((one[0] - y[i]).abs().max() / y[i].abs().max()).item())
        print(f"step {step}: {nodes} nodes, accepted {len(path)}, prefix {drafted.length}")
    same = all(torch.equal(x, y) for x, y in zip(drafted.rows(), plain.rows()))
    print(f"{a.bits}-bit cache: accepted rows {'equal' if same else 'DIFFER'}, "
          f"outputs within {worst:.1e} of one token at a time")
    return same and worst < 1e-4


if __name__ == "__main__":
    sys.exit(0 if main() else 1)
