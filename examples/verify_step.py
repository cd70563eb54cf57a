"""Verification of drafted trees with FP8 weights and an adapter a request: a small
decoder with random weights takes prompts of several requests, then a tree of
drafted tokens for each, and scores all nodes of all trees in one step:

    norms       residual_norm: the block's result normed, gated and added to the
                residual (kept in fp32), and the next block's norm, in one pass
    q, k, v     FP8 GEMM, whose default output is column-major, and beside it
                lora_add: each request's own low-rank adapter
    cache       kv_append_rope: queries and keys turned by the nodes' positions
                (siblings share one), keys and values into the paged 8-bit cache
    attention   kv_attention_tree: a node sees the cache and its ancestors,
                scores are capped
    output, feed-forward, logits   FP8 GEMMs
    choice      token_logprobs; the longest path whose drafts are the model's own
                choices is accepted, and its tokens are appended anew at their places

Run: python examples/verify_step.py [--layers 2] [--nodes 12]
"""
from __future__ import annotations

import argparse
import os
import sys
from dataclasses import dataclass

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-fp8-ampere_b200"))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import torch

import fp8imma_b200
from decode_step import Fp8Weight, PagedCache

ops = fp8imma_b200.ext()


@dataclass
class Config:
    layers: int = 2
    hidden: int = 512
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    inter: int = 768
    vocab: int = 2048
    page: int = 16
    max_len: int = 256
    adapters: int = 3
    rank: int = 16
    cap: float = 30.0
    dtype: torch.dtype = torch.bfloat16


def tree_bits(parents: list[int], words: int) -> torch.Tensor:
    """[nodes, words] int32: each node's ancestors and itself; parents come before their children, -1: a root."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    out = torch.tensor([[r >> 32 * w & 0xFFFFFFFF for w in range(words)] for r in rows], dtype=torch.int64)
    return torch.where(out >= 2 ** 31, out - 2 ** 32, out).to(torch.int32)


class Layer:
    def __init__(self, c: Config, g: torch.Generator):
        def w(n, k):
            return torch.randn(n, k, generator=g, device="cuda") / k ** 0.5

        def near_one():
            return (1 + 0.1 * torch.randn(c.hidden, generator=g, device="cuda")).to(c.dtype)

        self.width = (c.heads + 2 * c.kv_heads) * c.head_dim
        self.qkv = Fp8Weight(w(self.width, c.hidden))
        self.out = Fp8Weight(w(c.hidden, c.heads * c.head_dim))
        self.up, self.down = Fp8Weight(w(c.inter, c.hidden)), Fp8Weight(w(c.hidden, c.inter))
        self.lora_a = torch.stack([w(c.rank, c.hidden) for _ in range(c.adapters)]).to(c.dtype)
        self.lora_b = torch.stack([w(self.width, c.rank) for _ in range(c.adapters)]).to(c.dtype)
        # norms before and after the attention and the feed-forward block
        self.pre, self.post = [near_one(), near_one()], [near_one(), near_one()]
        self.gate = [near_one(), near_one()]


class Model:
    def __init__(self, c: Config, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.c = c
        self.embed = torch.randn(c.vocab, c.hidden, generator=g, device="cuda").to(c.dtype)
        self.blocks = [Layer(c, g) for _ in range(c.layers)]
        self.last = torch.ones(c.hidden, device="cuda", dtype=c.dtype)
        self.head = Fp8Weight(4.0 * torch.randn(c.vocab, c.hidden, generator=g, device="cuda") / c.hidden ** 0.5)
        self.inv_freq = (10000.0 ** (-torch.arange(0, c.head_dim, 2, device="cuda", dtype=torch.float64) / c.head_dim)).float()
        self.scales = torch.full((c.adapters,), 0.5, device="cuda")

    def forward(self, ids, adapters, cache, offsets, tree=None, positions=None):
        """ids, adapters: the step's packed tokens and each one's adapter (-1: none); cache.lens already counts them.
        tree, positions: mask rows and places of the tokens (none: a causal step). Returns hidden states [tokens, hidden]."""
        c = self.c
        r, h = ops.residual_norm(self.embed[ids], pre_weight=self.blocks[0].pre[0], residual_out=torch.empty(len(ids), c.hidden, device="cuda"))
        for i, b in enumerate(self.blocks):
            qkv = b.qkv(h, "col").t()  # [tokens, width], tokens contiguous
            qkv = ops.lora_add(qkv, h, b.lora_a, b.lora_b, adapters, self.scales, out=qkv)
            qkv = qkv.contiguous().view(-1, c.heads + 2 * c.kv_heads, c.head_dim)
            q, k, v = qkv.split((c.heads, c.kv_heads, c.kv_heads), 1)
            where = (cache.k[i], cache.v[i], cache.k_scale[i], cache.v_scale[i], cache.table, cache.lens)
            ops.kv_append_rope(q, k, v, *where, self.inv_freq, offsets, positions, q_out=q)
            a, _ = ops.kv_attention_tree(q, *where, tree, offsets, positions if tree is not None else None, softcap=c.cap)
            r, h = ops.residual_norm(b.out(a.view(-1, c.heads * c.head_dim)), r, b.post[0], b.pre[1], b.gate[0], residual_out=r)
            y = b.down(torch.nn.functional.silu(b.up(h)))
            following = self.blocks[i + 1].pre[0] if i + 1 < len(self.blocks) else self.last
            r, h = ops.residual_norm(y, r, b.post[1], following, b.gate[1], residual_out=r)
        return h

    def choices(self, h):
        """The best token of each row and its log probability."""
        none = torch.full((h.shape[0],), -1, dtype=torch.int32, device="cuda")
        _, _, ids, logprobs = ops.token_logprobs(self.head(h, "col").t(), none, top=1)
        return ids[:, 0], logprobs[:, 0]


def packed(lists):
    offsets = torch.tensor([0] + [len(x) for x in lists]).cumsum(0).to(torch.int32).cuda()
    return torch.tensor([t for x in lists for t in x], device="cuda"), offsets


def verify(model: Model, cache: PagedCache, drafts, parents, adapter_of):
    """Scores the drafted trees (tokens and parents of each request) in one step and keeps the accepted paths:
    (hidden states of all nodes, each request's accepted nodes, the choices after each node)."""
    ids, offsets = packed(drafts)
    start = cache.lens.tolist()
    words = -(-max(len(p) for p in parents) // 32)
    tree = torch.cat([tree_bits(p, words) for p in parents]).cuda()
    place, depth = [], []
    for s, p in zip(start, parents):
        d = []
        for x in p:
            d.append(d[x] + 1 if x >= 0 else 0)
        depth.append(d)
        place += [s + x for x in d]
    positions = torch.tensor(place, dtype=torch.int32, device="cuda")
    adapters = torch.tensor([a for a, d in zip(adapter_of, drafts) for _ in d], dtype=torch.int32, device="cuda")
    cache.lens += torch.tensor([len(d) for d in drafts], dtype=torch.int32, device="cuda")
    h = model.forward(ids, adapters, cache, offsets, tree, positions)
    best = model.choices(h)[0].tolist()
    # the root of each tree is the token that the step before chose; a child is accepted when it is its parent's choice
    kept = []
    for b, (d, p) in enumerate(zip(drafts, parents)):
        at, path = 0, [0]
        base = int(offsets[b])
        while True:
            then = [i for i, x in enumerate(p) if x == at and d[i] == best[base + at]]
            if not then:
                break
            at = then[0]
            path.append(at)
        kept.append(path)
    # the cache goes back to where the step began, and the accepted paths enter it as plain steps
    cache.lens.copy_(torch.tensor([s + len(k) for s, k in zip(start, kept)], dtype=torch.int32))
    ids, offsets = packed([[d[i] for i in k] for d, k in zip(drafts, kept)])
    adapters = torch.tensor([a for a, k in zip(adapter_of, kept) for _ in k], dtype=torch.int32, device="cuda")
    model.forward(ids, adapters, cache, offsets)
    return h, kept, best


def draft(g: torch.Generator, nodes: int, vocab: int, first: int):
    """A tree of random tokens below the token `first`."""
    parents = [-1] + [int(torch.randint(max(0, i - 3), i, (1,), generator=g)) for i in range(1, nodes)]
    return [first] + torch.randint(0, vocab, (nodes - 1,), generator=g).tolist(), parents


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--nodes", type=int, default=12)
    a = ap.parse_args()
    model = Model(Config(layers=a.layers))
    prompts, adapter_of = [[1, 2, 3], list(range(10, 47)), list(range(100, 180))], [0, -1, 2]
    cache = PagedCache(model.c, len(prompts))
    ids, offsets = packed(prompts)
    cache.lens += torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda")
    adapters = torch.tensor([x for x, p in zip(adapter_of, prompts) for _ in p], dtype=torch.int32, device="cuda")
    h = model.forward(ids, adapters, cache, offsets)[offsets[1:].long() - 1]
    g = torch.Generator().manual_seed(1)
    first = model.choices(h)[0].tolist()
    trees = [draft(g, a.nodes, model.c.vocab, t) for t in first]
    _, kept, best = verify(model, cache, [t[0] for t in trees], [t[1] for t in trees], adapter_of)
    torch.cuda.synchronize()
    for i, (p, k) in enumerate(zip(prompts, kept)):
        last = i * a.nodes + k[-1]
        print("prompt of %d tokens: %d of %d drafted nodes accepted, next token %d, cache holds %d" % (len(p), len(k), a.nodes, best[last], int(cache.lens[i])))


if __name__ == "__main__":
    main()
