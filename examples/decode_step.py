"""Decode with FP8 weights, end to end: a small mixture-of-experts decoder with
random weights generates a few tokens for a batch of prompts of different
lengths, and every step runs through the library's operators:

    q, k, v   FP8 GEMM (imma_fp8_gemm, native FP8 path)
    cache     kv_append: the step's keys and values into a paged 8-bit cache
    attention kv_attention over that cache (prompts: all tokens at once, ragged)
    output    FP8 GEMM
    experts   moe_forward (prompt tokens go through it 64 at a time)
    logits    FP8 GEMM, whose default output is column-major
    choice    token_logprobs: the best alternative is taken, its log probability
              and the distribution's entropy are reported

Run: python examples/decode_step.py [--layers 2] [--steps 8]
"""
from __future__ import annotations

import argparse
import os
import sys
from dataclasses import dataclass

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-fp8-ampere_b200"))

import torch

import fp8imma_b200

ops = fp8imma_b200.ext()


@dataclass
class Config:
    layers: int = 2
    hidden: int = 512
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    experts: int = 8
    top_k: int = 2
    inter: int = 384
    vocab: int = 4096
    page: int = 16
    max_len: int = 256
    dtype: torch.dtype = torch.bfloat16


class Fp8Weight:
    """A [N, K] weight as FP8 bytes with one scale a row."""

    def __init__(self, w: torch.Tensor):
        self.codes, self.scale, _ = ops.quantize_weights(w.contiguous(), "e4m3")

    def __call__(self, x: torch.Tensor, layout: str = "row") -> torch.Tensor:
        out = "float16" if x.dtype == torch.float16 else "bfloat16"
        return ops.imma_fp8_gemm(x.contiguous(), self.codes, col_scales_f32=self.scale, path="fp8", out_dtype=out, out_layout=layout)[0]


class Layer:
    def __init__(self, c: Config, g: torch.Generator):
        def w(n, k):
            return torch.randn(n, k, generator=g, device="cuda") / k ** 0.5

        self.c = c
        self.qkv = Fp8Weight(w((c.heads + 2 * c.kv_heads) * c.head_dim, c.hidden))
        self.out = Fp8Weight(w(c.hidden, c.heads * c.head_dim))
        self.router = w(c.experts, c.hidden).to(c.dtype)
        self.up = Fp8Weight(w(c.experts * 2 * c.inter, c.hidden))
        self.down = Fp8Weight(w(c.experts * c.hidden, c.inter))

    def experts(self, x: torch.Tensor) -> torch.Tensor:
        c = self.c
        up, down = self.up.codes.view(c.experts, 2 * c.inter, c.hidden), self.down.codes.view(c.experts, c.hidden, c.inter)
        parts = [ops.moe_forward(t, self.router, up, self.up.scale, down, self.down.scale, c.top_k)[0] for t in x.split(64)]
        return parts[0] if len(parts) == 1 else torch.cat(parts)


class PagedCache:
    """One pool of pages a layer; a sequence takes its pages as it grows."""

    def __init__(self, c: Config, batch: int):
        width = -(-c.max_len // c.page)
        pages = batch * width
        shape = (pages, c.kv_heads, c.page, c.head_dim)
        self.k = [torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(c.layers)]
        self.v = [torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(c.layers)]
        self.k_scale = [torch.zeros(pages, c.kv_heads, device="cuda") for _ in range(c.layers)]
        self.v_scale = [torch.zeros(pages, c.kv_heads, device="cuda") for _ in range(c.layers)]
        # pages in no order, as an allocator that has served others would hand them out
        self.table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).view(batch, width).to(torch.int32).cuda()
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")


class Decoder:
    def __init__(self, c: Config, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.c = c
        self.embed = torch.randn(c.vocab, c.hidden, generator=g, device="cuda").to(c.dtype)
        self.blocks = [Layer(c, g) for _ in range(c.layers)]
        self.head = Fp8Weight(3.0 * torch.randn(c.vocab, c.hidden, generator=g, device="cuda") / c.hidden ** 0.5)

    def forward(self, ids: torch.Tensor, cache: PagedCache, offsets: torch.Tensor | None) -> torch.Tensor:
        """ids: the step's packed tokens; offsets: where each sequence's begin (None: one token each).
        cache.lens already counts them. Returns hidden states [tokens, hidden]."""
        c = self.c
        x = self.embed[ids]
        for i, b in enumerate(self.blocks):
            h = torch.nn.functional.rms_norm(x, (c.hidden,))
            qkv = b.qkv(h).view(-1, c.heads + 2 * c.kv_heads, c.head_dim)
            q, k, v = qkv.split((c.heads, c.kv_heads, c.kv_heads), 1)
            where = (cache.k[i], cache.v[i], cache.k_scale[i], cache.v_scale[i], cache.table, cache.lens, offsets)
            ops.kv_append(k, v, *where)
            a, _ = ops.kv_attention(q, *where)
            x = x + b.out(a.view(-1, c.heads * c.head_dim))
            x = x + b.experts(torch.nn.functional.rms_norm(x, (c.hidden,)))
        return torch.nn.functional.rms_norm(x, (c.hidden,))

    def score(self, h: torch.Tensor, top: int = 4):
        """Log probability and entropy of the best token of each row, and the alternatives."""
        logits = self.head(h, "col").t()  # [tokens, vocab], tokens contiguous
        best = torch.empty(h.shape[0], dtype=torch.int32, device="cuda").fill_(-1)
        _, entropy, ids, logprobs = ops.token_logprobs(logits, best, top=top)
        return entropy, ids, logprobs

    def generate(self, prompts: list[list[int]], steps: int):
        c = self.c
        cache = PagedCache(c, len(prompts))
        sizes = [len(p) for p in prompts]
        offsets = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).cuda()
        ids = torch.tensor([t for p in prompts for t in p], device="cuda")
        cache.lens += torch.tensor(sizes, dtype=torch.int32, device="cuda")
        h = self.forward(ids, cache, offsets)[offsets[1:].long() - 1]  # the prompts' last tokens
        out = []
        for _ in range(steps):
            entropy, ids, logprobs = self.score(h)
            out.append((ids[:, 0], logprobs[:, 0], entropy))
            cache.lens += 1
            h = self.forward(ids[:, 0].long(), cache, None)
        return [torch.stack(x, 1) for x in zip(*out)]


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    model = Decoder(Config(layers=a.layers))
    prompts = [[1, 2, 3], list(range(10, 47)), [5], list(range(100, 180))]
    ids, logprobs, entropy = model.generate(prompts, a.steps)
    torch.cuda.synchronize()
    for i, p in enumerate(prompts):
        print("prompt of %d tokens -> %s" % (len(p), ids[i].tolist()))
        print("  log probabilities %s" % ["%.3f" % v for v in logprobs[i].tolist()])
        print("  entropies         %s" % ["%.3f" % v for v in entropy[i].tolist()])


if __name__ == "__main__":
    main()
