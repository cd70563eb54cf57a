"""The verification example as a whole: nodes of drafted trees against plain torch in fp32 on the dequantised weights,
path by path, and the cache after the accepted paths against one that took them token by token."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def example(cuda):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import verify_step

    return verify_step


def plain_hidden(model, ids, adapter):
    """One sequence's hidden states in fp32 on the dequantised weights, no cache."""
    c = model.c
    f8 = torch.float8_e4m3fn
    n = len(ids)

    def w(x):
        return x.codes.view(f8).float() * x.scale[:, None]

    def norm(x, g):
        return x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6) * g.float()

    angle = torch.arange(n, device="cuda").double()[:, None] * model.inv_freq.double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def turn(x):  # [heads, tokens, dim]
        u, v = x.chunk(2, -1)
        return torch.cat((u * cos - v * sin, v * cos + u * sin), -1)

    r = model.embed[ids].float()
    for i, b in enumerate(model.blocks):
        h = norm(r, b.pre[0])
        qkv = h @ w(b.qkv).T
        if adapter >= 0:
            qkv = qkv + model.scales[adapter] * (h @ b.lora_a[adapter].float().T) @ b.lora_b[adapter].float().T
        q, k, v = qkv.view(n, -1, c.head_dim).transpose(0, 1).split((c.heads, c.kv_heads, c.kv_heads))
        q, k = turn(q), turn(k)
        k, v = (t.repeat_interleave(c.heads // c.kv_heads, 0) for t in (k, v))
        s = c.cap * torch.tanh((q @ k.transpose(1, 2)) / c.head_dim ** 0.5 / c.cap)
        s = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), float("-inf"))
        a = (s.softmax(-1) @ v).transpose(0, 1).reshape(n, -1)
        r = r + b.gate[0].float() * norm(a @ w(b.out).T, b.post[0])
        h = norm(r, b.pre[1])
        r = r + b.gate[1].float() * norm(torch.nn.functional.silu(h @ w(b.up).T) @ w(b.down).T, b.post[1])
    return norm(r, model.last)


def prompts_in(example, model, prompts, adapter_of):
    cache = example.PagedCache(model.c, len(prompts))
    ids, offsets = example.packed(prompts)
    cache.lens += torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda")
    adapters = torch.tensor([x for x, p in zip(adapter_of, prompts) for _ in p], dtype=torch.int32, device="cuda")
    model.forward(ids, adapters, cache, offsets)
    return cache


def test_nodes_against_plain_torch(example):
    """What remains are the roundings to 8 bits (2^-4 of each activation in four products a layer, of each key and value),
    averaged over the sums: within an eighth of a state's norm, as in the decode example."""
    model = example.Model(example.Config(layers=1), seed=2)
    prompts, adapter_of = [[3, 1, 4], list(range(50, 120)), list(range(9, 30))], [1, -1, 0]
    cache = prompts_in(example, model, prompts, adapter_of)
    g = torch.Generator().manual_seed(4)
    trees = [example.draft(g, n, model.c.vocab, 5 + n) for n in (1, 40, 9)]
    h, kept, _ = example.verify(model, cache, [t[0] for t in trees], [t[1] for t in trees], adapter_of)
    at = 0
    for p, a, (tokens, parents) in zip(prompts, adapter_of, trees):
        for i in range(0, len(tokens), 3):
            path, x = [], i
            while x >= 0:
                path.append(tokens[x])
                x = parents[x]
            ref = plain_hidden(model, torch.tensor(p + path[::-1], device="cuda"), a)[-1]
            assert float((h[at + i].float() - ref).norm() / ref.norm()) < 0.125
        at += len(tokens)


def test_accepted_paths_stay_in_the_cache(example):
    """Drafts that follow the model's own choices are accepted as a whole, and the cache then holds what token-by-token
    steps would have left in it, up to the 8-bit rounding under a page's scale (2^-4, doubled: a page may have had a
    larger scale for a draft)."""
    model = example.Model(example.Config(layers=1), seed=3)
    prompts, adapter_of = [[3, 1, 4], list(range(50, 83))], [2, 1]
    cache = prompts_in(example, model, prompts, adapter_of)
    plain = prompts_in(example, model, prompts, adapter_of)
    adapters = torch.tensor(adapter_of, dtype=torch.int32, device="cuda")
    now = torch.tensor([7, 8], device="cuda")
    chain = [now.tolist()]
    for _ in range(3):
        plain.lens += 1
        now = model.choices(model.forward(now, adapters, plain, None))[0].long()
        chain.append(now.tolist())
    plain.lens += 1
    model.forward(now, adapters, plain, None)
    # the chain with a wrong sibling before each of its tokens
    drafts, parents = [], []
    for b in range(2):
        t, p, last = [chain[0][b]], [-1], 0
        for step in chain[1:]:
            t += [(step[b] + 1) % model.c.vocab, step[b]]
            p += [last, last]
            last = len(t) - 1
        drafts.append(t)
        parents.append(p)
    h, kept, _ = example.verify(model, cache, drafts, parents, adapter_of)
    # the two ways differ by the cache's rounding, so that a near tie may go the other way: then the path ends there
    logprobs = torch.log_softmax(model.head(h, "row").float(), 1)
    for b in range(2):
        full = [0, 2, 4, 6]
        assert kept[b] == full[: len(kept[b])]
        if len(kept[b]) < 4:
            at = logprobs[b * 7 + kept[b][-1]]
            assert float(at.max() - at[chain[len(kept[b])][b]]) < 0.25
    assert cache.lens.tolist() == [len(p) + len(k) for p, k in zip(prompts, kept)]
    f8 = torch.float8_e4m3fn
    for mine, other, s_mine, s_other in ((cache.k, plain.k, cache.k_scale, plain.k_scale), (cache.v, plain.v, cache.v_scale, plain.v_scale)):
        a = mine[0].view(f8).float() * s_mine[0][..., None, None]
        b = other[0].view(f8).float() * s_other[0][..., None, None]
        for q, n in enumerate(cache.lens.tolist()):
            for j in range(n):
                page = int(cache.table[q, j // model.c.page])
                x, y = a[page, :, j % model.c.page], b[page, :, j % model.c.page]
                assert float((x - y).norm() / y.norm()) < 0.125


def test_main_runs(example, monkeypatch):
    monkeypatch.setattr(sys, "argv", ["verify_step.py", "--layers", "1", "--nodes", "5"])
    example.main()
