"""Cases and plain forms of the operators that stand between a decode step's products: the residual connection with the
norms before and after it, low-rank adapters of many requests beside a projection, the paged 8-bit cache's append with the
position rotation on the way, and attention over that cache for trees of drafted tokens with capped scores.

`run` computes an operator in its plain form (elementary torch operations in fp32) or, with `own` set, through
fp8imma_ext. `exact` gives the same values from the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
_ext = None


def _ops():
    global _ext
    if _ext is None:
        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(here, "cuda-fp8-ampere_b200"))
        import fp8imma_b200

        _ext = fp8imma_b200.ext()
    return _ext


# ------------------------------------------------------------------ cases --


def listed():
    return [
        # one token between two blocks: the residual sum and the next block's norm, where only latency counts
        {"name": "norm one token", "op": "norm", "tokens": 1, "hidden": 4096, "dtype": "bf16", "res": "bf16", "post": False, "gate": "none",
         "offset": 0.0, "alpha": 1.0, "pad": 0},
        # a decode batch of a model with a norm on both sides of each block and a learned gate, residuals kept in fp32
        {"name": "norm both sides 64", "op": "norm", "tokens": 64, "hidden": 8192, "dtype": "f16", "res": "f32", "post": True, "gate": "channel",
         "offset": 1.0, "alpha": 0.5, "pad": 0},
        # a whole prompt, a gate for each token (rows of a projection twice as wide)
        {"name": "norm prompt 8192", "op": "norm", "tokens": 8192, "hidden": 4096, "dtype": "bf16", "res": "bf16", "post": True, "gate": "token",
         "offset": 0.0, "alpha": 1.0, "pad": 4096},
        # one request with its adapter
        {"name": "lora one token", "op": "lora", "tokens": 1, "in": 4096, "out": 4096, "rank": 16, "adapters": 8, "runs": 1, "layout": "row",
         "dtype": "bf16", "base": "bf16"},
        # a decode batch of as many requests as tokens, the GEMM's default column-major result
        {"name": "lora decode 64", "op": "lora", "tokens": 64, "in": 4096, "out": 11008, "rank": 32, "adapters": 48, "runs": 64, "layout": "col",
         "dtype": "bf16", "base": "f16"},
        # ragged prompts of a few requests
        {"name": "lora prompts", "op": "lora", "tokens": 4001, "in": 8192, "out": 8192, "rank": 64, "adapters": 8, "runs": 7, "layout": "row",
         "dtype": "bf16", "base": "bf16"},
        # one new token of each of 64 sequences, far along (a window of a long stream is what the cache holds)
        {"name": "rope append 64", "op": "append", "batch": 64, "kv_len": 4000, "new": 1, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "rotary": 128, "interleaved": False, "theta": 500000.0, "at": "given", "far": 900000, "dtype": "bf16", "fmt": "e4m3"},
        # drafted trees enter the cache: nodes of one depth share a position; half of the channels turn, in neighbouring pairs
        {"name": "rope append drafts", "op": "append", "batch": 32, "kv_len": 3001, "new": 16, "heads": 28, "kv_heads": 4, "dim": 64, "page": 32,
         "rotary": 32, "interleaved": True, "theta": 10000.0, "at": "given", "far": 0, "dtype": "f16", "fmt": "e5m2"},
        # ragged prompts after a prefill, none of them a whole number of pages
        {"name": "rope append prompts", "op": "append", "batch": 6, "kv_len": 3001, "new": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "rotary": 128, "interleaved": False, "theta": 10000.0, "at": "slot", "far": 0, "dtype": "f16", "fmt": "e4m3"},
        # a small tree over one short conversation
        {"name": "tree one short", "op": "tree", "batch": 1, "kv_len": 700, "new": 8, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 0, "cap": 0.0, "dtype": "bf16", "fmt": "e4m3"},
        # a served batch, up to 16 nodes each, scores capped
        {"name": "tree batch 32", "op": "tree", "batch": 32, "kv_len": 8192, "new": 16, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 0, "cap": 50.0, "dtype": "bf16", "fmt": "e4m3"},
        # wide trees over two long documents
        {"name": "tree two long", "op": "tree", "batch": 2, "kv_len": 100001, "new": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 128,
         "window": 0, "cap": 30.0, "dtype": "f16", "fmt": "e4m3"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(("norm", "lora", "lora", "append", "tree", "tree"))
    dt, fmt = rng.choice(("f16", "bf16")), rng.choice(("e4m3", "e4m3", "e5m2"))
    if op == "norm":
        h = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            h = max(64, h // 64 * 64)
        return {"op": op, "tokens": _log(rng, 1, min(16384, 8192 * 4096 // h)), "hidden": h, "dtype": dt, "res": rng.choice(("none", "f32", dt, dt)),
                "post": rng.random() < 0.5, "gate": rng.choice(("none", "channel", "token")), "offset": rng.choice((0.0, 1.0)),
                "alpha": rng.choice((1.0, 0.5, 0.22)), "pad": rng.choice((0, 0, 8, 64))}
    if op == "lora":
        t = _log(rng, 1, 4001)
        return {"op": op, "tokens": t, "in": 8 * _log(rng, 32, 1024), "out": _log(rng, 100, min(28672, 4001 * 8192 // t)), "rank": 8 * _log(rng, 1, 8),
                "adapters": _log(rng, 1, 64), "runs": rng.choice((1, rng.randint(1, t), min(t, rng.randint(2, 9)), t if t <= 128 else min(t, 9))),
                "layout": rng.choice(("row", "col")), "dtype": dt, "base": rng.choice(("f16", "bf16"))}
    c = {"op": op, "batch": _log(rng, 1, 64), "kv_len": 0, "new": 1, "heads": 0, "kv_heads": rng.choice((1, 2, 4, 8)),
         "dim": rng.choice((64, 128, 128, 256)), "page": rng.choice((16, 32, 64, 128)), "dtype": dt, "fmt": fmt}
    if op == "append":
        c["heads"] = c["kv_heads"] * rng.choice((1, 2, 4, 7, 8))
        c["new"] = rng.choice((1, rng.randint(2, 32), _log(rng, 9, 2048)))
        c["batch"] = min(c["batch"], max(1, 9000 * 32 * 128 // (c["new"] * c["dim"] * max(32, c["heads"]))))
        c["kv_len"] = c["new"] + _log(rng, 1, 4096)
        at = "slot" if c["new"] > 64 else rng.choice(("slot", "given"))
        return c | {"rotary": rng.choice((c["dim"], c["dim"], c["dim"] // 2, 32)), "interleaved": rng.random() < 0.4,
                    "theta": rng.choice((10000.0, 500000.0)), "at": at, "far": 0 if at == "slot" else rng.choice((0, _log(rng, 1000, 1000000)))}
    c["heads"] = c["kv_heads"] * rng.choice((1, 2, 4, 5, 7, 8))
    c["new"] = rng.choice((1, rng.randint(2, 16), rng.randint(17, 64)))
    c["batch"] = min(c["batch"], 32)
    keys = 32 * 8192 * 8 * 128 // (c["batch"] * c["kv_heads"] * c["dim"])  # a sequence's, within the largest case's cache
    keys = min(keys, 32 * 8192 * 64 * 128 * 16 // (c["batch"] * c["heads"] * c["dim"] * c["new"]))  # and its products
    c["kv_len"] = max(c["new"], _log(rng, 16, min(131072, max(32, keys))))
    return c | {"window": rng.choice((0, 0, _log(rng, 100, 4096))), "cap": rng.choice((0.0, 20.0, 50.0))}


# ----------------------------------------------------------------- inputs --


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pow2(amax, fmt):
    """The smallest power of two s (2^-126 at least) with amax <= fmax * s."""
    s = torch.ldexp(torch.ones_like(amax), torch.frexp(amax / _FMAX[fmt])[1] - 1)
    s = torch.where(amax > s * _FMAX[fmt], 2 * s, s)
    return torch.where(amax == 0, 0.0, s).clamp_min(2.0 ** -126)


def _lengths(case, g):
    """Ragged lengths up to kv_len; new tokens a sequence from half of new up to new, the same counts for every seed in another order."""
    b, n = case["batch"], case["new"]
    news = n - (torch.arange(b, device="cuda") * max(1, n // 7)) % (n // 2 + 1)
    news = news[torch.randperm(b, generator=g, device="cuda")]
    lens = torch.randint(max(n, case["kv_len"] // 8), case["kv_len"] + 1, (b,), generator=g, device="cuda")
    lens[0] = case["kv_len"]
    return torch.maximum(lens, news).to(torch.int32), news.to(torch.int32)


def _cache(case, g):
    """A paged pool whose pages lie in no order, filled with keys and values as a model writes them: unit normal with a few
    strong channels, blocks of several magnitudes; what lies behind a sequence's end is what an earlier user left."""
    b, hk, d, ps, fmt = case["batch"], case["kv_heads"], case["dim"], case["page"], case["fmt"]
    width = -(-case["kv_len"] // ps)
    pages = b * width + 3
    table = torch.randperm(pages, generator=g, device="cuda")[: b * width].view(b, width).to(torch.int32)
    made = []
    for strong in (6.0, 1.0):
        x = torch.randn(pages, hk, ps, d, generator=g, device="cuda", dtype=torch.float32)
        x[..., :: max(1, d // 3)] *= strong
        x *= torch.exp(0.5 * torch.randn(pages, hk, 1, 1, generator=g, device="cuda"))
        s = _pow2(x.abs().amax((2, 3)), fmt)
        made += [(x / s[:, :, None, None]).to(_F8[fmt]).view(torch.uint8), s]
    return table, made[0], made[2], made[1], made[3]


def _trees(case, g):
    """Trees of up to `new` nodes for each sequence, parents before children: the nodes' ancestors (themselves among them)
    as truth values [batch, new, new], and their depths [batch, new]."""
    b, n = case["batch"], case["new"]
    see = torch.zeros(b, n, n, dtype=torch.bool, device="cuda")
    depth = torch.zeros(b, n, dtype=torch.int64, device="cuda")
    at = torch.arange(b, device="cuda")
    pick = torch.rand(b, n, generator=g, device="cuda")
    for i in range(n):
        if i:
            parent = (i - 1 - (pick[:, i] ** 2 * i).long()).clamp(0, i - 1)  # mostly one of the last nodes
            see[:, i] = see[at, parent]
            depth[:, i] = depth[at, parent] + 1
        see[:, i, i] = True
    return see, depth


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    s = {"case": dict(case)}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "norm":
        t, h = case["tokens"], case["hidden"]
        wide = h + case["pad"]
        y = randn(t, wide) * torch.exp(0.5 * randn(t, 1))
        y[:, :: max(1, h // 5)] *= 20.0  # a few strong channels
        s["y"] = y.to(dt)[:, :h]
        s["residual"] = None if case["res"] == "none" else (randn(t, h) * 3.0).to(_DT[case["res"]])
        s["post"] = (1.0 - case["offset"] + 0.2 * randn(h)).to(dt) if case["post"] else None
        s["pre"] = (1.0 - case["offset"] + 0.2 * randn(h)).to(dt)
        s["gate"] = {"none": None, "channel": randn(h).to(dt), "token": randn(t, wide).to(dt)[:, :h] if case["gate"] == "token" else None}[case["gate"]]
        return s
    if case["op"] == "lora":
        t, k, n, r, a = (case[x] for x in ("tokens", "in", "out", "rank", "adapters"))
        s["x"] = randn(t, k).to(dt)
        s["a"] = (randn(a, r, k) / math.sqrt(k)).to(dt)
        s["b"] = (randn(a, n, r) * (0.3 / math.sqrt(r))).to(dt)
        s["scales"] = 0.5 + 1.5 * torch.rand(a, generator=g, device="cuda")
        # requests one after another, each with its adapter (about one in twelve with none); lengths from the seed
        runs = case["runs"]
        ids = torch.randint(0, a, (runs,), generator=g, device="cuda")
        if runs <= a:
            ids = torch.randperm(a, generator=g, device="cuda")[:runs]
        if runs > 1:
            ids = torch.where(torch.rand(runs, generator=g, device="cuda") < 1 / 12, -1, ids)
        cuts = torch.sort(torch.randperm(t - 1, generator=g, device="cuda")[: runs - 1] + 1)[0] if t > 1 else torch.zeros(0, dtype=torch.int64, device="cuda")
        s["ids"] = ids[torch.searchsorted(cuts, torch.arange(t, device="cuda"), right=True)].to(torch.int32)
        base = randn(t, n).to(_DT[case["base"]])
        s["base"] = base.t().contiguous().t() if case["layout"] == "col" else base
        return s
    lens, news = _lengths(case, g)
    table, kc, vc, ks, vs = _cache(case, g)
    cu = torch.zeros(case["batch"] + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(news, 0)
    t = int(cu[-1])
    s |= {"lens": lens, "table": table, "k_cache": kc, "v_cache": vc, "k_scale": ks, "v_scale": vs,
          "cu": None if case["new"] == 1 else cu, "cu_all": cu}
    tree = case["op"] == "tree" or case["at"] == "given"
    live = torch.arange(case["new"], device="cuda")[None] < news[:, None]
    if tree:
        see, depth = _trees(case, g)
        start = (lens - news).long()[:, None] + case.get("far", 0)
        s["positions"] = (start + depth)[live].to(torch.int32)
        words = -(-case["new"] // 32)
        bits = torch.zeros(case["batch"], case["new"], 32 * words, dtype=torch.int64, device="cuda")
        bits[:, :, : case["new"]] = see.long()
        bits = (bits.view(case["batch"], case["new"], words, 32) << torch.arange(32, device="cuda")).sum(-1)
        s["mask"] = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits)[live].to(torch.int32)
    if case["op"] == "append":
        # rows of a fused q/k/v projection: token stride wider than the row
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        qkv = (randn(t, h + 2 * hk, d) * torch.exp(randn(t, 1, 1))).to(dt)
        s |= {"q": qkv[:, :h], "k": qkv[:, h: h + hk], "v": qkv[:, h + hk:]}
        half = torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64)
        s["inv_freq"] = (case["theta"] ** (-half / case["rotary"])).float()
        if not tree:
            s["positions"] = None
    else:
        s["q"] = randn(t, case["heads"], case["dim"]).to(dt)
    return s


# ------------------------------------------------------------ plain forms --


def _rms(x, w, offset):
    return x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6) * (w.float() + offset)


def _plain_norm(s):
    c = s["case"]
    z = s["y"].float()
    if s["post"] is not None:
        z = _rms(z, s["post"], c["offset"])
    if s["gate"] is not None:
        z = z * s["gate"].float()
    z = z * c["alpha"]
    if s["residual"] is not None:
        z = z + s["residual"].float()
    kept = z.dtype if c["res"] == "f32" else s["y"].dtype
    return z.to(kept), _rms(z, s["pre"], c["offset"]).to(s["y"].dtype)


def _plain_lora(s):
    c = s["case"]
    x = s["x"].float()
    y = s["base"].float().contiguous()
    at = s["ids"].long()
    if c["tokens"] <= 128:  # a product of its own for each token
        pick = at.clamp_min(0)
        u = (s["a"][pick].float() @ x[:, :, None])
        d = (s["b"][pick].float() @ u)[:, :, 0] * s["scales"][pick][:, None]
        y = y + torch.where(at[:, None] >= 0, d, 0.0)
    else:  # all tokens through every adapter, those of the others dropped
        for e in range(c["adapters"]):
            d = (x @ s["a"][e].float().t()) @ s["b"][e].float().t()
            y = y + torch.where((at == e)[:, None], d * s["scales"][e], 0.0)
    y = y.to(s["base"].dtype)
    return y.t().contiguous().t() if c["layout"] == "col" else y


def _plain_turn(x, pos, s):
    """[tokens, heads, dim] with its first `rotary` channels turned by the angles of the positions."""
    c = s["case"]
    r = c["rotary"]
    a = pos.double()[:, None] * s["inv_freq"].double()[None]
    cos, sin = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    x = x.float()
    y = x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    y[..., first] = x[..., first] * cos - x[..., second] * sin
    y[..., second] = x[..., second] * cos + x[..., first] * sin
    return y


def _plain_append(s):
    c = s["case"]
    fmt, ps = c["fmt"], c["page"]
    t = s["k"].shape[0]
    tok = torch.arange(t, device="cuda")
    seq = torch.searchsorted(s["cu_all"][1:].contiguous(), tok, right=True)
    news = s["cu_all"][1:] - s["cu_all"][:-1]
    start = (s["lens"] - news).long()  # position of each sequence's first new token
    pos = start[seq] + tok - s["cu_all"][:-1].long()[seq]
    turn = pos if s["positions"] is None else s["positions"]
    page = s["table"].long()[seq, pos // ps]
    # the one page of a sequence that may hold earlier tokens
    part = s["table"].long().gather(1, (start // ps).clamp_max(s["table"].shape[1] - 1)[:, None])[:, 0]
    has = (start % ps) > 0
    earlier = has[:, None, None] & (torch.arange(ps, device="cuda")[None, None, :] < (start % ps)[:, None, None])
    for name in ("k", "v"):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        x = _plain_turn(s["k"], turn, s) if name == "k" else s["v"].float()
        pages, hk = scale.shape
        amax = torch.zeros(pages, hk, device="cuda").index_reduce_(0, page, torch.where(torch.isfinite(x), x.abs(), 0.0).amax(2), "amax")
        base = torch.zeros(pages, hk, device="cuda")
        base[part] = torch.where(has[:, None], scale[part], 0.0)
        touched = torch.zeros(pages, dtype=torch.bool, device="cuda")
        touched[page] = True
        fresh = torch.where(touched[:, None], torch.maximum(_pow2(amax, fmt), base), scale)
        rows = cache[part]
        moved = (rows.view(_F8[fmt]).float() * (scale[part] / fresh[part])[:, :, None, None]).to(_F8[fmt])
        cache[part] = torch.where(earlier[..., None], moved.view(torch.uint8), rows)
        codes = (x / fresh[page][:, :, None]).clamp(-_FMAX[fmt], _FMAX[fmt]).to(_F8[fmt])
        cache[page, :, pos % ps] = codes.view(torch.uint8)
        scale.copy_(fresh)
    return _plain_turn(s["q"], turn, s).to(s["q"].dtype)


def _plain_tree(s):
    c = s["case"]
    q, fmt, hk = s["q"], c["fmt"], c["kv_heads"]
    b, d, n = c["batch"], c["dim"], c["new"]
    grp = c["heads"] // hk
    table = s["table"].long()

    def rows(cache, scale):
        x = cache[table].view(_F8[fmt]).float() * scale[table][..., None, None]  # [B, P, Hk, page, D]
        return x.permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)

    k, v = rows(s["k_cache"], s["k_scale"]), rows(s["v_cache"], s["v_scale"])
    cu, lens = s["cu_all"].long(), s["lens"].long()
    news = cu[1:] - cu[:-1]
    start = lens - news
    i = torch.arange(n, device="cuda")
    j = torch.arange(k.shape[2], device="cuda")
    at = (cu[:-1, None] + i[None]).clamp_max(q.shape[0] - 1)
    pos = s["positions"].long()[at]  # [B, n]
    before = j[None, None] < start[:, None, None]
    if c["window"]:
        before = before & (j[None, None] > pos[..., None] - c["window"])
    step = j[None] - start[:, None]  # [B, J]: number of the step's token behind the key
    word = s["mask"].long()[at].gather(2, (step // 32).clamp(0, s["mask"].shape[1] - 1)[:, None].expand(b, n, -1))
    drafted = ((word >> (step % 32)[:, None]) & 1).bool() & (step >= 0)[:, None] & (j[None] < lens[:, None])[:, None]
    seen = before | drafted
    v = torch.where((j[None] < lens[:, None])[:, None, :, None], v, 0.0)
    qp = q[at].float().view(b, n, hk, grp, d).permute(0, 2, 1, 3, 4).reshape(b, hk, n * grp, d)
    sc = (qp @ k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    if c["cap"]:
        sc = c["cap"] * torch.tanh(sc / c["cap"])
    sc = sc.view(b, hk, n, grp, -1).masked_fill(~seen[:, None, :, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(m), 0.0, m))
    l = p.sum(-1, keepdim=True)
    o = (p.view(b, hk, n * grp, -1) @ v).view(b, hk, n, grp, d) / torch.where(l == 0, 1.0, l)
    lse = (m + torch.log(l)).squeeze(-1)
    live = i[None] < news[:, None]
    o = o.permute(0, 2, 1, 3, 4).reshape(b, n, hk * grp, d)[live]
    return o.to(q.dtype), lse.permute(0, 2, 1, 3).reshape(b, n, hk * grp)[live]


# -------------------------------------------------------------- one pass --


def run(state):
    s, c = state, state["case"]
    ops = _ops() if own else None
    if c["op"] == "norm":
        if own:
            return ops.residual_norm(s["y"], s["residual"], post_weight=s["post"], pre_weight=s["pre"], gate=s["gate"], alpha=c["alpha"],
                                     eps=1e-6, weight_offset=c["offset"])
        return _plain_norm(s)
    if c["op"] == "lora":
        if own:
            return ops.lora_add(s["base"], s["x"], s["a"], s["b"], s["ids"], scales=s["scales"])
        return _plain_lora(s)
    where = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lens"])
    if c["op"] == "append":
        if own:
            q = ops.kv_append_rope(s["q"], s["k"], s["v"], *where, s["inv_freq"], cu_seqlens=s["cu"], positions=s["positions"],
                                   interleaved=c["interleaved"], fmt=c["fmt"])
        else:
            q = _plain_append(s)
        f8 = _F8[c["fmt"]]
        return q, s["k_cache"].view(f8), s["v_cache"].view(f8), s["k_scale"], s["v_scale"]
    if own:
        return ops.kv_attention_tree(s["q"], *where, s["mask"], cu_seqlens=s["cu"], positions=s["positions"], softcap=c["cap"],
                                     window=c["window"], fmt=c["fmt"])
    return _plain_tree(s)


def work(case):
    """Bytes each read or written once, and the products' flops; ragged lengths and adapters at their expectation."""
    c = case
    if c["op"] == "norm":
        t, h = c["tokens"], c["hidden"]
        res = 4 if c["res"] == "f32" else 2
        each = 4 + res * (1 if c["res"] == "none" else 2) + (2 if c["gate"] == "token" else 0)
        return {"bytes": t * h * each + 2 * h * (1 + c["post"] + (c["gate"] == "channel")), "flops": 0}
    if c["op"] == "lora":
        t, k, n, r = c["tokens"], c["in"], c["out"], c["rank"]
        held = 1.0 if c["runs"] == 1 else 11 / 12
        busy = held * (c["runs"] if c["runs"] <= c["adapters"] else c["adapters"] * (1 - (1 - 1 / c["adapters"]) ** c["runs"]))
        return {"bytes": 2 * (held * t * k + 2 * t * n + busy * r * (k + n)), "flops": 2 * held * t * r * (k + n)}
    b = c["batch"]
    new = b * 0.75 * c["new"] if c["new"] > 1 else b
    row = c["kv_heads"] * c["dim"]
    if c["op"] == "append":
        return {"bytes": new * (row * 2 * 3 + c["heads"] * c["dim"] * 4), "flops": 0}
    keys = (c["kv_len"] + (b - 1) * c["kv_len"] * 9 / 16) if b > 1 else c["kv_len"]
    keys = min(keys, b * (c["window"] + c["new"])) if c["window"] else keys
    rows = c["heads"] * c["dim"]
    return {"bytes": 2 * keys * row + 4 * new * rows, "flops": 4 * keys * (new / b) * rows}


# ------------------------------------------------------- 64-bit definition --


def _exact_norm(s):
    c = s["case"]

    def norm(x, w):
        return x / torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + 1e-6) * (w.double() + c["offset"])

    b = s["y"].double()
    b = b if s["post"] is None else norm(b, s["post"])
    b = c["alpha"] * b * (1.0 if s["gate"] is None else s["gate"].double())
    r = b if s["residual"] is None else s["residual"].double() + b
    return r, norm(r, s["pre"])


def _exact_lora(s):
    y = s["base"].double()
    for e in s["ids"].unique().tolist():
        if e >= 0:
            t = torch.nonzero(s["ids"] == e)[:, 0]
            y[t] += s["scales"][e].double() * (s["x"][t].double() @ (s["b"][e].double() @ s["a"][e].double()).t() if t.numel() > 2 * s["x"].shape[1]
                                               else (s["x"][t].double() @ s["a"][e].double().t()) @ s["b"][e].double().t())
    return y


def _exact_turn(x, at, s):
    c = s["case"]
    r = c["rotary"]
    z = x[..., :r].double()
    z = z.unflatten(-1, (r // 2, 2)) if c["interleaved"] else z.unflatten(-1, (2, r // 2)).transpose(-1, -2)
    angle = (at.double()[:, None] * s["inv_freq"].double())[:, None]
    w = torch.view_as_complex(z.contiguous()) * torch.polar(torch.ones_like(angle), angle)
    w = torch.view_as_real(w)
    w = w.flatten(-2) if c["interleaved"] else w.transpose(-1, -2).flatten(-2)
    return torch.cat((w, x[..., r:].double()), -1)


def _exact_append(s):
    """Token by token in the order of the pages: gather what a page gets, take its scale, move the earlier codes, write the new ones."""
    c = s["case"]
    ps, fmax = c["page"], _FMAX[c["fmt"]]
    f8 = _F8[c["fmt"]]
    lens, cu, table = s["lens"].tolist(), s["cu_all"].tolist(), s["table"].tolist()
    at = s["positions"]
    if at is None:
        at = torch.cat([torch.arange(lens[b] - (cu[b + 1] - cu[b]), lens[b], device="cuda") for b in range(c["batch"])])
    got = []
    for name in ("k", "v"):
        vals = s[name + "_cache"].view(f8).double()
        scale = s[name + "_scale"].double()
        x = _exact_turn(s["k"], at, s) if name == "k" else s["v"].double()
        for b in range(c["batch"]):
            n = cu[b + 1] - cu[b]
            pos = lens[b] - n
            done = 0
            while done < n:
                page, slot = table[b][(pos + done) // ps], (pos + done) % ps
                take = min(ps - slot, n - done)
                rows = x[cu[b] + done: cu[b] + done + take].transpose(0, 1)  # [Hk, take, D]
                amax = rows.abs().amax((1, 2))
                sc = torch.exp2(torch.ceil(torch.log2((amax / fmax).clamp_min(2.0 ** -126))))
                sc = torch.where(sc / 2 * fmax >= amax, sc / 2, sc).clamp_min(2.0 ** -126)
                if slot:
                    sc = torch.maximum(sc, scale[page])
                    old = vals[page, :, :slot] * (scale[page] / sc)[:, None, None]
                    vals[page, :, :slot] = old.float().to(f8).double()
                vals[page, :, slot: slot + take] = (rows / sc[:, None, None]).clamp(-fmax, fmax).float().to(f8).double()
                scale[page] = sc
                done += take
        got.append((vals, scale))
    return _exact_turn(s["q"], at, s), got[0][0], got[1][0], got[0][1], got[1][1]


def _exact_tree(s):
    c = s["case"]
    f8, ps, hk = _F8[c["fmt"]], c["page"], c["kv_heads"]
    grp = c["heads"] // hk
    lens, cu = s["lens"].tolist(), s["cu_all"].tolist()
    outs, lses = [], []
    for b in range(c["batch"]):
        n, ln = cu[b + 1] - cu[b], lens[b]
        pages = s["table"][b, : -(-ln // ps)].long()

        def keys(cache, scale):
            x = cache[pages].view(f8).double() * scale[pages].double()[:, :, None, None]
            return x.transpose(0, 1).flatten(1, 2)[:, :ln]

        k, v = keys(s["k_cache"], s["k_scale"]), keys(s["v_cache"], s["v_scale"])
        pos = s["positions"][cu[b]: cu[b + 1]].long()
        hide = torch.zeros(n, ln, dtype=torch.bool, device="cuda")
        if c["window"]:
            hide[:, : ln - n] = torch.arange(ln - n, device="cuda")[None] <= pos[:, None] - c["window"]
        m = s["mask"][cu[b]: cu[b + 1]].long() & 0xFFFFFFFF
        for i in range(n):
            hide[:, ln - n + i] = (m[:, i // 32] // 2 ** (i % 32)) % 2 == 0
        step = max(1, 2 ** 28 // max(1, hk * grp * ln))  # rows at a time
        for i in range(0, n, step):
            q = s["q"][cu[b] + i: min(cu[b] + i + step, cu[b + 1])].double().unflatten(1, (hk, grp))
            sc = torch.einsum("nhgd,hjd->hngj", q, k) / math.sqrt(c["dim"])
            if c["cap"]:
                sc = c["cap"] * torch.tanh(sc / c["cap"])
            sc = sc.masked_fill(hide[i: i + step][None, :, None], -math.inf)
            lse = torch.logsumexp(sc, -1)
            outs.append(torch.einsum("hngj,hjd->nhgd", torch.exp(sc - lse[..., None]), v).flatten(1, 2))
            lses.append(lse.permute(1, 0, 2).flatten(1, 2))
    return torch.cat(outs), torch.cat(lses)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "lora": _exact_lora, "append": _exact_append, "tree": _exact_tree}[case["op"]](s)
