"""Cases and plain forms of the serving operators: the paged 8-bit KV cache (append and attention), the
mixture-of-experts layer with FP8 weights for a few tokens, and the scoring of logits.

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
        # one new token of each of 64 sequences enters the cache (a decode step of a served batch)
        {"name": "append decode 64", "op": "append", "batch": 64, "kv_len": 4000, "new": 1, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "fmt": "e4m3"},
        # ragged prompts enter the cache after a prefill, page of 16, none of them a whole number of pages
        {"name": "append prompts", "op": "append", "batch": 6, "kv_len": 3001, "new": 2048, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "f16", "fmt": "e4m3"},
        # one short conversation: the smallest call, where only latency counts
        {"name": "attend one short", "op": "attend", "batch": 1, "kv_len": 517, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 0, "dtype": "bf16", "fmt": "e4m3"},
        # a served batch at mixed lengths, grouped heads as in a 70B-style model
        {"name": "attend batch 128", "op": "attend", "batch": 128, "kv_len": 8192, "new": 1, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 0, "dtype": "bf16", "fmt": "e4m3"},
        # one long document: few rows, the work has to be split along the keys
        {"name": "attend one long", "op": "attend", "batch": 1, "kv_len": 131000, "new": 1, "heads": 64, "kv_heads": 8, "dim": 128, "page": 128,
         "window": 0, "dtype": "f16", "fmt": "e4m3"},
        # drafts of up to 6 tokens are verified, ragged, over a sliding window, heads of 64
        {"name": "attend drafts", "op": "attend", "batch": 24, "kv_len": 6000, "new": 6, "heads": 28, "kv_heads": 4, "dim": 64, "page": 16,
         "window": 2048, "dtype": "f16", "fmt": "e5m2"},
        # one token through fine-grained experts: latency counts
        {"name": "moe one token", "op": "moe", "tokens": 1, "experts": 64, "top_k": 6, "hidden": 2048, "inter": 1408, "renorm": True, "act": "silu",
         "dtype": "bf16", "fmt": "e4m3"},
        # a decode batch of 8 through 8 wide experts (4096 x 11008 projections)
        {"name": "moe batch 8", "op": "moe", "tokens": 8, "experts": 8, "top_k": 2, "hidden": 4096, "inter": 11008, "renorm": True, "act": "silu",
         "dtype": "bf16", "fmt": "e4m3"},
        # the largest batch of the path, every expert busy
        {"name": "moe batch 64", "op": "moe", "tokens": 64, "experts": 32, "top_k": 4, "hidden": 4096, "inter": 2048, "renorm": False, "act": "gelu",
         "dtype": "f16", "fmt": "e5m2"},
        # the sampled token of one stream with a few alternatives
        {"name": "score one token", "op": "score", "tokens": 1, "vocab": 32000, "top": 8, "dtype": "bf16", "layout": "row", "temperature": 1.0,
         "masked": 0.0},
        # a decode batch on the GEMM's default column-major logits, part of the vocabulary masked by a grammar
        {"name": "score batch 16 col", "op": "score", "tokens": 16, "vocab": 128000, "top": 20, "dtype": "f16", "layout": "col",
         "temperature": 0.7, "masked": 0.3},
        # log probabilities of a whole prompt, odd vocabulary (rows of every alignment)
        {"name": "score prompt 4096", "op": "score", "tokens": 4096, "vocab": 32001, "top": 5, "dtype": "bf16", "layout": "row",
         "temperature": 1.0, "masked": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "moe", "moe", "score"))
    dt, fmt = rng.choice(("f16", "bf16")), rng.choice(("e4m3", "e4m3", "e5m2"))
    if op in ("append", "attend"):
        c = {"op": op, "batch": _log(rng, 1, 128), "kv_len": 0, "new": 1, "kv_heads": rng.choice((1, 2, 4, 8)), "dim": rng.choice((64, 128, 128, 256)),
             "page": rng.choice((16, 32, 64, 128)), "dtype": dt, "fmt": fmt}
        if op == "append":
            c["new"] = rng.choice((1, rng.randint(2, 8), _log(rng, 9, 4096)))
            c["batch"] = min(c["batch"], max(1, 12288 // c["new"]))
            c["kv_len"] = c["new"] + _log(rng, 1, 4096)
            return c
        c["heads"] = c["kv_heads"] * rng.choice((1, 2, 4, 5, 7, 8, 16))
        c["new"] = rng.choice((1, 1, rng.randint(2, 8)))
        most = 128 * 8192 * 8 * 128 // (c["batch"] * c["kv_heads"] * c["dim"])  # keys a sequence within the largest case's cache
        c["kv_len"] = max(c["new"], _log(rng, 16, min(131072, max(32, most))))
        c["window"] = rng.choice((0, 0, _log(rng, 100, 4096)))
        return c
    if op == "moe":
        e = rng.choice((4, 8, 16, 60, 64, 128))
        h = 16 * _log(rng, 32, 256)
        i = 16 * _log(rng, 16, max(17, min(688, 270_000_000 // (e * h * 16))))
        return {"op": op, "tokens": _log(rng, 1, 64), "experts": e, "top_k": rng.randint(1, min(8, e)), "hidden": h, "inter": i,
                "renorm": rng.random() < 0.5, "act": rng.choice(("silu", "gelu")), "dtype": dt, "fmt": fmt}
    t = _log(rng, 1, 2048)
    return {"op": op, "tokens": t, "vocab": _log(rng, 500, min(200000, 4096 * 32000 // (2 * t))), "top": rng.choice((0, 1, 5, 20, 32)),
            "dtype": rng.choice(("f16", "bf16", "f32")), "layout": rng.choice(("row", "row", "col")), "temperature": rng.choice((1.0, 0.7, 1.3)),
            "masked": rng.choice((0.0, 0.0, 0.5))}


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


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] in ("append", "attend"):
        lens, news = _lengths(case, g)
        table, kc, vc, ks, vs = _cache(case, g)
        cu = torch.zeros(case["batch"] + 1, dtype=torch.int32, device="cuda")
        cu[1:] = torch.cumsum(news, 0)
        t = int(cu[-1])
        s |= {"lens": lens, "table": table, "k_cache": kc, "v_cache": vc, "k_scale": ks, "v_scale": vs,
              "cu": None if case["new"] == 1 else cu, "cu_all": cu, "max_new": case["new"]}
        if case["op"] == "append":
            # rows of a fused q/k/v projection: token stride wider than the row
            kv = torch.randn(t, 3, case["kv_heads"], case["dim"], generator=g, device="cuda") * torch.exp(torch.randn(t, 1, 1, 1, generator=g, device="cuda"))
            kv = kv.to(dt)
            s |= {"k": kv[:, 1], "v": kv[:, 2]}
        else:
            s["q"] = torch.randn(t, case["heads"], case["dim"], generator=g, device="cuda").to(dt)
        return s
    if case["op"] == "moe":
        e, h, i, fmt = case["experts"], case["hidden"], case["inter"], case["fmt"]
        for name, n, k in (("up", 2 * i, h), ("down", h, i)):
            w = torch.empty(e, n, k, dtype=torch.uint8, device="cuda")
            sc = torch.empty(e, n, dtype=torch.float32, device="cuda")
            for j in range(e):
                x = torch.randn(n, k, generator=g, device="cuda", dtype=torch.float32) * (0.8 / math.sqrt(k))
                sc[j] = x.abs().amax(1).clamp_min(1e-30) / _FMAX[fmt]
                w[j] = (x / sc[j][:, None]).to(_F8[fmt]).view(torch.uint8)
            s |= {"w_" + name: w, "s_" + name: sc}
        s["x"] = torch.randn(case["tokens"], h, generator=g, device="cuda").to(dt)
        s["router"] = (torch.randn(e, h, generator=g, device="cuda") * (1.5 / math.sqrt(h))).to(dt)
        return s
    t, v = case["tokens"], case["vocab"]
    x = torch.randn(t, v, generator=g, device="cuda") * 2.5
    if case["masked"]:
        x.masked_fill_(torch.rand(t, v, generator=g, device="cuda") < case["masked"], -math.inf)
    at = torch.randint(0, v, (t,), generator=g, device="cuda")
    at = torch.where(torch.rand(t, generator=g, device="cuda") < 0.7, x.argmax(1), at)  # most given tokens are likely ones
    x[torch.arange(t, device="cuda"), at] = x[torch.arange(t, device="cuda"), at].clamp_min(-20.0)
    x = x.to(dt)
    if case["layout"] == "col":
        x = x.t().contiguous().t()
    return s | {"logits": x, "tokens": at.to(torch.int32)}


# ------------------------------------------------------------ plain forms --


def _plain_append(s):
    c = s["case"]
    fmt, ps = c["fmt"], c["page"]
    t = s["k"].shape[0]
    tok = torch.arange(t, device="cuda")
    seq = torch.searchsorted(s["cu_all"][1:].contiguous(), tok, right=True)
    news = s["cu_all"][1:] - s["cu_all"][:-1]
    start = (s["lens"] - news).long()  # position of each sequence's first new token
    pos = start[seq] + tok - s["cu_all"][:-1].long()[seq]
    page = s["table"].long()[seq, pos // ps]
    # the one page of a sequence that may hold earlier tokens
    part = s["table"].long().gather(1, (start // ps).clamp_max(s["table"].shape[1] - 1)[:, None])[:, 0]
    has = (start % ps) > 0
    earlier = has[:, None, None] & (torch.arange(ps, device="cuda")[None, None, :] < (start % ps)[:, None, None])
    for name in ("k", "v"):
        cache, scale, x = s[name + "_cache"], s[name + "_scale"], s[name].float()
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


def _plain_attend(s):
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
    i = torch.arange(n, device="cuda")
    j = torch.arange(k.shape[2], device="cuda")
    at = (cu[:-1, None] + i[None]).clamp_max(q.shape[0] - 1)
    pos = (lens - news)[:, None] + i[None]  # [B, n]
    seen = (j[None, None] <= pos[..., None]) & (j[None, None] < lens[:, None, None])
    if c["window"]:
        seen &= j[None, None] > pos[..., None] - c["window"]
    v = torch.where((j[None] < lens[:, None])[:, None, :, None], v, 0.0)
    qp = q[at].float().view(b, n, hk, grp, d).permute(0, 2, 1, 3, 4).reshape(b, hk, n * grp, d)
    sc = (qp @ k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    sc = sc.view(b, hk, n, grp, -1).masked_fill(~seen[:, None, :, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(m), 0.0, m))
    l = p.sum(-1, keepdim=True)
    o = (p.view(b, hk, n * grp, -1) @ v).view(b, hk, n, grp, d) / torch.where(l == 0, 1.0, l)
    lse = (m + torch.log(l)).squeeze(-1)
    live = i[None] < news[:, None]
    o = o.permute(0, 2, 1, 3, 4).reshape(b, n, hk * grp, d)[live]
    return o.to(q.dtype), lse.permute(0, 2, 1, 3).reshape(b, n, hk * grp)[live]


def _act(x, act):
    if act == "silu":
        return x * torch.sigmoid(x)
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def _plain_moe(s):
    c = s["case"]
    fmt, k, i = c["fmt"], c["top_k"], c["inter"]
    x = s["x"].float()
    r = x @ s["router"].float().t()
    ids = torch.sort(r, dim=1, descending=True, stable=True)[1][:, :k]
    w = torch.softmax(r.gather(1, ids) if c["renorm"] else r, 1)
    w = w if c["renorm"] else w.gather(1, ids)

    def weights(name, pick):
        codes, scale = s["w_" + name], s["s_" + name]
        codes, scale = (codes, scale) if pick is None else (codes[pick], scale[pick])
        return (codes.view(_F8[fmt]).float() * scale[..., None]).transpose(1, 2)

    t = x.shape[0]
    if t * k < c["experts"]:  # fewer picks than experts: the picked experts' weights
        pick = ids.reshape(-1)
        a = x.repeat_interleave(k, 0)[:, None]
        up = a @ weights("up", pick)
        y = ((_act(up[..., :i], c["act"]) * up[..., i:]) @ weights("down", pick)).view(t, k, -1)
    else:
        up = x[None] @ weights("up", None)
        y = (_act(up[..., :i], c["act"]) * up[..., i:]) @ weights("down", None)  # [E, T, H]
        y = y.transpose(0, 1).gather(1, ids[..., None].expand(-1, -1, y.shape[2]))
    return (y * w[..., None]).sum(1).to(s["x"].dtype), ids.to(torch.int32), w


def _order(x):
    """int64 keys that sort as x does, equal values by the lowest index first."""
    bits = x.float().view(torch.int32).long()
    bits = torch.where(bits < 0, -2147483648 - bits, bits)  # -0 and +0 are one value
    return (bits << 32) - torch.arange(x.shape[1], device=x.device)


def _plain_score(s):
    c = s["case"]
    z = s["logits"].float() * (1.0 / c["temperature"])
    m = z.amax(1, keepdim=True)
    p = torch.exp(z - m)
    l = p.sum(1, keepdim=True)
    lse = m + torch.log(l)
    lp = z - lse
    ent = -(p / l * torch.where(p == 0, 0.0, lp)).sum(1)
    at = s["tokens"].long()[:, None]
    top = torch.topk(_order(s["logits"]), c["top"], 1)[1]
    return lp.gather(1, at)[:, 0], ent, top.to(torch.int32), lp.gather(1, top)


# -------------------------------------------------------------- one pass --


def run(state):
    s, c = state, state["case"]
    if not own:
        if c["op"] == "append":
            _plain_append(s)
            f8 = _F8[c["fmt"]]
            return s["k_cache"].view(f8), s["v_cache"].view(f8), s["k_scale"], s["v_scale"]
        return {"attend": _plain_attend, "moe": _plain_moe, "score": _plain_score}[c["op"]](s)
    ops = _ops()
    if c["op"] == "append":
        ops.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lens"], s["cu"], c["fmt"])
        f8 = _F8[c["fmt"]]
        return s["k_cache"].view(f8), s["v_cache"].view(f8), s["k_scale"], s["v_scale"]
    if c["op"] == "attend":
        return ops.kv_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lens"], s["cu"],
                                window=c["window"], fmt=c["fmt"])
    if c["op"] == "moe":
        return ops.moe_forward(s["x"], s["router"], s["w_up"], s["s_up"], s["w_down"], s["s_down"], c["top_k"], renormalize=c["renorm"],
                               act=c["act"], b_format=c["fmt"])
    return ops.token_logprobs(s["logits"], s["tokens"], top=c["top"], temperature=c["temperature"])


def work(case):
    """Bytes each read or written once, and the products' flops; ragged lengths and routing at their expectation."""
    c = case
    if c["op"] in ("append", "attend"):
        b = c["batch"]
        new = b * 0.75 * c["new"] if c["new"] > 1 else b
        row = c["kv_heads"] * c["dim"]
        if c["op"] == "append":
            return {"bytes": new * row * 2 * 3, "flops": 0}
        keys = (c["kv_len"] + (b - 1) * c["kv_len"] * 9 / 16) if b > 1 else c["kv_len"]
        keys = min(keys, b * (c["window"] + c["new"])) if c["window"] else keys
        rows = c["heads"] * c["dim"]
        return {"bytes": 2 * keys * row + 4 * new * rows, "flops": 4 * keys * (new / b) * rows}
    if c["op"] == "moe":
        e, h, i, t, k = c["experts"], c["hidden"], c["inter"], c["tokens"], c["top_k"]
        busy = e * (1 - (1 - k / e) ** t)
        return {"bytes": busy * (3 * h * i + 4 * (2 * i + h)) + 2 * e * h + 4 * t * h, "flops": 2 * t * (3 * k * h * i + e * h)}
    size = 4 if c["dtype"] == "f32" else 2
    return {"bytes": c["tokens"] * (c["vocab"] * size + 12 + 8 * c["top"]), "flops": 0}


# ------------------------------------------------------- 64-bit definition --


def _exact_append(s):
    """Token by token in the order of the pages: gather what a page gets, take its scale, move the earlier codes, write the new ones."""
    c = s["case"]
    ps, fmax = c["page"], _FMAX[c["fmt"]]
    f8 = _F8[c["fmt"]]
    lens, cu, table = s["lens"].tolist(), s["cu_all"].tolist(), s["table"].tolist()
    got = []
    for name in ("k", "v"):
        vals = s[name + "_cache"].view(f8).double()
        scale = s[name + "_scale"].double()
        x = s[name].double()
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
    return got[0][0], got[1][0], got[0][1], got[1][1]


def _exact_attend(s):
    c = s["case"]
    f8, ps, hk = _F8[c["fmt"]], c["page"], c["kv_heads"]
    grp = c["heads"] // hk
    lens, cu = s["lens"].tolist(), s["cu_all"].tolist()
    outs, lses = [], []
    for b in range(c["batch"]):
        n, ln = cu[b + 1] - cu[b], lens[b]
        first = max(0, ln - n - c["window"]) // ps if c["window"] else 0
        pages = s["table"][b, first: -(-ln // ps)].long()

        def keys(cache, scale):
            x = cache[pages].view(f8).double() * scale[pages].double()[:, :, None, None]
            return x.transpose(0, 1).flatten(1, 2)[:, : ln - first * ps]

        k, v = keys(s["k_cache"], s["k_scale"]), keys(s["v_cache"], s["v_scale"])
        q = s["q"][cu[b]: cu[b + 1]].double().view(n, hk, grp, c["dim"])
        sc = torch.einsum("nhgd,hjd->hngj", q, k) / math.sqrt(c["dim"])
        j = torch.arange(first * ps, ln, device="cuda")
        pos = torch.arange(ln - n, ln, device="cuda")[:, None]
        hide = (j[None] > pos) | ((j[None] <= pos - c["window"]) if c["window"] else torch.zeros_like(j[None] > pos))
        sc = sc.masked_fill(hide[None, :, None], -math.inf)
        lse = torch.logsumexp(sc, -1)
        outs.append(torch.einsum("hngj,hjd->nhgd", torch.exp(sc - lse[..., None]), v).reshape(n, c["heads"], -1))
        lses.append(lse.permute(1, 0, 2).reshape(n, c["heads"]))
    return torch.cat(outs), torch.cat(lses)


def _exact_moe(s):
    c = s["case"]
    f8, k, i = _F8[c["fmt"]], c["top_k"], c["inter"]
    x = s["x"].double()
    r = x @ s["router"].double().t()
    w, ids = torch.topk(r, k, 1)
    full = torch.logsumexp(w if c["renorm"] else r, 1, keepdim=True)
    w = torch.exp(w - full)
    y = torch.zeros_like(x)
    for e in ids.unique().tolist():
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        up = (x[t] @ s["w_up"][e].view(f8).double().t()) * s["s_up"][e].double()
        a, b = up[:, :i], up[:, i:]
        a = a / (1 + torch.exp(-a)) if c["act"] == "silu" else a / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)))
        y[t] += w[t, slot][:, None] * ((a * b) @ s["w_down"][e].view(f8).double().t()) * s["s_down"][e].double()
    return y, None, w


def _exact_score(s):
    c = s["case"]
    lps, ents, tops = [], [], []
    for x, at in zip(s["logits"].split(256), s["tokens"].split(256)):
        z = x.double() / c["temperature"]
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        lps.append(lp.gather(1, at.long()[:, None])[:, 0])
        ents.append(-torch.special.xlogy(lp.exp(), lp.exp()).sum(1))
        tops.append(torch.topk(lp, c["top"], 1)[0])
    return torch.cat(lps), torch.cat(ents), None, torch.cat(tops)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "moe": _exact_moe, "score": _exact_score}[case["op"]](s)
