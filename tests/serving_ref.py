"""Plain 64-bit restatements of the decode-step operators, from their
definitions, for the tests. They run on whatever device the inputs are on."""
from __future__ import annotations

import math

import torch

F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of the type, relative


def codes_to_f64(codes: torch.Tensor, fmt: str) -> torch.Tensor:
    return codes.view(F8[fmt]).float().double()


def quantize(x: torch.Tensor, scale: torch.Tensor, fmt: str) -> torch.Tensor:
    """Codes of x / scale (to nearest even, saturating, NaN kept); the quotient is exact for powers of two."""
    q = (x.double() / scale.double()).float()
    return q.clamp(-FMAX[fmt], FMAX[fmt]).to(F8[fmt]).view(torch.uint8)


def pow2_scale(amax: float, fmt: str) -> float:
    e = -126
    while amax > FMAX[fmt] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def ref_append(k, v, k_cache, v_cache, k_scale, v_scale, table, lens, cu, fmt):
    """The cache and scales after the append, page by page."""
    out = [t.clone() for t in (k_cache, v_cache, k_scale, v_scale)]
    pages, hk, ps, _ = k_cache.shape
    for x, cache, scale in ((k, out[0], out[2]), (v, out[1], out[3])):
        for b in range(table.shape[0]):
            n = cu[b + 1] - cu[b]
            start = lens[b] - n
            for pi in range(table.shape[1]):
                lo, hi = max(start, pi * ps, 0), min(lens[b], (pi + 1) * ps)
                page = int(table[b, pi])
                if lo >= hi or not 0 <= page < pages:
                    continue
                for h in range(hk):
                    rows = x[cu[b] + lo - start: cu[b] + hi - start, h].double()
                    fin = rows[torch.isfinite(rows)].abs()
                    need = pow2_scale(float(fin.max()) if fin.numel() else 0.0, fmt)
                    s = need
                    if lo > pi * ps:
                        old = float(scale[page, h])
                        s = max(old, need)
                        if s != old:
                            c = codes_to_f64(cache[page, h, : lo - pi * ps], fmt) * (old / s)
                            cache[page, h, : lo - pi * ps] = c.float().to(F8[fmt]).view(torch.uint8)
                    cache[page, h, lo - pi * ps: hi - pi * ps] = quantize(rows, torch.tensor(s), fmt).to(cache.device)
                    scale[page, h] = s
    return out


def ref_attention(q, k_cache, v_cache, k_scale, v_scale, table, lens, cu, scale, window, fmt):
    """(out, lse, bound): the result in 64 bits and how far a kernel may be from it.

    The bound: weights e^(s - max) are rounded to fp16 (2^-11 relative, 2^-25 of the largest weight * value scale
    where they fall below fp16's range), scores carry fp32 sums of head_dim products (2^-20 of the sum of their
    magnitudes, fp32 accumulation and the exponential), and the result is rounded once to its type."""
    pages, hk, ps, d = k_cache.shape
    t, hq, _ = q.shape
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    grp = hq // hk
    for b in range(table.shape[0]):
        n = cu[b + 1] - cu[b]
        ln = min(lens[b], table.shape[1] * ps)
        for i in range(n):
            tok = cu[b] + i
            pos = lens[b] - n + i
            j = torch.arange(max(0, pos - window + 1) if window else 0, max(0, min(pos + 1, ln)), device=q.device)
            if j.numel() == 0:
                continue
            pg = table[b].to(q.device)[j // ps].long()
            live = (pg >= 0) & (pg < pages)
            j, pg = j[live], pg[live]
            if j.numel() == 0:
                continue
            for h in range(hk):
                kk = codes_to_f64(k_cache[pg, h, j % ps], fmt) * k_scale[pg, h].double()[:, None]
                vv = codes_to_f64(v_cache[pg, h, j % ps], fmt) * v_scale[pg, h].double()[:, None]
                qq = q[tok, h * grp: (h + 1) * grp].double()
                s = qq @ kk.T * scale
                big = (qq.abs() @ kk.abs().T * abs(scale)).amax(1, keepdim=True)
                m = torch.logsumexp(s, 1, keepdim=True)
                p = torch.exp(s - m)
                o = p @ vv
                out[tok, h * grp: (h + 1) * grp] = o
                lse[tok, h * grp: (h + 1) * grp] = m[:, 0]
                mag = p @ vv.abs()
                top = (p * v_scale[pg, h].double()[None]).amax(1, keepdim=True) * FMAX[fmt]
                bound[tok, h * grp: (h + 1) * grp] = (
                    mag * (2.0 ** -11 + 2 * 2.0 ** -20 * big + 2.0 ** -18) + j.numel() * 2.0 ** -25 * top
                    + o.abs() * UNIT[q.dtype] + 2.0 ** -25)
    return out, lse, bound


def act64(x, act):
    if act == "silu":
        return x / (1 + torch.exp(-x))
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def ref_moe(x, router, wu, su, wd, sd, top_k, renorm, act, fmt):
    """(out, ids, weights, bound) in 64 bits.

    The bound: gate and up sums to 2^-18 of the sum of their terms' magnitudes (fp32 sums of exact products, and the
    activation's own rounding), the inner product rounded to fp16 (2^-11, or 2^-25 where it falls below fp16's normal
    range, the row having been scaled by a power of two for which the bound on |gate| |up|, the largest scales times
    fmax times sum |x|, lies between 2^13 and 2^15), the down sum to 2^-18, the result rounded once to its type."""
    t, hdim = x.shape
    inter = wd.shape[2]
    r = x.double() @ router.double().T
    ids = torch.sort(r, dim=1, descending=True, stable=True)[1][:, :top_k]
    w = r.gather(1, ids)
    w = torch.exp(w - torch.logsumexp(w if renorm else r, 1, keepdim=True))
    out = torch.zeros(t, hdim, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(out)
    for i in range(t):
        for s in range(top_k):
            e = int(ids[i, s])
            up = codes_to_f64(wu[e], fmt) * su[e].double()[:, None]
            dn = codes_to_f64(wd[e], fmt) * sd[e].double()[:, None]
            xi = x[i].double()
            gu, mag = up @ xi, up.abs() @ xi.abs()
            g, u = gu[:inter], gu[inter:]
            a = act64(g, act)
            h = a * u
            dh = 1.2 * 2.0 ** -18 * (mag[:inter] * u.abs() + a.abs() * mag[inter:] + mag[:inter] * mag[inter:] * 2.0 ** -18)
            most = su[e].double().view(2, -1).amax(1).prod() * (FMAX[fmt] * xi.abs().sum()) ** 2
            dh = dh + h.abs() * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -25 * 2.0 ** -13 * most
            out[i] += w[i, s] * (dn @ h)
            bound[i] += w[i, s] * (dn.abs() @ dh + 2.0 ** -18 * (dn.abs() @ h.abs()))
    bound += out.abs() * (UNIT[x.dtype] + 2.0 ** -18) + 2.0 ** -25
    return out, ids.to(torch.int32), w, bound


def ref_scores(logits, tokens, top, temperature):
    """(logprobs, entropy, top ids, top logprobs) in 64 bits; ties to the lowest index, NaN largest."""
    z = logits.double() / temperature
    bad = torch.isnan(z).any(1) | (z == math.inf).any(1) | (z == -math.inf).all(1)
    lp = z - torch.logsumexp(z, 1, keepdim=True)
    lp[bad] = math.nan
    p = lp.exp()
    ent = -torch.where(p == 0, 0.0, p * lp).sum(1)
    v = logits.shape[1]
    ok = (tokens >= 0) & (tokens < v)
    at = lp.gather(1, tokens.long().clamp(0, v - 1)[:, None])[:, 0]
    at = torch.where(ok, at, torch.nan)
    ids = torch.sort(logits.double(), dim=1, descending=True, stable=True)[1][:, :top]
    return at, ent, ids.to(torch.int32), lp.gather(1, ids)
