"""Plain 64-bit restatements of the operators between the products (residual and
norms, adapters, rotation, tree attention), from their definitions, each with a
bound on what a kernel in 32 bits may be off by."""
from __future__ import annotations

import math

import torch

from serving_ref import FMAX, UNIT, codes_to_f64

UNIT8 = {"e4m3": 2.0 ** -4, "e5m2": 2.0 ** -3}       # half a step of a normal code, relative
STEP8 = {"e4m3": 2.0 ** -10, "e5m2": 2.0 ** -17}     # half the smallest step
HALF = UNIT | {torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -149}  # half the smallest step


def ref_residual_norm(y, residual, post, pre, gate, alpha, eps, offset, r_type):
    """((r, h), (bound of r, bound of h)); h is None without pre.

    A row's sum of squares passes at most 32 sums of a thread, 5 of a warp and 32 of the warps: 70 roundings, 2^-17.8
    relative, half of that after the root; with the quotients' and products' own 2^-24 each, a normed value is off by
    less than 2^-18 relative. h has its own norm's 2^-18 besides what its sums are off by."""
    def norm(x, w):
        return x / torch.sqrt(x.square().mean(1, keepdim=True) + eps) * (w.double() + offset)

    b = y.double() if post is None else norm(y.double(), post)
    b = alpha * b * (1.0 if gate is None else gate.double())
    r = b if residual is None else residual.double() + b
    dr = b.abs() * 2.0 ** -18 + r.abs() * 2.0 ** -24
    bound_r = dr + r.abs() * HALF[r_type] + TINY[r_type]
    if pre is None:
        return (r, None), (bound_r, None)
    h = norm(r, pre)
    f = (pre.double() + offset).abs() / torch.sqrt(r.square().mean(1, keepdim=True) + eps)
    off = torch.sqrt(dr.square().mean(1, keepdim=True)) / torch.sqrt(r.square().mean(1, keepdim=True) + eps)
    bound_h = f * dr + h.abs() * (off + 2.0 ** -18 + HALF[y.dtype]) + TINY[y.dtype]
    return (r, h), (bound_r, bound_h)


def ref_lora(base, x, a, b, ids, scales):
    """(out, bound). Sums of fp32 products to 2^-18 of their magnitudes; the inner sums as two 16-bit numbers to 2^-16
    of each (bf16: 2^-8 of 2^-8) or 2^-24 of a token's largest (fp16's smallest step); the result rounded once."""
    out = base.double().clone()
    bound = torch.zeros_like(out)
    for t in range(x.shape[0]):
        e = int(ids[t])
        if not 0 <= e < a.shape[0]:
            continue
        xe, ae, be = x[t].double(), a[e].double(), b[e].double()
        s = 1.0 if scales is None else float(scales[e])
        u = ae @ xe
        du = 2.0 ** -18 * (ae.abs() @ xe.abs()) + 2.0 ** -16 * u.abs() + 2.0 ** -24 * u.abs().max()
        d = s * (be @ u)
        out[t] += d
        bound[t] = abs(s) * (be.abs() @ du + 2.0 ** -18 * (be.abs() @ u.abs())) + 2.0 ** -23 * (d.abs() + base[t].double().abs())
        bound[t] += out[t].abs() * HALF[base.dtype] + TINY[base.dtype]
    return out, bound


def turn64(x, at, inv_freq, interleaved, scale=1.0):
    """x [tokens, heads, dim] in 64 bits, its first 2 * len(inv_freq) channels turned; and how large a pair is."""
    r = 2 * inv_freq.shape[0]
    y = x.double().clone()
    big = x.double().abs()
    angle = at.double()[:, None] * inv_freq.double()[None]
    c, s = (scale * torch.cos(angle))[:, None], (scale * torch.sin(angle))[:, None]
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    u, v = x[..., first].double(), x[..., second].double()
    y[..., first] = u * c - v * s
    y[..., second] = v * c + u * s
    big[..., first] = big[..., second] = abs(scale) * (u.abs() + v.abs())
    return y, big


def ref_tree(q, k_cache, v_cache, k_scale, v_scale, table, lens, cu, scale, window, fmt, cap=0.0, mask=None, positions=None):
    """(out, lse, bound of out, bound of lse): as serving_ref.ref_attention, over the keys that each token sees.

    Scores are off by 2^-20 of their products' magnitudes; capped ones besides by cap * 2^-20: of 1 - 2 / (1 + e^2y) the
    quotient is off by 2^-22 relative, doubled, the exponential by as much, which moves the quotient by half of it at
    most, and sum and difference by 2^-24. What a score is off by, its weight and lse are too."""
    pages, hk, ps, d = k_cache.shape
    t, hq, _ = q.shape
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device=q.device)
    bound, dlse = torch.zeros_like(out), torch.zeros_like(lse)
    grp = hq // hk
    for b in range(table.shape[0]):
        n = cu[b + 1] - cu[b]
        start = lens[b] - n
        ln = max(0, min(lens[b], table.shape[1] * ps))
        j = torch.arange(ln, device=q.device)
        for i in range(n):
            tok = cu[b] + i
            pos = start + i
            if mask is None:
                see = j <= pos
                if window:
                    see &= j > pos - window
            else:
                if positions is not None:
                    pos = min(max(int(positions[tok]), start), lens[b] - 1)
                see = j < start
                if window:
                    see &= j > pos - window
                row = mask[tok].tolist()
                bits = [(row[x // 32] >> (x % 32)) & 1 if x // 32 < len(row) else 0 for x in range(n)]
                bits = torch.tensor(bits, dtype=torch.bool, device=q.device)
                see |= (j >= start) & bits[(j - start).clamp(0, n - 1)]
            jj = j[see]
            if jj.numel() == 0:
                continue
            pg = table[b].to(q.device)[jj // ps].long()
            live = (pg >= 0) & (pg < pages)
            jj, pg = jj[live], pg[live]
            if jj.numel() == 0:
                continue
            for h in range(hk):
                kk = codes_to_f64(k_cache[pg, h, jj % ps], fmt) * k_scale[pg, h].double()[:, None]
                vv = codes_to_f64(v_cache[pg, h, jj % ps], fmt) * v_scale[pg, h].double()[:, None]
                qq = q[tok, h * grp: (h + 1) * grp].double()
                s = qq @ kk.T * scale
                off = 2.0 ** -20 * (qq.abs() @ kk.abs().T * abs(scale)).amax(1, keepdim=True)
                if cap:
                    s = cap * torch.tanh(s / cap)
                    off = off.clamp_max(2 * cap) + cap * 2.0 ** -20
                m = torch.logsumexp(s, 1, keepdim=True)
                p = torch.exp(s - m)
                at = (tok, slice(h * grp, (h + 1) * grp))
                out[at] = p @ vv
                lse[at] = m[:, 0]
                mag = p @ vv.abs()
                top = (p * v_scale[pg, h].double()[None]).amax(1, keepdim=True) * FMAX[fmt]
                bound[at] = mag * (2.0 ** -11 + 2 * off + 2.0 ** -18) + jj.numel() * 2.0 ** -25 * top + out[at].abs() * UNIT[q.dtype] + 2.0 ** -25
                dlse[at] = (off + 2.0 ** -18 + m.abs() * 2.0 ** -22)[:, 0]
    return out, lse, bound, dlse


def tree_mask(parents, words=None):
    """[tokens, words] int32 bits of each node's ancestors and itself; parents: index within the sequence, -1 for a root."""
    n = len(parents)
    words = words or max(1, -(-n // 32))
    rows = []
    for i, p in enumerate(parents):
        bits = (rows[p] if p >= 0 else 0) | (1 << i)
        rows.append(bits)
    out = torch.zeros(n, words, dtype=torch.int64)
    for i, bits in enumerate(rows):
        for w in range(words):
            out[i, w] = (bits >> (32 * w)) & 0xFFFFFFFF
    return torch.where(out >= 2 ** 31, out - 2 ** 32, out).to(torch.int32)
