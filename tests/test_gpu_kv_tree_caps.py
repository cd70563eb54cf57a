"""kv_attention_tree's capped scores on the GPU for caps of any size, on tiles that all rows see whole and on those at the
step, against 64 bits."""
import math

import pytest
import torch

from layer_ref import tree_mask
from serving_ref import FMAX, UNIT, codes_to_f64
from test_gpu_kv_cache import gen, i32, make_cache, offsets
from test_gpu_kv_tree import B, H, attend, ops, queries  # noqa: F401

pytestmark = pytest.mark.gpu


def define(q, cache, lens, cu, fmt, cap, scale, see):
    """(out, lse, bounds of both): see[b][i, j] says whether token i of the step sees key j.

    A score is off by 2^-20 of its products' magnitudes and the capped one by what that moves the tanh; besides by
    2^-20 of the row's largest capped score: 2^-21 of its own for the tanh (2^-21.8 for the polynomial, 2^-22 beyond
    it, tanh 1 being 0.76), and 2^-24 each for the value scale's logarithm and the reference, which are added to it.
    What a score is off by, its weight and lse are too."""
    table, kc, vc, ks, vs = cache
    t, hq, d = q.shape
    hk, ps = kc.shape[1], kc.shape[2]
    out = torch.zeros(t, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(t, hq, dtype=torch.float64, device="cuda")
    bound, dlse = torch.zeros_like(out), torch.zeros_like(lse)
    for b, ln in enumerate(lens):
        j = torch.arange(ln, device="cuda")
        pg = table[b].long()[j // ps]
        rows = slice(cu[b], cu[b + 1])
        for h in range(hq):
            g = h // (hq // hk)
            kk = codes_to_f64(kc[pg, g, j % ps], fmt) * ks[pg, g].double()[:, None]
            vv = codes_to_f64(vc[pg, g, j % ps], fmt) * vs[pg, g].double()[:, None]
            qq = q[rows, h].double()
            s, e = qq @ kk.T * scale, 2.0 ** -20 * abs(scale) * (qq.abs() @ kk.abs().T)
            off = cap * (torch.tanh((s + e) / cap) - torch.tanh((s - e) / cap))
            s = (cap * torch.tanh(s / cap)).masked_fill(~see[b], -math.inf)
            off = off.masked_fill(~see[b], 0.0).amax(1, keepdim=True) + 2.0 ** -20 * s.masked_fill(~see[b], 0.0).abs().amax(1, keepdim=True)
            m = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - m)
            out[rows, h], lse[rows, h] = p @ vv, m[:, 0]
            top = (p * vs[pg, g].double()[None]).amax(1, keepdim=True) * FMAX[fmt]
            bound[rows, h] = (p @ vv.abs()) * (2.0 ** -11 + torch.expm1(2 * off) + 2.0 ** -18) + ln * 2.0 ** -25 * top * torch.exp(off) + out[rows, h].abs() * UNIT[q.dtype] + 2.0 ** -25
            dlse[rows, h] = (off + 2.0 ** -18 + m.abs() * 2.0 ** -22)[:, 0]
    return out, lse, bound, dlse


def check(got, want):
    (out, lse), (ref, ref_lse, bound, dlse) = got, want
    assert bool(((lse.double() - ref_lse).abs() <= dlse).all()), float(((lse.double() - ref_lse).abs() / dlse).max())
    assert bool(((out.double() - ref).abs() <= bound).all()), float(((out.double() - ref).abs() / bound).max())


def bits(mask, n, ln):
    """The truth values [n, ln] of a sequence's mask rows; keys before the step are seen."""
    see = torch.ones(n, ln, dtype=torch.bool, device="cuda")
    for i in range(n):
        for j in range(n):
            see[i, ln - n + j] = bool(int(mask[i, j // 32]) >> (j % 32) & 1)
    return see


CAPS = [1e-38, 1e-4, 2e-3, 0.5, 50.0, 1100.0, 2000.0, 1e4, 1e6, 3e38]


@pytest.mark.parametrize("dt, fmt", [(H, "e4m3"), (B, "e5m2")])
@pytest.mark.parametrize("d", [64, 128, 256])
# scores beyond a cap of 3e38 are none
@pytest.mark.parametrize("cap, near", [(c, near) for c in CAPS for near in (False, True) if not (near and c > 1e6)])
def test_caps_of_any_size(ops, cap, near, d, dt, fmt):
    """Ordinary scores under any cap, and scores from far below the cap to four times it."""
    g = gen(d)
    lens, news = [400, 305, 140], [12, 3, 1]
    cache = make_cache(g, 3, 400 // 16 + 1, 2, 16, d, fmt)
    cu = offsets(news)
    q = queries(g, cu[-1], 8, d, dt)
    q *= torch.logspace(-3, 0, 8, base=10.0, device="cuda")[None, :, None].to(dt)  # heads of small and large scores
    scale = 1 / math.sqrt(d)
    if near:
        scale *= cap / 2.5  # products have a deviation of some 2 for the last heads
    parents = [-1, 0, 0, 1, 2, 3, 4, 5, 5, 5, 9, 10]
    mask = torch.cat([tree_mask(parents[:n], 1) for n in news]).cuda()
    see = [bits(mask[a:b], b - a, ln) for a, b, ln in zip(cu, cu[1:], lens)]
    a = dict(cap=cap, scale=scale)
    check(attend(ops, q, cache, lens, cu, fmt, mask=mask, **a), define(q, cache, lens, cu, fmt, cap, scale, see))
    see = [torch.arange(ln, device="cuda")[None] <= (ln - n + torch.arange(n, device="cuda"))[:, None] for ln, n in zip(lens, news)]
    check(attend(ops, q, cache, lens, cu, fmt, **a), define(q, cache, lens, cu, fmt, cap, scale, see))


@pytest.mark.parametrize("cap", [3e5, 1e30])
def test_a_cap_far_above_the_scores_is_none(ops, cap):
    g = gen(1)
    lens, news = [700, 260], [16, 9]
    cache = make_cache(g, 2, 700 // 32 + 1, 1, 32, 128, "e4m3")
    cu = offsets(news)
    q = queries(g, cu[-1], 8, 128, H)
    plain, capped = (attend(ops, q, cache, lens, cu, "e4m3", cap=c) for c in (0.0, cap))
    # scores of up to some 30, which the cap moves by s^3 / 3 cap^2 = 2^-23 at most: the same but for their 2^-20
    assert bool(((plain[1] - capped[1]).abs() <= 30 * 2.0 ** -20 + plain[1].abs() * 2.0 ** -22).all())


@pytest.mark.parametrize("d", [64, 128])
def test_products_of_zero_under_the_smallest_cap(ops, d):
    """Every score is 0, whatever the scales."""
    g = gen(2)
    table, kc, vc, ks, vs = cache = make_cache(g, 1, 300 // 16 + 1, 1, 16, d, "e4m3")
    kc.zero_()
    q = queries(g, 12, 4, d, B)
    out, lse = attend(ops, q, cache, [300], [0, 12], "e4m3", cap=1e-45, scale=1e6)
    want = torch.log(torch.arange(289, 301, device="cuda").double())[:, None].expand(12, 4)
    assert bool(((lse.double() - want).abs() <= 2.0 ** -18 + want * 2.0 ** -22).all())
    assert bool(torch.isfinite(out).all())
