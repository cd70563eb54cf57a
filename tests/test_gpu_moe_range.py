"""The inner product of the experts' layer, act(g) * u, over the range that weights and scales give it: rows of weights
that do not fill their format's range, rows of zeros with a large scale, single rows far larger than the others. What
the result may be off by is measured by the sizes of the inner products themselves."""
import math

import pytest
import torch

import fp8imma_b200 as F
from serving_ref import F8, UNIT, act64, codes_to_f64

pytestmark = pytest.mark.gpu

H, I = 320, 208


@pytest.fixture
def ops(cuda):
    return F.ext()


def layer(g, t, e, dtype, h=H, i=I):
    """Activations, router and the weights in fp32."""
    x = torch.randn(t, h, generator=g, device="cuda").to(dtype)
    router = (torch.randn(e, h, generator=g, device="cuda") * (2 / math.sqrt(h))).to(dtype)
    up = torch.randn(e, 2 * i, h, generator=g, device="cuda") / math.sqrt(h)
    down = torch.randn(e, h, i, generator=g, device="cuda") / math.sqrt(i)
    return x, router, up, down


def quantize(ops, w, fmt):
    codes, sigma, _ = ops.quantize_weights(w.reshape(-1, w.shape[2]), fmt)
    return codes.view(w.shape), sigma.view(w.shape[:2]).clone()


def direct(w, fmt):
    return w.to(F8[fmt]).view(torch.uint8), torch.ones(w.shape[:2], device="cuda")


def check(ops, x, router, up, down, k, act, fmt, tells=True):
    """Against 64 bits with the kernel's own weights of the experts. Gate and up sums are good to 2^-18 of the sum of
    their terms' magnitudes (fp32 sums, and the activation's rounding); h is rounded to fp16 (2^-11) beside columns
    that are brought to the row's largest (2^-24 of that); the down sum is good to 2^-18 of its terms' magnitudes; the
    result is rounded once."""
    (wu, su), (wd, sd) = up, down
    out, ids, wts = ops.moe_forward(x, router, wu, su, wd, sd, k, act=act, b_format=fmt)
    want, bound = torch.zeros_like(out, dtype=torch.float64), torch.zeros_like(out, dtype=torch.float64)
    for t in range(x.shape[0]):
        for s in range(k):
            e, w = int(ids[t, s]), float(wts[t, s])
            a, b = codes_to_f64(wu[e], fmt) * su[e].double()[:, None], codes_to_f64(wd[e], fmt) * sd[e].double()[:, None]
            xi = x[t].double()
            gu, mag = a @ xi, a.abs() @ xi.abs()
            n = b.shape[1]
            act_g, u = act64(gu[:n], act), gu[n:]
            h = act_g * u
            dh = 1.2 * 2.0 ** -18 * (mag[:n] * u.abs() + act_g.abs() * mag[n:] + mag[:n] * mag[n:] * 2.0 ** -18)
            dh = dh + h.abs() * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -24 * h.abs().max()
            want[t] += w * (b @ h)
            bound[t] += w * (b.abs() @ dh + 2.0 ** -18 * (b.abs() @ h.abs()))
    # the smallest step of fp16 results; bf16 has fp32's range
    bound += want.abs() * (UNIT[x.dtype] + 2.0 ** -18) + (2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -134)
    err = (out.double() - want).abs()
    assert (err <= bound).all(), "worst %.3g of the bound" % float((err / bound).max())
    # the bound itself is a small part of the result, so that it can tell
    assert not tells or bound.norm() <= 0.02 * want.norm()


TOKENS = [1, 9, 40]  # the three forms of the kernel


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t", TOKENS)
def test_weights_cast_without_a_scale(ops, t, dtype, fmt):
    x, router, up, down = layer(torch.Generator(device="cuda").manual_seed(t), t, 6, dtype)
    check(ops, x, router, direct(up, fmt), direct(down, fmt), 2, "silu", fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("t", TOKENS)
@pytest.mark.parametrize("scale", [1.0, 1e9])
def test_rows_of_zeros_with_a_large_scale(ops, t, fmt, scale):
    """Gate and up rows that were added to fill the width."""
    x, router, up, down = layer(torch.Generator(device="cuda").manual_seed(t + 1), t, 5, torch.bfloat16)
    (wu, su), dn = quantize(ops, up, fmt), quantize(ops, down, fmt)
    for part in (slice(I - 40, I), slice(2 * I - 40, 2 * I)):
        wu[:, part], su[:, part] = 0, scale
    check(ops, x, router, (wu, su), dn, 3, "gelu", fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("t", TOKENS)
@pytest.mark.parametrize("factor", [2.0 ** 10, 2.0 ** 20])
@pytest.mark.parametrize("silent", [True, False])
def test_one_channel_far_larger(ops, t, fmt, factor, silent):
    """A gate and an up row far larger than the others, with inputs that leave them silent, and with inputs that do
    not: the other channels keep their bits in the one case, and their part of the largest in the other."""
    x, router, up, down = layer(torch.Generator(device="cuda").manual_seed(t + 2), t, 5, torch.bfloat16)
    x[:, 250:] = 0
    for row in (37, I + 37):
        up[:, row] *= factor
        if silent:
            up[:, row, :250] = 0
    # a large negative gate sum of the only token: its h is 0, but the bound counts the sum
    check(ops, x, router, quantize(ops, up, fmt), quantize(ops, down, fmt), 2, "silu", fmt, tells=silent or t > 1)


@pytest.mark.parametrize("t", TOKENS)
@pytest.mark.parametrize("mult", [2.0 ** -24, 2.0 ** 24])
def test_columns_of_every_size(ops, t, mult):
    """Inner products that grow by powers of two along the row, and whole rows far from 1."""
    x, router, up, down = layer(torch.Generator(device="cuda").manual_seed(t + 3), t, 4, torch.bfloat16)
    up[:, :I] *= torch.exp2(-torch.arange(I, device="cuda") % 23.0)[:, None]
    x = (x.float() * mult).bfloat16()
    check(ops, x, (router.float() / mult).bfloat16(), quantize(ops, up, "e4m3"), quantize(ops, down, "e4m3"), 2, "silu", "e4m3")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("t", TOKENS)
def test_rows_that_stay_zero(ops, t, act):
    """A token whose inner products are all zero gives zeros beside tokens that do not."""
    x, router, up, down = layer(torch.Generator(device="cuda").manual_seed(t + 4), t, 4, torch.float16)
    up[:, I:, 100:] = 0
    x[0, :100] = 0
    out = ops.moe_forward(x, router, *quantize(ops, up, "e5m2"), *quantize(ops, down, "e5m2"), 2, act=act, b_format="e5m2")[0]
    assert (out[0] == 0).all() and torch.isfinite(out).all()
    if t > 1:
        assert (out[1:] != 0).any(1).all()
