"""Scores of logits masked by finite values, and of logits far from zero: what counts is the distance from the row's
largest, however large the numbers are."""
import math

import pytest
import torch

import fp8imma_b200 as F

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops(cuda):
    return F.ext()


def reference(x, tokens, top, temperature):
    """Log probabilities, entropy, top ids and their log probabilities, and each logit's distance from the row's
    largest, which is taken in 64 bits before anything else: 1e30 and its logarithm do not fit one number."""
    d = (x.double() - x.double().amax(1, keepdim=True)) / temperature
    lp = d - torch.log(torch.exp(d).sum(1, keepdim=True))
    p = lp.exp()
    ent = -torch.where(p == 0, 0.0, p * lp).sum(1)
    ids = torch.sort(x.double(), dim=1, descending=True, stable=True)[1][:, :top]
    return lp.gather(1, tokens.long()[:, None])[:, 0], ent, ids.to(torch.int32), lp.gather(1, ids), d


def check(ops, x, tokens, top, temperature):
    """fp32 results: the distance from the row's reference and its product with 1 / temperature are rounded (2^-22 of
    the distance in all), the sum of exponentials is good to 2^-18 of itself (the exponential's own error and that of
    an argument of up to 25 binary orders), and the entropy, a mean of such distances, to 2^-17 (1 + log vocab)."""
    lp, ent, ids, tlp = ops.token_logprobs(x, tokens, top=top, temperature=temperature)
    a, e, i, t, d = reference(x, tokens, top, temperature)
    assert torch.equal(ids, i)

    def near(got, want, tol):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        same = (got == want.float()) | torch.isnan(got)
        assert (same | ((got.double() - want).abs() <= tol)).all(), "worst %.3g" % float((got.double() - want).abs()[~same].max())

    near(lp, a, 2.0 ** -18 + 2.0 ** -22 * d.gather(1, tokens.long()[:, None])[:, 0].abs())
    near(ent, e, torch.full_like(e, 2.0 ** -17 * (1 + math.log(x.shape[1]))))
    near(tlp, t, 2.0 ** -18 + 2.0 ** -22 * d.gather(1, i.long()).abs())


def masked(g, v, dtype, mask):
    x = torch.randn(7, v, generator=g, device="cuda") * 2.5
    x[0, torch.rand(v, generator=g, device="cuda") < 0.5] = mask
    x[1, 40:] = mask                   # most lanes see masked logits only
    x[2, : v - 40] = mask
    x[3] = mask                        # all masked: every token as likely as the others
    x[4], x[4, v // 2] = mask, 1.0     # one left
    x[5, ::2] = mask
    x[5, 1::4] = -math.inf             # both kinds
    return x.to(dtype)


MASKS = [(torch.float32, m) for m in (-1e9, -1e10, -1e12, -1e30, torch.finfo(torch.float32).min)] + \
        [(torch.bfloat16, m) for m in (-1e9, -1e10, -1e12, -1e30, torch.finfo(torch.bfloat16).min)] + \
        [(torch.float16, m) for m in (-1e4, torch.finfo(torch.float16).min)]


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("dtype, mask", MASKS)
@pytest.mark.parametrize("v", [61, 5003, 66001])
def test_finite_masks(ops, v, dtype, mask, layout):
    x = masked(torch.Generator(device="cuda").manual_seed(v), v, dtype, mask)
    tok = x.argmax(1).to(torch.int32)
    tok[0], tok[3], tok[6] = int((x[0] == x[0].min()).nonzero()[0, 0]), v - 1, 5
    x = x.t().contiguous().t() if layout == "col" else x
    for temperature in (0.05, 0.2, 0.48, 0.6, 1.0, 1.05, 1.5):
        check(ops, x, tok, 20, temperature)


@pytest.mark.parametrize("layout", ["row", "col"])
def test_many_rows_of_finite_masks(ops, layout):
    """Enough rows for one part and one warp a row."""
    g = torch.Generator(device="cuda").manual_seed(9)
    x = masked(g, 2003, torch.float32, -1e9).repeat(700, 1)
    tok = torch.zeros(x.shape[0], dtype=torch.int32, device="cuda")
    x = x.t().contiguous().t() if layout == "col" else x
    for temperature in (0.2, 0.63, 1.0):
        check(ops, x, tok, 5, temperature)


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("at", [1e6, 2.0 ** 30, -(2.0 ** 33), 1e30])
def test_logits_far_from_zero(ops, at, layout):
    """Rows that lie far from zero as a whole: neighbouring numbers there are the only other logits."""
    g = torch.Generator(device="cuda").manual_seed(10)
    step = 2.0 ** (math.frexp(at)[1] - 24)
    x = (at + step * torch.randint(0, 4, (5, 4099), generator=g, device="cuda").double()).float()
    x[1, 100:] = -1e9
    x[2, :4000] = torch.finfo(torch.float32).min
    x[3, 17] = -math.inf
    tok = torch.tensor([0, 5, 4050, 18, 4098], dtype=torch.int32, device="cuda")
    x = x.t().contiguous().t() if layout == "col" else x
    for temperature in (1.0, 0.3, 100.0):
        check(ops, x, tok, 8, temperature)
