"""Scoring of logits on the GPU (log probabilities, entropy, top alternatives), against 64 bits."""
import math

import pytest
import torch

import fp8imma_b200 as F
from serving_ref import ref_scores

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops(cuda):
    return F.ext()


def check(got, logits, tokens, top, temperature):
    """fp32 results: the scaled logit is rounded once (2^-24 of it), the sum of exponentials is good to 2^-19 of
    itself (fp32 sums, the exponential's own error and that of its argument), the entropy adds the logits' spread
    times that."""
    lp, ent, ids, tlp = got
    a, e, i, t = ref_scores(logits, tokens, top, temperature)
    z = logits.double().abs() / temperature
    big = torch.where(torch.isfinite(z), z, 0.0).amax(1)
    tol = 2.0 ** -19 + 2.0 ** -22 * big
    etol = 2.0 ** -18 * (1 + math.log(logits.shape[1]) + 2.0 ** -4 * big)
    assert torch.equal(ids, i)

    def near(x, y, tol):
        same = (x.double() == y) | (torch.isnan(x) & torch.isnan(y))
        assert torch.equal(torch.isnan(x), torch.isnan(y))
        bad = ~same & ~((x.double() - y).abs() <= tol)
        assert not bad.any(), "worst %.3g" % float((x.double() - y).abs()[bad].max())

    near(lp, a, tol)
    near(ent, e, etol)
    near(tlp, t, tol[:, None])


def make(g, t, v, dtype, layout, sigma=2.5):
    x = (torch.randn(t, v, generator=g, device="cuda") * sigma).to(dtype)
    return x.t().contiguous().t() if layout == "col" else x


SIZES = [(1, 1, 1), (1, 7, 3), (3, 33, 32), (2, 1000, 0), (5, 4097, 5), (1, 32000, 8), (1, 200001, 32), (16, 50257, 20), (300, 515, 1), (17, 128000, 4)]


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", range(len(SIZES)))
def test_scores_match_definition(ops, size, dtype, layout):
    t, v, top = SIZES[size]
    g = torch.Generator(device="cuda").manual_seed(size)
    x = make(g, t, v, dtype, layout)
    tok = torch.randint(0, v, (t,), generator=g, device="cuda", dtype=torch.int32)
    for temperature in (1.0, 0.6):
        check(ops.token_logprobs(x, tok, top=top, temperature=temperature), x, tok, top, temperature)


@pytest.mark.parametrize("layout", ["row", "col"])
def test_scores_of_masked_rows(ops, layout):
    """-inf logits take no part; a row with one logit left is certain of it; a row with none, with NaN or with +inf
    has no probabilities; token ids outside the vocabulary have none."""
    g = torch.Generator(device="cuda").manual_seed(30)
    v = 5003
    x = make(g, 9, v, torch.bfloat16, "row")
    x[0, torch.rand(v, generator=g, device="cuda") < 0.9] = -math.inf
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, 77] = 3.0
    x[3, 4000] = math.nan
    x[4, 10] = math.inf
    x[5] = torch.finfo(torch.bfloat16).min
    x[6] = torch.finfo(torch.bfloat16).min
    x[6, v - 1] = -2.0
    x[7, 1:] = -math.inf
    x = x.t().contiguous().t() if layout == "col" else x
    tok = torch.tensor([5, 0, 77, 1, 10, 3, v - 1, 0, v], dtype=torch.int32, device="cuda")
    check(ops.token_logprobs(x, tok, top=12), x, tok, 12, 1.0)
    tok[:] = -1
    assert torch.isnan(ops.token_logprobs(x, tok)[0]).all()


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("v", [50, 3000, 70000])
def test_scores_ties_go_to_the_lowest_index(ops, v, layout):
    """Logits with few distinct values, equal ones everywhere, and +-0."""
    g = torch.Generator(device="cuda").manual_seed(31)
    x = torch.randint(0, 3, (4, v), generator=g, device="cuda").half()
    x[1] = 1.5
    x[2] = -0.0
    x[2, 1::2] = 0.0
    x[3] = torch.arange(v, device="cuda").half().clamp_max(2000)  # rising: each new maximum comes last
    x = x.t().contiguous().t() if layout == "col" else x
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    check(ops.token_logprobs(x, tok, top=32), x, tok, 32, 1.0)


def test_scores_of_large_logits_and_low_temperature(ops):
    g = torch.Generator(device="cuda").manual_seed(32)
    x = make(g, 6, 9001, torch.float32, "row", sigma=3000.0)
    x[2] += 1e6
    tok = torch.randint(0, 9001, (6,), generator=g, device="cuda", dtype=torch.int32)
    for temperature in (1.0, 50.0):
        check(ops.token_logprobs(x, tok, top=5, temperature=temperature), x, tok, 5, temperature)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_scores_of_strided_rows(ops, dtype):
    """Rows (or columns) inside a wider buffer, at offsets of every alignment, on another stream."""
    g = torch.Generator(device="cuda").manual_seed(33)
    wide = torch.randn(8, 3011, generator=g, device="cuda").to(dtype)
    st = torch.cuda.Stream()
    for off in (0, 1, 3, 8):
        for x in (wide[:, off: off + 3000], wide.t()[off: off + 3000].t(), wide.t()[off: off + 40]):
            tok = torch.zeros(x.shape[0], dtype=torch.int32, device="cuda")
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got = ops.token_logprobs(x, tok, top=3)
            torch.cuda.current_stream().wait_stream(st)
            check(got, x, tok, 3, 1.0)


def test_scores_repeat_bit_for_bit(ops):
    g = torch.Generator(device="cuda").manual_seed(34)
    x = make(g, 2, 128000, torch.bfloat16, "row")
    tok = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    first = ops.token_logprobs(x, tok, top=20)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for r in range(6):
        with torch.cuda.stream(streams[r % 2]):
            outs.append(ops.token_logprobs(x, tok, top=20))
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_scores_in_a_graph(ops):
    g = torch.Generator(device="cuda").manual_seed(35)
    x = make(g, 3, 60001, torch.float16, "row")
    tok = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        ops.token_logprobs(x, tok, top=6)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        got = ops.token_logprobs(x, tok, top=6)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda").half())
        graph.replay()
        torch.cuda.synchronize()
        check(got, x, tok, 6, 1.0)


def test_scores_of_32_bit_offsets(ops):
    """More than 2^31 logits."""
    t, v = 17000, 131072
    x = torch.full((t, v), -1.0, dtype=torch.float16, device="cuda")
    tok = torch.full((t,), v - 1, dtype=torch.int32, device="cuda")
    x[t - 1, v - 1] = 4.0
    lp, ent, ids, tlp = ops.token_logprobs(x, tok, top=2)
    want = ref_scores(x[-2:], tok[-2:], 2, 1.0)
    assert ids[-1].tolist() == [v - 1, 0] and ids[0].tolist() == [0, 1]
    assert ((lp[-2:].double() - want[0]).abs() <= 2.0 ** -18).all()


@pytest.mark.parametrize("change, message", [
    (dict(top=33), "top must be"), (dict(top=-1), "top must be"), (dict(top=20), "top must be"),
    (dict(temperature=0.0), "temperature must be"), (dict(temperature=math.inf), "temperature must be"),
    (dict(logits=lambda x: x.double()), "fp16, bf16 or fp32"),
    (dict(logits=lambda x: x.cpu()), "logits must be a CUDA tensor"),
    (dict(logits=lambda x: x[0]), "logits must have shape"),
    (dict(logits=lambda x: torch.zeros(4, 64, device="cuda")[:, ::4]), "contiguous along one dimension"),
    (dict(tokens=lambda t: t.long()), "tokens must be"),
    (dict(tokens=lambda t: t[:2]), "tokens must have shape"),
])
def test_scores_refuse(ops, change, message):
    args = dict(logits=torch.randn(4, 16, device="cuda"), tokens=torch.zeros(4, dtype=torch.int32, device="cuda"), top=2, temperature=1.0)
    for name, f in change.items():
        args[name] = f(args[name]) if callable(f) else f
    with pytest.raises(RuntimeError, match=message):
        ops.token_logprobs(**args)


def test_scores_of_no_tokens(ops):
    got = ops.token_logprobs(torch.empty(0, 16, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), top=2)
    assert got[0].shape == (0,) and got[2].shape == (0, 2)
