"""The few-token mixture-of-experts layer on the GPU, against 64 bits within the bound that its roundings give."""
import math

import pytest
import torch

import fp8imma_b200 as F
from serving_ref import ref_moe

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops(cuda):
    return F.ext()


def make(g, t, e, h, i, dtype, fmt, x_scale=1.0):
    ops = F.ext()
    w = []
    for n, k in ((2 * i, h), (h, i)):
        full = torch.randn(e * n, k, generator=g, device="cuda") * (1 / math.sqrt(k)) * torch.exp(0.5 * torch.randn(e * n, 1, generator=g, device="cuda"))
        codes, sigma, _ = ops.quantize_weights(full, fmt)
        w += [codes.view(e, n, k), sigma.view(e, n)]
    x = (torch.randn(t, h, generator=g, device="cuda") * x_scale).to(dtype)
    router = (torch.randn(e, h, generator=g, device="cuda") * (2 / math.sqrt(h))).to(dtype)
    return x, router, w[0], w[1], w[2], w[3]


def check(got, args, top_k, renorm, act, fmt):
    out, ids, wts = got
    o, i, w, bound = ref_moe(*args, top_k, renorm, act, fmt)
    assert torch.equal(ids, i)
    assert ((wts.double() - w).abs() <= 1e-5 * w + 1e-7).all()
    bound = bound + o.abs() * 1e-5 + (wts.double() - w).abs().amax() * 0
    err = (out.double() - o).abs()
    assert (err <= bound).all(), "worst %.3g of the bound" % float((err / bound).max())


CASES = [
    # tokens, experts, top_k, hidden, inter, renormalize, act
    (1, 4, 1, 16, 16, True, "silu"),
    (1, 64, 6, 512, 352, True, "silu"),
    (2, 8, 2, 1040, 144, False, "gelu"),
    (7, 8, 3, 256, 1040, True, "silu"),
    (8, 1, 1, 128, 128, False, "silu"),
    (9, 16, 4, 640, 208, True, "gelu"),
    (17, 3, 2, 384, 96, True, "silu"),
    (33, 40, 8, 144, 80, False, "silu"),
    (64, 2, 2, 256, 256, True, "silu"),
    (64, 100, 16, 128, 48, True, "gelu"),
    (5, 1024, 5, 64, 32, False, "silu"),
]


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_moe_matches_definition(ops, case, dtype, fmt):
    t, e, k, h, i, renorm, act = CASES[case]
    args = make(torch.Generator(device="cuda").manual_seed(case), t, e, h, i, dtype, fmt)
    check(ops.moe_forward(*args, k, renormalize=renorm, act=act, b_format=fmt), args, k, renorm, act, fmt)


def test_moe_ties_go_to_the_lowest_expert(ops):
    g = torch.Generator(device="cuda").manual_seed(20)
    args = make(g, 4, 12, 128, 64, torch.float16, "e4m3")
    args[1][:] = args[1][:1]  # every expert scores the same
    got = ops.moe_forward(*args, 5)
    assert torch.equal(got[1].cpu(), torch.arange(5, dtype=torch.int32).expand(4, 5))
    check(got, args, 5, True, "silu", "e4m3")


def test_moe_one_expert_takes_every_token(ops):
    g = torch.Generator(device="cuda").manual_seed(21)
    args = list(make(g, 64, 6, 256, 128, torch.bfloat16, "e4m3"))
    args[0] = args[0].abs()
    args[1] = torch.zeros_like(args[1])
    args[1][4] = 1.0
    got = ops.moe_forward(*args, 1)
    assert (got[1] == 4).all()
    check(got, args, 1, True, "silu", "e4m3")


@pytest.mark.parametrize("scale", [2.0 ** -20, 3000.0, 2.0 ** 30])
def test_moe_bf16_activations_outside_fp16(ops, scale):
    """Inputs and inner products far outside fp16's range: rows are brought into it by powers of two."""
    g = torch.Generator(device="cuda").manual_seed(22)
    args = list(make(g, 3, 4, 256, 256, torch.bfloat16, "e4m3", x_scale=scale))
    args[1] = (args[1].float() / scale).bfloat16()
    check(ops.moe_forward(*args, 2), args, 2, True, "silu", "e4m3")


def test_moe_strided_rows_zero_rows_and_streams(ops):
    g = torch.Generator(device="cuda").manual_seed(23)
    args = list(make(g, 6, 8, 320, 96, torch.float16, "e4m3"))
    wide = torch.randn(6, 700, generator=g, device="cuda").half()
    wide[2] = 0
    st = torch.cuda.Stream()
    for off in (0, 3, 320):
        args[0] = wide[:, off: off + 320]
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got = ops.moe_forward(*args, 3)
        torch.cuda.current_stream().wait_stream(st)
        check(got, args, 3, True, "silu", "e4m3")
        assert (got[0][2] == 0).all()


def test_moe_nan_stays_in_its_row(ops):
    g = torch.Generator(device="cuda").manual_seed(24)
    args = list(make(g, 9, 8, 128, 64, torch.bfloat16, "e4m3"))
    clean = ops.moe_forward(*args, 2)[0]
    args[0] = args[0].clone()
    args[0][4, 5] = math.nan
    out, ids, _ = ops.moe_forward(*args, 2)
    assert torch.isnan(out[4]).all() and ids[4].tolist() == [0, 1]
    keep = torch.arange(9, device="cuda") != 4
    assert not torch.isnan(out[keep]).any()
    assert ((out[keep].float() - clean[keep].float()).abs() <= 2.0 ** -7 * clean[keep].float().abs() + 1e-6).all()


def test_moe_repeats_bit_for_bit(ops):
    """Several calls, also on two streams at once and with another shape between them."""
    g = torch.Generator(device="cuda").manual_seed(25)
    args = make(g, 8, 16, 1024, 704, torch.bfloat16, "e4m3")
    other = make(g, 40, 5, 256, 128, torch.float16, "e5m2")
    first = ops.moe_forward(*args, 4)
    ops.moe_forward(*other, 2, b_format="e5m2")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for r in range(6):
        with torch.cuda.stream(streams[r % 2]):
            outs.append(ops.moe_forward(*args, 4))
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    assert F.lib().fp8imma_device_error(0) == 0


def test_moe_in_a_graph(ops):
    g = torch.Generator(device="cuda").manual_seed(26)
    args = list(make(g, 4, 8, 256, 128, torch.float16, "e4m3"))
    x = args[0]
    out = torch.empty_like(x)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        ops.moe_forward(*args, 2, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        _, ids, wts = ops.moe_forward(*args, 2, out=out)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda").half())
        graph.replay()
        torch.cuda.synchronize()
        check((out, ids, wts), args, 2, True, "silu", "e4m3")


@pytest.mark.parametrize("change, message", [
    (dict(top_k=0), "top_k must be"),
    (dict(top_k=5), "top_k must be"),
    (dict(act="relu"), "act must be"),
    (dict(b_format="int8"), "b_format must be"),
    (dict(x=lambda x: x.float()), "x must be fp16 or bf16"),
    (dict(x=lambda x: x.cpu()), "x must be a CUDA tensor"),
    (dict(x=lambda x: x.repeat(40, 1)), "at most 64 tokens"),
    (dict(router=lambda r: r.bfloat16()), "router must be"),
    (dict(router=lambda r: r[:3]), "w_gate_up must have shape"),
    (dict(w_gate_up=lambda w: w.float()), "uint8"),
    (dict(w_down=lambda w: w[..., :24].contiguous()), "w_gate_up must have shape"),
    (dict(s_down=lambda s: s[:, :-1].contiguous()), "one scale per weight row"),
    (dict(out=lambda o: torch.empty(2, 64, device="cuda")), "out must be"),
])
def test_moe_refuses(ops, change, message):
    x, router, wu, su, wd, sd = make(torch.Generator(device="cuda").manual_seed(27), 2, 4, 64, 32, torch.float16, "e4m3")
    args = dict(x=x, router=router, w_gate_up=wu, s_gate_up=su, w_down=wd, s_down=sd, top_k=2, act="silu", b_format="e4m3", out=None)
    for name, f in change.items():
        args[name] = f(args[name]) if callable(f) else f
    with pytest.raises(RuntimeError, match=message):
        ops.moe_forward(**args)


def test_moe_of_no_tokens(ops):
    x, *rest = make(torch.Generator(device="cuda").manual_seed(28), 2, 4, 64, 32, torch.float16, "e4m3")
    out, ids, wts = ops.moe_forward(x[:0], *rest, 2)
    assert out.shape == (0, 64) and ids.shape == (0, 2) and wts.shape == (0, 2)
