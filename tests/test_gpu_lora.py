"""lora_add on the GPU against 64 bits, within the bound that its roundings give."""
import pytest
import torch

import fp8imma_b200 as F
from layer_ref import ref_lora

pytestmark = pytest.mark.gpu

H, B = torch.float16, torch.bfloat16


@pytest.fixture
def ops(cuda):
    yield F.ext()
    assert F.lib().fp8imma_device_error(1) == 0


def inputs(seed, ids, k, n, r, adapters, dt, base_dt, col=False, scales=True, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    t = len(ids)
    base = randn(t, n).to(base_dt)
    return dict(base=base.t().contiguous().t() if col else base, x=randn(t, k + pad).to(dt)[:, :k], lora_a=(randn(adapters, r, k) / k ** 0.5).to(dt),
                lora_b=(randn(adapters, n, r) / r ** 0.5).to(dt), adapter_ids=torch.tensor(ids, dtype=torch.int32, device="cuda"),
                scales=0.5 + torch.rand(adapters, generator=g, device="cuda") if scales else None)


def check(got, x, layout=True):
    want, bound = ref_lora(x["base"], x["x"], x["lora_a"], x["lora_b"], x["adapter_ids"].tolist(), x["scales"])
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    if layout and got.numel() > got.shape[0] > 1:
        assert got.stride() == x["base"].stride()


def runs(*lengths, ids):
    return [i for n, i in zip(lengths, ids) for _ in range(n)]


# up to 128 tokens go through one kernel, more through the other
IDS = {
    "one": [2],
    "own": list(range(7)) + [-1, 3, 3, 99, 0],
    "runs": runs(9, 3, 1, 20, 30, ids=[1, 0, -1, 2, 2]),
    "full": [1] * 128,
    "many": runs(1, 63, 64, 65, 3, 7, 100, ids=[0, 1, 2, 3, -5, 1, 0]),
    "many own": [i % 5 for i in range(131)],
    "many none": [-1] * 140,
}
WIDTHS = {"one": 3, "own": 7, "runs": 3, "full": 2, "many": 4, "many own": 5, "many none": 1}


@pytest.mark.parametrize("name", list(IDS))
@pytest.mark.parametrize("k, n, r", [(8, 1, 8), (256, 64, 16), (520, 333, 24), (1320, 100, 32), (128, 1000, 40), (2048, 512, 64), (96, 72, 128), (264, 31, 104)])
@pytest.mark.parametrize("dt, base_dt, col", [(B, H, True), (H, H, False), (B, B, False), (H, B, True)])
def test_matches_definition(ops, name, k, n, r, dt, base_dt, col):
    x = inputs(k + n + r, IDS[name], k, n, r, WIDTHS[name], dt, base_dt, col, scales=n % 2 == 0, pad=8 * (k % 3))
    check(ops.lora_add(**x), x)


@pytest.mark.parametrize("t", [129, 600, 1024, 1025])
@pytest.mark.parametrize("length", [1, 3, 4, 5, 90])
@pytest.mark.parametrize("col", [False, True])
def test_runs_of_any_length(ops, t, length, col):
    """Whichever kernel the runs' length chooses, to the border of the range where the ids choose."""
    x = inputs(t + length, [i // length % 4 - 1 for i in range(t)], 72, 90, 16, 3, B, H, col)
    check(ops.lora_add(**x), x)


@pytest.mark.parametrize("t", [1, 60, 128, 129, 200])
@pytest.mark.parametrize("col", [False, True])
def test_in_place_strided_base_and_tokens_without_adapter(ops, t, col):
    ids = [(i // 11) % 4 - 1 for i in range(t)]
    x = inputs(t, ids, 136, 50, 16, 3, B, H)
    # a slice of a wider result: the neighbours stay as they are
    wide = torch.randn(*((200, t) if col else (t, 200)), device="cuda").to(H)
    before = wide.clone()
    view = (wide[64:114].t() if col else wide[:, 64:114])
    x["base"] = view
    want = ref_lora(before[64:114].t() if col else before[:, 64:114], x["x"], x["lora_a"], x["lora_b"], ids, x["scales"])
    got = ops.lora_add(**x, out=view)
    assert got.data_ptr() == view.data_ptr()
    assert bool(((got.double() - want[0]).abs() <= want[1]).all())
    none = [i for i, e in enumerate(ids) if e < 0]
    w, b = (wide.t(), before.t()) if col else (wide, before)
    assert torch.equal(w[:, :64], b[:, :64]) and torch.equal(w[:, 114:], b[:, 114:])
    assert torch.equal(w[none], b[none])


@pytest.mark.parametrize("t", [5, 150])
@pytest.mark.parametrize("dt", [H, B])
@pytest.mark.parametrize("mult", [2.0 ** -12, 2.0 ** 12])
def test_inner_sums_outside_the_type(ops, t, dt, mult):
    """x * A far above fp16's largest number or below its smallest: the sums keep their precision."""
    x = inputs(1, [i % 2 for i in range(t)], 512, 96, 16, 2, dt, dt)
    x["lora_a"] = (x["lora_a"].float() * mult).to(dt)
    x["x"] = (x["x"].float() * (8.0 if mult > 1 else 1.0)).to(dt)
    x["scales"] = x["scales"] / mult
    check(ops.lora_add(**x), x)


@pytest.mark.parametrize("t", [9, 140])
@pytest.mark.parametrize("dt", [H, B])
def test_a_base_that_cancels(ops, t, dt):
    x = inputs(2, [0] * t, 256, 64, 32, 1, dt, dt, scales=False)
    x["base"] = (-ref_lora(torch.zeros_like(x["base"]), x["x"], x["lora_a"], x["lora_b"], [0] * t, None)[0]).to(dt)
    check(ops.lora_add(**x), x)


@pytest.mark.parametrize("t", [12, 150])
@pytest.mark.parametrize("dt", [H, B])
def test_nan_and_infinity_stay_in_their_row(ops, t, dt):
    x = inputs(3, [i // 5 % 3 for i in range(t)], 256, 80, 16, 3, dt, dt)
    clean = ops.lora_add(**x)
    x["x"][4, 7] = float("nan")
    x["x"][9, 0] = float("inf")
    x["lora_a"][2, :, 3] = float("nan")
    x["lora_b"][2, 5] = float("inf")
    got = ops.lora_add(**x)
    assert not torch.isfinite(got[4]).any() and not torch.isfinite(got[9]).any()
    for i in range(t):
        if i not in (4, 9) and i // 5 % 3 != 2:
            assert torch.equal(got[i], clean[i])


def test_more_tokens_than_one_launch_takes(ops):
    t = 16384 + 70
    x = inputs(4, [i // 97 % 4 - 1 for i in range(t)], 64, 40, 8, 3, H, H)
    got = ops.lora_add(**x)
    ids = x["adapter_ids"].long()
    d = torch.zeros(t, 40, dtype=torch.float64, device="cuda")
    for e in range(3):
        at = ids == e
        d[at] = (x["x"][at].double() @ x["lora_a"][e].double().t()) @ x["lora_b"][e].double().t() * x["scales"][e].double()
    want = x["base"].double() + d
    # result rounded once; sums to 2^-16 of |B| |A| |x|, at most rank * in_features of terms below 40 here
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -10).all())


@pytest.mark.parametrize("t", [33, 300])
def test_graph_stream_and_repeat(ops, t):
    x = inputs(5, [i // 20 % 3 for i in range(t)], 1024, 1000, 16, 3, B, H, col=True)
    want = ops.lora_add(**x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.lora_add(**x) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(want, y) for y in got)
    # two graphs captured on one stream, replayed at once on two
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.lora_add(**x))
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(want, y) for y in outs)


def test_empty(ops):
    x = inputs(6, [0], 64, 40, 8, 1, H, H)
    x |= dict(base=x["base"][:0], x=x["x"][:0], adapter_ids=x["adapter_ids"][:0])
    assert ops.lora_add(**x).shape == (0, 40)


@pytest.mark.parametrize("change, message", [
    (dict(x=torch.float32), "x must be fp16 or bf16"), (dict(base=torch.float32), "base must be fp16 or bf16"), (dict(lora_a=torch.bfloat16), "lora_a must be"),
    (dict(lora_b=(2, 40, 8)), "lora_b must have shape"), (dict(lora_a=(2, 16, 72)), "lora_a must have shape"), (dict(adapter_ids=torch.int64), "adapter_ids must be"),
    (dict(base=(4, 39)), "base must have shape"), (dict(scales=(3,)), "scales must have shape"),
    (dict(lora_a=(2, 12, 64), lora_b=(2, 40, 12)), "rank must be"), (dict(lora_a=(2, 136, 64), lora_b=(2, 40, 136)), "rank must be"),
    (dict(x=(4, 60), lora_a=(2, 16, 60)), "in_features must be")])
def test_refuses(ops, change, message):
    x = inputs(7, [0, 1, 1, 0], 64, 40, 16, 2, H, H)
    for k, v in change.items():
        x[k] = x[k].to(v) if isinstance(v, torch.dtype) else torch.zeros(v, dtype=torch.float32 if k == "scales" else H, device="cuda")
    with pytest.raises(RuntimeError, match=message):
        ops.lora_add(**x)


def test_refuses_layouts(ops):
    x = inputs(8, [0, 1, 1, 0], 64, 40, 16, 2, H, H)
    with pytest.raises(RuntimeError, match="same dimension"):
        ops.lora_add(**x, out=torch.zeros(40, 4, dtype=H, device="cuda").t())
    with pytest.raises(RuntimeError, match="contiguous along one"):
        ops.lora_add(**(x | dict(base=torch.zeros(4, 80, dtype=H, device="cuda")[:, ::2])))
    with pytest.raises(RuntimeError, match="contiguous along one"):  # rows that lie on one another
        ops.lora_add(**(x | dict(base=torch.zeros(1, 40, dtype=H, device="cuda").expand(4, 40))))
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        ops.lora_add(**(x | dict(x=torch.zeros(4, 68, dtype=H, device="cuda")[:, :64])))
    big = torch.zeros(5, 40, dtype=H, device="cuda")
    with pytest.raises(RuntimeError, match="apart"):
        ops.lora_add(**(x | dict(base=big[:4])), out=big[1:])
