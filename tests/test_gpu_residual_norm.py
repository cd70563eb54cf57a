"""residual_norm on the GPU against 64 bits, within the bound that its roundings give."""
import pytest
import torch

import fp8imma_b200 as F
from layer_ref import ref_residual_norm

pytestmark = pytest.mark.gpu

H, B, S = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture
def ops(cuda):
    return F.ext()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def inputs(seed, t, h, dt, res=None, post=True, pre=True, gate=None, w_type=None, pad=0, offset=0.0):
    g = gen(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    w_type = w_type or dt
    y = (randn(t, h + pad) * torch.exp(randn(t, 1))).to(dt)[:, :h]
    return dict(y=y, residual=None if res is None else (3 * randn(t, h)).to(res),
                post_weight=(1 - offset + 0.2 * randn(h)).to(w_type) if post else None,
                pre_weight=(1 - offset + 0.2 * randn(h)).to(w_type) if pre else None,
                gate={None: None, "channel": randn(h).to(dt), "token": randn(t, h + pad).to(dt)[:, :h], "f32": randn(h)}[gate])


def check(got, x, alpha=1.0, eps=1e-6, offset=0.0):
    r_type = x["y"].dtype if x["residual"] is None else x["residual"].dtype
    want, bound = ref_residual_norm(x["y"], x["residual"], x["post_weight"], x["pre_weight"], x["gate"], alpha, eps, offset, r_type)
    assert got[0].dtype == r_type
    for a, w, b in zip(got, want, bound):
        assert (a is None) == (w is None)
        if w is not None:
            off = (a.double() - w).abs()
            assert bool((off <= b).all()), float((off / b).max())


@pytest.mark.parametrize("t, h", [(1, 1), (3, 7), (1, 8), (5, 64), (2, 255), (9, 256), (300, 1000), (1, 2048), (33, 2049), (7, 4096), (3, 5121),
                                  (2, 16384), (2, 16392), (1, 32768), (2, 32767)])
@pytest.mark.parametrize("dt", [H, B])
def test_sizes(ops, t, h, dt):
    x = inputs(h, t, h, dt, res=dt, gate="token")
    check(ops.residual_norm(**x), x)


@pytest.mark.parametrize("dt", [H, B])
@pytest.mark.parametrize("res", ["own", "f32", None])
@pytest.mark.parametrize("post, pre", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("gate", [None, "channel", "token", "f32"])
@pytest.mark.parametrize("h, pad", [(512, 0), (512, 8), (514, 3)])
def test_forms(ops, dt, res, post, pre, gate, h, pad):
    x = inputs(1, 6, h, dt, res={"own": dt, "f32": S, None: None}[res], post=post, pre=pre, gate=gate, pad=pad, offset=1.0)
    check(ops.residual_norm(**x, alpha=0.3, eps=1e-5, weight_offset=1.0), x, 0.3, 1e-5, 1.0)


def test_fp32_weights_and_residual_without_one(ops):
    x = inputs(2, 4, 640, B, w_type=S)
    check(ops.residual_norm(**x), x)
    out = torch.empty(4, 640, device="cuda")
    got = ops.residual_norm(**x, residual_out=out)
    assert got[0].data_ptr() == out.data_ptr()
    want, bound = ref_residual_norm(*(x[k] for k in ("y", "residual", "post_weight", "pre_weight", "gate")), 1.0, 1e-6, 0.0, S)
    assert bool(((out.double() - want[0]).abs() <= bound[0]).all())


@pytest.mark.parametrize("t, h", [(9601, 64), (20000, 8), (5000, 1000), (1301, 4096), (701, 8192), (450, 16384)])
@pytest.mark.parametrize("dt, res, gate, pad", [(B, B, "token", 8), (H, S, "channel", 0), (B, None, None, 0), (H, H, "f32", 16)])
def test_many_rows(ops, t, h, dt, res, gate, pad):
    """Several rounds of rows for each CTA, copied ahead."""
    x = inputs(t, t, h, dt, res=res, gate=gate, pad=pad)
    got = ops.residual_norm(**x)
    check(got, x)
    if res is not None:  # and in place
        r2, _ = ops.residual_norm(**x, residual_out=x["residual"])
        assert torch.equal(r2, got[0])
    assert F.lib().fp8imma_device_error(1) == 0


@pytest.mark.parametrize("h", [512, 515])
def test_in_place_is_the_same(ops, h):
    x = inputs(3, 50, h, H, res=H, gate="channel")
    r, o = ops.residual_norm(**x)
    y, res = x["y"].clone(), x["residual"].clone()
    r2, o2 = ops.residual_norm(y, res, x["post_weight"], x["pre_weight"], x["gate"], residual_out=res, out=y)
    assert r2.data_ptr() == res.data_ptr() and o2.data_ptr() == y.data_ptr()
    assert torch.equal(r, res) and torch.equal(o, y)


def test_zero_rows_and_values_out_of_range(ops):
    x = inputs(4, 6, 256, B, res=B)
    x["y"][0] = 0
    x["residual"][0] = 0
    x["y"][1, 3] = float("nan")
    x["y"][2, 5] = float("inf")
    x["residual"][3, 7] = float("-inf")
    r, h = ops.residual_norm(**x)
    assert bool((r[0] == 0).all()) and bool((h[0] == 0).all())
    assert bool(torch.isnan(r[1]).all()) and bool(torch.isnan(h[1]).all())  # the row's norm is NaN
    assert bool(torch.isnan(r[2, 5])) and bool(torch.isnan(h[2]).all())     # inf / inf there, 0 elsewhere
    assert r[3, 7] == float("-inf") and bool(torch.isnan(h[3, 7]))
    y = {k: None if v is None else v[4:] if v.dim() == 2 else v for k, v in x.items()}
    check((r[4:], h[4:]), y)


def test_large_sums_stay_in_range(ops):
    x = inputs(5, 3, 4096, B, res=B)
    x["y"] = (x["y"].float() * 2.0 ** 40).to(B)
    check(ops.residual_norm(**x), x)


def test_graph_stream_and_repeat(ops):
    x = inputs(6, 64, 1024, H, res=S, gate="token")
    want = ops.residual_norm(**x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.residual_norm(**x)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.residual_norm(**x)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_empty(ops):
    r, h = ops.residual_norm(torch.empty(0, 64, dtype=H, device="cuda"), pre_weight=torch.ones(64, dtype=H, device="cuda"))
    assert r.shape == h.shape == (0, 64)


@pytest.mark.parametrize("change, message", [
    (dict(y=torch.float32), "y must be fp16 or bf16"), (dict(residual=torch.bfloat16), "residual must have y's dtype or fp32"),
    (dict(residual=(4, 63)), "shaped like y"), (dict(gate=(4, 3)), "gate must"), (dict(gate=(63,)), "gate must"),
    (dict(post_weight=(63,)), r"shape \[hidden\]"), (dict(post_weight=torch.float32), "same dtype"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(alpha=float("inf")), "finite")])
def test_refuses(ops, change, message):
    x = dict(inputs(7, 4, 64, H, res=H, gate="token"))
    for k, v in change.items():
        x[k] = x[k].to(v) if isinstance(v, torch.dtype) else torch.zeros(v, dtype=H, device="cuda") if isinstance(v, tuple) else v
    if change.get("gate") == (4, 3):
        message = "shaped like y"
    with pytest.raises(RuntimeError, match=message):
        ops.residual_norm(**x)


def test_refuses_overlap_and_strides(ops):
    x = inputs(8, 4, 64, H, res=H)
    buf = torch.zeros(5, 64, dtype=H, device="cuda")
    with pytest.raises(RuntimeError, match="apart"):
        ops.residual_norm(buf[:4], out=buf[1:], pre_weight=x["pre_weight"])
    with pytest.raises(RuntimeError, match="apart"):
        ops.residual_norm(x["y"], out=buf[:4], residual_out=buf[:4], pre_weight=x["pre_weight"])
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.residual_norm(torch.zeros(64, 4, dtype=H, device="cuda").t())
    with pytest.raises(RuntimeError, match="pre_weight only"):
        ops.residual_norm(x["y"], out=buf[:4])
    with pytest.raises(RuntimeError, match="hidden must be"):
        ops.residual_norm(torch.zeros(1, 32769, dtype=H, device="cuda"))
