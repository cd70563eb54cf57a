"""Offsets of a step's tokens that do not ascend: an error is set and nothing is written, by the append and by both
attention kernels; offsets that leave tokens out are followed."""
import pytest
import torch

import fp8imma_b200 as F
from test_gpu_kv_cache import gen, i32, make_cache

pytestmark = pytest.mark.gpu

BAD_OFFSETS = 7
DESCENDING = {
    "overlap": [0, 5, 3, 8],
    "first": [4, 2, 6, 8],
    "last": [0, 4, 8, 7],
    "late": [min(b, 650) for b in range(700)] + [649],  # more sequences than a CTA looks at in one go
}


@pytest.fixture(params=[1 << 20, 1], ids=["mma", "tcgen05"])
def ops(cuda, request):
    L = F.lib()
    assert L.fp8imma_set_attention_tc_rows(request.param) == 0
    assert L.fp8imma_device_error(1) == 0
    yield F.ext()
    L.fp8imma_set_attention_tc_rows(0)
    assert L.fp8imma_device_error(1) == 0


@pytest.mark.parametrize("name", DESCENDING)
def test_descending_offsets(ops, name):
    cu = DESCENDING[name]
    b, t, hk, d, ps, fmt = len(cu) - 1, max(cu), 2, 64, 16, "e4m3"
    g = gen(80)
    table, kc, vc, ks, vs = make_cache(g, b, 2, hk, ps, d, fmt)
    lens = i32([20] * b)
    kv = torch.randn(t, hk, d, generator=g, device="cuda").half()
    before = [x.clone() for x in (kc, vc, ks, vs)]
    ops.kv_append(kv, kv, kc, vc, ks, vs, table, lens, i32(cu), fmt)
    assert F.lib().fp8imma_device_error(1) == BAD_OFFSETS
    assert all(torch.equal(x, y) for x, y in zip((kc, vc, ks, vs), before))
    out = torch.full((t, 4, d), 3.0, dtype=torch.float16, device="cuda")
    q = torch.randn(t, 4, d, generator=g, device="cuda").half()
    ops.kv_attention(q, kc, vc, ks, vs, table, lens, i32(cu), fmt=fmt, out=out)
    assert F.lib().fp8imma_device_error(1) == BAD_OFFSETS
    assert (out == 3.0).all()
    # the next call is served
    good = i32([t * k // b for k in range(b + 1)])
    got, _ = ops.kv_attention(q, kc, vc, ks, vs, table, lens, good, fmt=fmt)
    again, _ = ops.kv_attention(q, kc, vc, ks, vs, table, lens, good, fmt=fmt)
    assert torch.equal(got, again) and torch.isfinite(got).all()


def test_offsets_that_leave_tokens_out(ops):
    g = gen(81)
    b, t, hk, d, ps, fmt = 3, 12, 1, 128, 32, "e5m2"
    table, kc, vc, ks, vs = make_cache(g, b, 2, hk, ps, d, fmt)
    lens, cu = i32([20, 33, 64]), i32([2, 5, 5, 9])
    q = torch.randn(t, 4, d, generator=g, device="cuda").half()
    out = torch.full((t, 4, d), 3.0, dtype=torch.float16, device="cuda")
    ops.kv_attention(q, kc, vc, ks, vs, table, lens, cu, fmt=fmt, out=out)
    part = ops.kv_attention(q[2:9].contiguous(), kc, vc, ks, vs, table, lens, i32([0, 3, 3, 7]), fmt=fmt)[0]
    assert torch.equal(out[2:9], part) and (out[:2] == 3.0).all() and (out[9:] == 3.0).all()
