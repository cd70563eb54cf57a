"""Values in the cache that are no numbers."""
import pytest
import torch

import fp8imma_b200 as F
from serving_ref import F8
from test_gpu_kv_cache import gen, i32, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[1 << 20, 1], ids=["mma", "tcgen05"])
def ops(cuda, request):
    L = F.lib()
    assert L.fp8imma_set_attention_tc_rows(request.param) == 0
    yield F.ext()
    L.fp8imma_set_attention_tc_rows(0)
    assert L.fp8imma_device_error(1) == 0


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("length", [20, 128, 150])  # in a tile that ends early, in a whole one, in the first of two
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_nan_that_a_row_sees_with_the_least_weight(ops, d, length, fmt):
    """A key whose weight is below fp32's range still has a weight: a NaN of its values reaches the row, and only in
    its channels."""
    g = gen(d + length)
    hk, ps = 2, 16
    table, kc, vc, ks, vs = make_cache(g, 1, 10, hk, ps, d, fmt)
    kc.zero_()
    page = int(table[0, 0])
    kc[page, :, 3] = torch.tensor(-4.0, device="cuda").to(F8[fmt]).view(torch.uint8)  # score -4 d, the others' is 0
    ks.fill_(1.0)
    vc[page, 1, 3, 5::16] = 0x7F
    q = torch.ones(1, 8, d, device="cuda").half()
    out, lse = ops.kv_attention(q, kc, vc, ks, vs, table, i32([length]), softmax_scale=1.0, fmt=fmt)
    want = torch.zeros(8, d, dtype=torch.bool, device="cuda")
    want[4:, 5::16] = True
    assert torch.equal(torch.isnan(out[0]), want) and torch.isfinite(lse).all()
