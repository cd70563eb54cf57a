"""Which of the two attention kernels a call takes by itself. They differ in the last bits, so the one taken shows."""
import pytest
import torch

import fp8imma_b200 as F
from test_gpu_kv_cache import gen, i32, make_cache

pytestmark = pytest.mark.gpu

FEW_ROWS, TCGEN05 = 1 << 20, 1  # settings that force one of them


@pytest.fixture
def ops(cuda):
    yield F.ext()
    F.lib().fp8imma_set_attention_tc_rows(0)


@pytest.mark.parametrize("batch, keys, new, heads, kv_heads, dim, window, taken", [
    (16, 4000, 4, 32, 8, 128, 0, FEW_ROWS),    # 16 rows a KV head, however many tiles
    (16, 4000, 5, 32, 8, 128, 0, TCGEN05),     # 20 rows, 28 tiles an SM
    (8, 2000, 5, 32, 8, 128, 0, FEW_ROWS),     # 7 tiles an SM
    (16, 1000, 5, 64, 8, 128, 0, TCGEN05),     # 40 rows, 7 tiles an SM
    (1, 1000, 5, 64, 8, 128, 0, FEW_ROWS),     # less than one
    (16, 4000, 5, 64, 8, 128, 100, TCGEN05),   # a window leaves two tiles a sequence and head: 1.7 an SM
    (8, 4000, 5, 64, 8, 128, 100, FEW_ROWS),
    (16, 4000, 4, 28, 4, 64, 0, FEW_ROWS),     # 28 rows of 64 channels
    (16, 4000, 5, 28, 4, 64, 0, TCGEN05),      # 35 rows, 14 tiles an SM
    (16, 1000, 5, 28, 4, 64, 0, FEW_ROWS),     # 3.5
    (16, 1000, 16, 28, 4, 64, 0, TCGEN05),     # 112 rows
])
def test_the_kernel_that_is_taken(ops, batch, keys, new, heads, kv_heads, dim, window, taken):
    g = gen(keys + new)
    ps = 64
    table, kc, vc, ks, vs = make_cache(g, batch, -(-keys // ps), kv_heads, ps, dim, "e4m3")
    q = torch.randn(batch * new, heads, dim, generator=g, device="cuda").half()
    out = {}
    for rows in (0, FEW_ROWS, TCGEN05):
        assert F.lib().fp8imma_set_attention_tc_rows(rows) == 0
        out[rows] = ops.kv_attention(q, kc, vc, ks, vs, table, i32([keys] * batch), None, window=window)[0]
    assert not torch.equal(out[FEW_ROWS], out[TCGEN05])
    assert torch.equal(out[0], out[taken])
