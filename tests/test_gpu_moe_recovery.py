"""The experts' layer after a wait between its CTAs that ran out: an error is reported, and the next call on the
same stream is right."""
import pytest
import torch

import fp8imma_b200 as F
from serving_ref import ref_moe
from test_gpu_moe import make

pytestmark = pytest.mark.gpu


def test_moe_after_a_barrier_that_ran_out(cuda):
    """One token of four million channels and one expert: a single warp makes the router's sum, for longer than the
    shortest limit (1 ms) that the other CTAs may be given for their wait."""
    ops, L = F.ext(), F.lib()
    g = torch.Generator(device="cuda").manual_seed(70)
    small = [make(g, 5, 8, 256, 128, torch.float16, "e4m3"), make(g, 40, 100, 128, 64, torch.bfloat16, "e4m3")]
    first = [ops.moe_forward(*a, 3) for a in small]
    h, i = 1 << 22, 16
    x = torch.randn(1, h, generator=g, device="cuda").half()
    router = torch.randn(1, h, generator=g, device="cuda").half()
    w_up = torch.randint(0, 64, (1, 2 * i, h), generator=g, device="cuda", dtype=torch.uint8)
    w_down = torch.randint(0, 64, (1, h, i), generator=g, device="cuda", dtype=torch.uint8)
    s_up, s_down = torch.full((1, 2 * i), 2.0 ** -12, device="cuda"), torch.full((1, h), 2.0 ** -12, device="cuda")
    torch.cuda.synchronize()
    assert L.fp8imma_device_error(1) == 0
    assert L.fp8imma_set_wait_limit_ns(1_000_000) == 0
    try:
        ops.moe_forward(x, router, w_up, s_up, w_down, s_down, 1)
        torch.cuda.synchronize()
    finally:
        assert L.fp8imma_set_wait_limit_ns(2_000_000_000) == 0
    assert L.fp8imma_device_error(1) == 6  # a CTA did not arrive in time
    for _ in range(2):
        for args, want in zip(small, first):
            got = ops.moe_forward(*args, 3)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert L.fp8imma_device_error(0) == 0
    out, ids, _, bound = ref_moe(*small[0], 3, True, "silu", "e4m3")
    assert torch.equal(first[0][1], ids) and ((first[0][0].double() - out).abs() <= bound + 1e-5 * out.abs()).all()
    # and the long call itself, given time
    got = ops.moe_forward(x, router, w_up, s_up, w_down, s_down, 1)
    torch.cuda.synchronize()
    assert L.fp8imma_device_error(0) == 0 and torch.isfinite(got[0]).all() and (got[1] == 0).all()
