"""residual_norm on the GPU where a CTA goes through several rounds of rows without copies ahead, with both norms and with
one: its sums over a row take turns in shared memory. Against 64 bits, and the same bits from every call."""
import pytest
import torch

import fp8imma_b200 as F
from test_gpu_residual_norm import B, H, S, check, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops(cuda):
    yield F.ext()
    assert F.lib().fp8imma_device_error(1) == 0


def same_each_time(ops, x, times=8):
    got = ops.residual_norm(**x)
    check(got, x)
    for _ in range(times):
        for a, b in zip(ops.residual_norm(**x), got):
            assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


NORMS = [(False, True), (True, False), (True, True)]


# rows past one round of the grid, below those from which they are copied ahead (on 148 SMs)
@pytest.mark.parametrize("t, h", [(2400, 512), (7100, 512), (300, 4096), (600, 4096), (880, 4096), (150, 8192), (400, 8192), (590, 8192),
                                  (150, 16384), (296, 16384), (1500, 1528), (700, 5000)])
@pytest.mark.parametrize("post, pre", NORMS)
@pytest.mark.parametrize("dt, res, gate", [(B, B, None), (H, S, "channel"), (H, None, "token")])
def test_rounds_without_copies_ahead(ops, t, h, post, pre, dt, res, gate):
    same_each_time(ops, inputs(t, t, h, dt, res=res, post=post, pre=pre, gate=gate))


@pytest.mark.parametrize("t, h", [(9000, 256), (2000, 4096), (900, 8192), (500, 16384)])
@pytest.mark.parametrize("post, pre", NORMS)
@pytest.mark.parametrize("w_type, gate", [(S, None), (S, "f32"), (None, "f32")])
def test_rounds_with_weights_or_gate_in_fp32(ops, t, h, post, pre, w_type, gate):
    same_each_time(ops, inputs(t, t, h, B, res=B, post=post, pre=pre, gate=gate, w_type=w_type))


@pytest.mark.parametrize("post, pre", NORMS)
def test_rows_too_wide_for_two_stages(ops, post, pre):
    same_each_time(ops, inputs(1, 700, 16384, H, res=S, post=post, pre=pre, gate="token"))


@pytest.mark.parametrize("post, pre", NORMS)
@pytest.mark.parametrize("t, h", [(20000, 512), (4000, 4096), (1300, 8192), (700, 16384)])
def test_rounds_with_copies_ahead(ops, t, h, post, pre):
    same_each_time(ops, inputs(t, t, h, B, res=B, post=post, pre=pre))
