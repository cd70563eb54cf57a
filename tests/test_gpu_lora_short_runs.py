"""lora_add on the GPU with short runs among many tokens: units of one to three tokens in the kernel for long runs (which
takes all of them above 1024 tokens), and on both sides of the mean length by which the ids choose below."""
import pytest
import torch

import fp8imma_b200 as F
from layer_ref import ref_lora
from test_gpu_lora import B, H, check, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops(cuda):
    yield F.ext()
    assert F.lib().fp8imma_device_error(1) == 0


@pytest.mark.parametrize("length", [1, 2, 3])
@pytest.mark.parametrize("k, n, r", [(264, 90, 40), (72, 333, 104), (520, 64, 128), (128, 200, 8), (96, 1000, 64)])
@pytest.mark.parametrize("dt, base_dt, col", [(B, H, True), (H, H, False), (B, B, False), (H, B, True)])
def test_short_runs_above_1024_tokens(ops, length, k, n, r, dt, base_dt, col):
    t = 1029
    x = inputs(k + n, [i // length % 6 - 1 for i in range(t)], k, n, r, 5, dt, base_dt, col)
    check(ops.lora_add(**x), x)


@pytest.mark.parametrize("t", [150, 1100])
@pytest.mark.parametrize("col", [False, True])
def test_one_prompt_beside_single_requests(ops, t, col):
    """A mean length that belongs to neither."""
    ids = [1] * (t - 60) + [i % 7 - 1 for i in range(60)]
    x = inputs(t, ids, 136, 210, 32, 6, B, H, col)
    check(ops.lora_add(**x), x)


@pytest.mark.parametrize("length", [1, 3])
@pytest.mark.parametrize("n", [96, 75])
@pytest.mark.parametrize("col", [False, True])
def test_in_place_above_1024_tokens(ops, length, n, col):
    t = 1027
    ids = [i // length % 4 - 1 for i in range(t)]
    x = inputs(n, ids, 80, n, 24, 3, H, B, col)
    want, bound = ref_lora(x["base"], x["x"], x["lora_a"], x["lora_b"], ids, x["scales"])
    before = x["base"].clone()
    got = ops.lora_add(**x, out=x["base"])
    assert got.data_ptr() == x["base"].data_ptr()
    assert bool(((got.double() - want).abs() <= bound).all())
    none = [i for i, e in enumerate(ids) if e < 0]
    assert torch.equal(got[none], before[none])
