"""kv_append_rope's cosines and sines where they are small: they keep their relative precision, as the 64-bit angle's do."""
import pytest
import torch

import fp8imma_b200 as F
from layer_ref import TINY
from serving_ref import UNIT
from test_gpu_kv_cache import gen, i32, make_cache
from test_gpu_kv_rope import B, H, freqs

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops(cuda):
    yield F.ext()
    assert F.lib().fp8imma_device_error(1) == 0


def near_quarter_turns(f, most):
    """The positions below `most` whose angle lies nearest to a quarter turn, 16 for each of the first frequencies."""
    p = torch.arange(most, device="cuda", dtype=torch.float64)
    out = []
    for i in range(6):
        a = p[1:] * f[i].double()
        out += (1 + torch.minimum(torch.cos(a).abs(), torch.sin(a).abs()).topk(16, largest=False)[1]).tolist()
    return out


@pytest.mark.parametrize("dt", [H, B])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("theta", [10000.0, 500000.0])
@pytest.mark.parametrize("sign", [1, -1])
def test_angles_near_quarter_turns(ops, theta, interleaved, dt, sign):
    """A position and a frequency multiply exactly in 64 bits (20 and 24 bits), so the reference's angle is exact. The
    kernel's fraction of a turn is off by 2^-50, its angle by 2^-47; cosine and sine come out of sincospif, off by 2^-22
    relative, and the first-order term of what the fraction lost as fp32 (2^-23.3, its square is 2^-47), rounded once
    more. With a second channel of 0 the product is one more rounding: 2^-21 relative and 2^-45 of x in all."""
    f = freqs(64, theta)
    pos = [sign * p for p in near_quarter_turns(f, 1 << 20)]
    t = len(pos)
    g = gen(0)
    table, kc, vc, ks, vs = make_cache(g, 1, -(-t // 16), 1, 16, 64, "e4m3")
    x = 2.0 ** 15
    q = torch.zeros(t, 1, 64, dtype=dt, device="cuda")
    first, second = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    q[..., first] = x
    k = torch.zeros(t, 1, 64, dtype=dt, device="cuda")
    out = ops.kv_append_rope(q, k, k, kc, vc, ks, vs, table, i32([t]), f, positions=i32(pos), interleaved=interleaved)
    a = torch.tensor(pos, dtype=torch.float64, device="cuda")[:, None] * f.double()[None]
    for part, want in ((first, x * torch.cos(a)), (second, x * torch.sin(a))):
        off = (out[:, 0, part].double() - want).abs()
        bound = want.abs() * (UNIT[dt] + 2.0 ** -21) + x * 2.0 ** -45 + TINY[dt]
        assert bool((off <= bound).all()), float((off / bound).max())
