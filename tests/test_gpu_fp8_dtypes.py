"""Caches and weights whose dtype names an FP8 format: taken when it is the one asked for, refused when it is not."""
import pytest
import torch

import fp8imma_b200 as F
from test_gpu_kv_cache import gen, i32, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops(cuda):
    return F.ext()


def test_a_cache_of_the_other_format_is_refused(ops):
    g = gen(90)
    table, kc, vc, ks, vs = make_cache(g, 2, 2, 2, 16, 64, "e5m2")
    q = torch.randn(2, 4, 64, generator=g, device="cuda").half()
    ln = i32([3, 30])
    f8 = [x.view(torch.float8_e5m2) for x in (kc, vc)]
    bytes_out, _ = ops.kv_attention(q, kc, vc, ks, vs, table, ln, fmt="e5m2")
    typed_out, _ = ops.kv_attention(q, *f8, ks, vs, table, ln, fmt="e5m2")
    assert torch.equal(bytes_out, typed_out)
    for call in (lambda a, b: ops.kv_attention(q, a, b, ks, vs, table, ln),
                 lambda a, b: ops.kv_append(q[:, :2], q[:, :2], a, b, ks, vs, table, ln)):
        for a, b in ((f8[0], f8[1]), (kc, f8[1]), (f8[0], vc)):
            with pytest.raises(RuntimeError, match="float8_e5m2|Float8_e5m2"):
                call(a, b)


def test_weights_of_the_other_format_are_refused(ops):
    x = torch.randn(2, 64, device="cuda").half()
    router = torch.randn(4, 64, device="cuda").half()
    wu, wd = torch.zeros(4, 64, 64, dtype=torch.float8_e5m2, device="cuda"), torch.zeros(4, 64, 32, dtype=torch.float8_e5m2, device="cuda")
    su, sd = torch.ones(4, 64, device="cuda"), torch.ones(4, 64, device="cuda")
    ops.moe_forward(x, router, wu, su, wd, sd, 2, b_format="e5m2")
    with pytest.raises(RuntimeError, match="float8_e5m2|Float8_e5m2"):
        ops.moe_forward(x, router, wu, su, wd, sd, 2)
