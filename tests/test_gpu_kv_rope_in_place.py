"""kv_append_rope with q_out as q: which slices of one buffer it takes, with the results of a call with its own output, and
the refusal of rows that lie on one another."""
import pytest
import torch

import fp8imma_b200 as F
from test_gpu_kv_cache import gen, i32, make_cache
from test_gpu_kv_rope import H, freqs

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops(cuda):
    yield F.ext()
    assert F.lib().fp8imma_device_error(1) == 0


def parts(kind, t, dim=64):
    """q, k, v: parts of one buffer."""
    g = gen(len(kind) + t)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(H)  # noqa: E731
    if kind == "rows":  # [tokens, heads + 2 kv heads, dim]
        return randn(t, 8, dim).split((4, 2, 2), 1)
    if kind == "v first":
        v, k, q = randn(t, 8, dim).split((2, 2, 4), 1)
        return q, k, v
    if kind == "heads in turn":  # [tokens, kv heads, 3, dim]
        return randn(t, 2, 3, dim).unbind(2)
    if kind == "heads first":  # [heads, tokens, dim]
        return [x.transpose(0, 1) for x in randn(8, t, dim).split((4, 2, 2), 0)]
    if kind == "channels in turn":  # [tokens, heads, 3 dim]: heads of q, k and v side by side
        return randn(t, 2, 3 * dim).split(dim, 2)
    return randn(t, 4, dim), randn(t, 2, dim), randn(t, 2, dim)  # "apart"


@pytest.mark.parametrize("kind", ["rows", "v first", "heads in turn", "heads first", "channels in turn", "apart"])
@pytest.mark.parametrize("t", [1, 2, 33])
def test_slices_of_one_buffer(ops, kind, t):
    q, k, v = parts(kind, t)
    cache = make_cache(gen(t), 1, 4, 2, 16, 64, "e4m3")[1:]
    again = [x.clone() for x in cache]
    table, lens, f = i32([[3, 0, 1, 2]]), i32([t + 5]), freqs(64)
    want = ops.kv_append_rope(q, k, v, *again, table, lens, f)
    kept = [k.clone(), v.clone()]
    got = ops.kv_append_rope(q, k, v, *cache, table, lens, f, q_out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    assert all(torch.equal(x, y) for x, y in zip(cache, again)) and torch.equal(k, kept[0]) and torch.equal(v, kept[1])


def overlaps(t, dim=64):
    qkv = torch.zeros(t, 8, dim, dtype=H, device="cuda")
    flat = torch.zeros(t * 8 * dim + 64 * dim, dtype=H, device="cuda")
    k, v = torch.zeros(t, 2, dim, dtype=H, device="cuda"), torch.zeros(t, 2, dim, dtype=H, device="cuda")
    at = lambda sizes, strides, off=0: flat.as_strided(sizes, strides, off)  # noqa: E731
    yield "q is k", qkv[:, :2], qkv[:, :2], v
    yield "q is v", qkv[:, :2], k, qkv[:, :2]
    yield "a head in common", qkv[:, :4], qkv[:, 3:5], qkv[:, 6:]
    yield "an element in common", at((t, 4, dim), (8 * dim, dim, 1)), at((t, 2, dim), (8 * dim, dim, 1), 4 * dim - 1), v
    yield "one head for all", qkv[:, :1].expand(t, 4, dim), k, v
    yield "rows half over one another", at((t, 4, dim), (8 * dim, dim // 2, 1)), k, v
    if t > 1:
        yield "the next token's head", at((t, 4, dim), (8 * dim, dim, 1)), at((t, 2, dim), (8 * dim, dim, 1), 8 * dim), v
        yield "one token for all", qkv[:1, :4].expand(t, 4, dim), k, v
        yield "other strides in one buffer", at((t, 4, dim), (8 * dim, dim, 1)), at((t, 2, dim), (6 * dim, dim, 1), 4 * dim), v
        yield "tokens half over one another", at((t, 1, dim), (dim // 2, dim, 1)), k, v


@pytest.mark.parametrize("t", [1, 2, 9])
def test_refuses_rows_that_lie_on_one_another(ops, t):
    table, kc, vc, ks, vs = make_cache(gen(0), 1, 2, 2, 16, 64, "e4m3")
    before = [x.clone() for x in (kc, vc, ks, vs)]
    for name, q, k, v in overlaps(t):
        with pytest.raises(RuntimeError, match="apart"):
            ops.kv_append_rope(q, k, v, kc, vc, ks, vs, table, i32([t]), freqs(64), q_out=q)
            pytest.fail(name)
    assert all(torch.equal(x, y) for x, y in zip(before, (kc, vc, ks, vs)))
