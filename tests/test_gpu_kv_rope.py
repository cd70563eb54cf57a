"""kv_append_rope on the GPU: the cache against kv_append's definition on keys turned in 64 bits, queries within the
bound that their rounding gives."""
import pytest
import torch

import fp8imma_b200 as F
from layer_ref import STEP8, TINY, UNIT8, turn64
from serving_ref import F8, UNIT, codes_to_f64, ref_append
from test_gpu_kv_cache import gen, i32, make_cache, offsets

pytestmark = pytest.mark.gpu

H, B = torch.float16, torch.bfloat16


@pytest.fixture
def ops(cuda):
    yield F.ext()
    assert F.lib().fp8imma_device_error(1) == 0


def freqs(rotary, theta=10000.0):
    return (theta ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)).float()


def places(lens, news):
    return i32([ln - n + i for ln, n in zip(lens, news) for i in range(n)])


def check_cache(got, want, key_big, at, fmt, scale_floor):
    """got, want: (codes, scale) of keys; at: (page, slot, token) of each stored row. Codes of stored rows may differ where
    the key's 32-bit value (off by 2^-21 of the pair) lies at a border between two codes, all others are equal."""
    (gc, gs), (wc, ws), values = got, want, scale_floor
    assert torch.equal(gs, ws)
    same = gc == wc
    for page, slot, tok in at:
        v = codes_to_f64(gc[page, :, slot], fmt) * gs[page].double()[:, None]
        off = (v - values[tok]).abs()
        bound = UNIT8[fmt] * values[tok].abs() + STEP8[fmt] * gs[page].double()[:, None] + 2.0 ** -21 * key_big[tok]
        assert bool((off <= bound).all()), float((off / bound).max())
        same[page, :, slot] = True
    assert bool(same.all())


def run(ops, seed, lens, news, heads, hk, d, ps, rotary, interleaved, dt, fmt, positions=None, scale=1.0, cu_none=False, theta=10000.0, q_in_place=False):
    g = gen(seed)
    width = max(1, -(-max(lens) // ps))
    table, kc, vc, ks, vs = make_cache(g, len(lens), width, hk, ps, d, fmt)
    cu = offsets(news)
    qkv = (torch.randn(cu[-1], heads + 2 * hk, d, generator=g, device="cuda") * torch.exp(torch.randn(cu[-1], 1, 1, generator=g, device="cuda"))).to(dt)
    q, k, v = qkv[:, :heads], qkv[:, heads: heads + hk], qkv[:, heads + hk:]
    f = freqs(rotary, theta)
    at = places(lens, news) if positions is None else positions
    turned, big = turn64(k, at, f, interleaved, scale)
    want_q, big_q = turn64(q, at, f, interleaved, scale)
    want = ref_append(turned.cpu(), v.cpu(), kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), table.cpu(), lens, cu, fmt)
    v_before, k_before = v.clone(), k.clone()
    out = ops.kv_append_rope(q, k, v, kc, vc, ks, vs, table, i32(lens), f, None if cu_none else i32(cu), positions, scale, interleaved, fmt,
                             q if q_in_place else None)
    assert torch.equal(v, v_before) and torch.equal(k, k_before)
    if q_in_place:
        assert out.data_ptr() == q.data_ptr() and out.stride() == q.stride()
    assert torch.equal(vc.cpu(), want[1]) and torch.equal(vs.cpu(), want[3])
    rows = []
    for b in range(len(lens)):
        for i in range(news[b]):
            p = lens[b] - news[b] + i
            if 0 <= p < width * ps:
                rows.append((int(table[b, p // ps]), p % ps, cu[b] + i))
    check_cache((kc.cpu(), ks.cpu()), (want[0], want[2]), big.cpu(), rows, fmt, turned.cpu())
    off = (out.double() - want_q).abs()
    bound = want_q.abs() * UNIT[dt] + 2.0 ** -21 * big_q + TINY[dt]
    assert bool((off <= bound).all()), float((off / bound).max())


STEPS = [
    # lens (counting the new tokens), new tokens, heads, kv heads, dim, page
    ([1, 16, 17, 40], [1, 1, 1, 1], 4, 2, 64, 16),
    ([5, 64, 65, 128, 200], [5, 64, 1, 3, 150], 7, 1, 128, 64),
    ([300, 0, 7], [130, 0, 7], 3, 3, 256, 128),
    ([33], [33], 8, 8, 128, 32),
    ([2, 30], [4, 2], 1, 1, 64, 16),  # two of the first sequence's tokens have no place
    ([128, 1], [128, 1], 40, 8, 128, 128),
]


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dt", [H, B])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("part", [1, 2, 4])
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_matches_definition(ops, case, part, interleaved, dt, fmt):
    lens, news, heads, hk, d, ps = STEPS[case]
    run(ops, case, lens, news, heads, hk, d, ps, d // part, interleaved, dt, fmt)


@pytest.mark.parametrize("far", [0, 1 << 20, (1 << 31) - 200, -77])
@pytest.mark.parametrize("theta", [10000.0, 500000.0])
def test_far_positions(ops, far, theta):
    """Angles of positions up to 2^31: 64 bits hold them to 2^-24 of a turn."""
    pos = i32([far + i * i for i in range(12)])
    run(ops, 1, [40, 12, 9], [6, 4, 2], 8, 2, 128, 16, 128, False, H, "e4m3", pos, 1.25, theta=theta)


def test_same_number_each_and_in_place(ops):
    run(ops, 2, [9, 70, 33], [1, 1, 1], 8, 2, 64, 32, 64, False, B, "e4m3", cu_none=True)
    run(ops, 3, [9, 70, 33], [5, 5, 5], 6, 2, 64, 32, 32, True, H, "e5m2", cu_none=True, q_in_place=True)
    run(ops, 4, [200] * 40, [3] * 40, 6, 2, 128, 64, 128, False, H, "e4m3", cu_none=True, q_in_place=True)


def test_tree_nodes_share_a_position(ops):
    run(ops, 5, [50, 8], [7, 5], 4, 2, 128, 16, 128, False, B, "e4m3", i32([43, 44, 44, 45, 45, 46, 45, 3, 4, 4, 5, 5]))


@pytest.mark.parametrize("d, rotary, ps", [(128, 96, 128), (256, 96, 128), (256, 48, 128), (64, 48, 64), (256, 256, 128), (128, 80, 32)])
def test_parts_of_a_head_that_are_no_power_of_two(ops, d, rotary, ps):
    """Any multiple of 16 turns; the tables of a full page's angles pass the sizes where shared memory changes its kind."""
    run(ops, d + rotary, [ps + 40, 5], [ps + 30, 3], 3, 1, d, ps, rotary, False, H, "e4m3")
    run(ops, d + rotary, [ps + 40, 5], [ps + 30, 3], 3, 1, d, ps, rotary, True, B, "e5m2")


def test_unaligned_rows_and_keys_only(ops):
    g = gen(6)
    table, kc, vc, ks, vs = make_cache(g, 1, 2, 1, 16, 64, "e4m3")
    qkv = torch.randn(3, 3 * 64 + 1, generator=g, device="cuda").to(H)
    q, k, v = (qkv[:, 1 + 64 * i: 65 + 64 * i].unflatten(1, (1, 64)) for i in range(3))
    f = freqs(64)
    again = [x.clone() for x in (kc, vc, ks, vs)]
    out = ops.kv_append_rope(q, k, v, kc, vc, ks, vs, table, i32([20]), f, i32([0, 3]))
    same = ops.kv_append_rope(q.contiguous(), k.contiguous(), v.contiguous(), *again, table, i32([20]), f, i32([0, 3]))
    assert torch.equal(out, same) and all(torch.equal(x, y) for x, y in zip((kc, vc, ks, vs), again))
    assert ops.kv_append_rope(None, k, v, kc, vc, ks, vs, table, i32([20]), f, i32([0, 3])) is None
    assert all(torch.equal(x, y) for x, y in zip((kc, vc, ks, vs), again))


def test_agrees_with_append_at_position_zero(ops):
    """No turn at position 0: the same cache as kv_append's, bit for bit; a NaN reaches its partner (NaN * sin 0)."""
    g = gen(7)
    for fmt in ("e4m3", "e5m2"):
        table, kc, vc, ks, vs = make_cache(g, 2, 3, 2, 32, 128, fmt, pow2=False)
        again = [x.clone() for x in (kc, vc, ks, vs)]
        kv = (torch.randn(45, 2, 2, 128, generator=g, device="cuda") * 300).to(H)
        kv[3, 0, 1, 9] = float("nan")
        kv[7, 1, 0, 100] = float("inf")
        args = (table, i32([50, 70]))
        turned = kv[:, 0].clone()
        turned[3, 1, 9 + 32] = float("nan")
        ops.kv_append(turned, kv[:, 1], *again, *args, i32([0, 20, 45]), fmt)
        ops.kv_append_rope(None, kv[:, 0], kv[:, 1], kc, vc, ks, vs, *args, freqs(64), i32([0, 20, 45]), torch.zeros(45, dtype=torch.int32, device="cuda"), fmt=fmt)
        f8 = F8[fmt]
        for x, y in zip((kc, vc, ks, vs), again):
            a, b = (x.view(f8).float(), y.view(f8).float()) if x.dtype == torch.uint8 else (x, y)
            assert torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


def test_holes_and_tokens_past_the_table(ops):
    """Keys without a place are not stored, queries turn all the same; rows that no sequence owns stay."""
    g = gen(8)
    table, kc, vc, ks, vs = make_cache(g, 2, 2, 2, 16, 64, "e4m3")
    table[0, 1] = -1
    before = [x.clone() for x in (kc, vc, ks, vs)]
    q, k, v = (torch.randn(14, 2, 64, generator=g, device="cuda").to(H) for _ in range(3))
    out = torch.full((14, 2, 64), 7.0, dtype=H, device="cuda")
    ops.kv_append_rope(q, k, v, kc, vc, ks, vs, table, i32([24, 40]), freqs(64), i32([0, 5, 12]), q_out=out)
    assert all(torch.equal(x, y) for x, y in zip((kc, vc, ks, vs), before))  # 19..23 fall into the hole, 33..39 past the table
    want, big = turn64(q[:12], i32(list(range(19, 24)) + list(range(33, 40))), freqs(64), False)
    assert bool(((out[:12].double() - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -21 * big + 2.0 ** -25).all())
    assert bool((out[12:] == 7.0).all())


def test_descending_offsets_write_nothing(ops):
    g = gen(9)
    table, kc, vc, ks, vs = make_cache(g, 2, 2, 2, 16, 64, "e4m3")
    before = [x.clone() for x in (kc, vc, ks, vs)]
    q, k, v = (torch.randn(6, 2, 64, generator=g, device="cuda").to(H) for _ in range(3))
    out = torch.full_like(q, 7.0)
    ops.kv_append_rope(q, k, v, kc, vc, ks, vs, table, i32([9, 9]), freqs(64), i32([0, 5, 3]), q_out=out)
    assert F.lib().fp8imma_device_error(1) == 7
    assert all(torch.equal(x, y) for x, y in zip((kc, vc, ks, vs), before)) and bool((out == 7.0).all())


def test_graph_stream_and_repeat(ops):
    g = gen(10)
    table, kc, vc, ks, vs = make_cache(g, 4, 4, 2, 16, 64, "e4m3")
    q, k, v = (torch.randn(4, 2, 64, generator=g, device="cuda").to(B) for _ in range(3))
    lens = i32([9, 20, 33, 60])
    first = [x.clone() for x in (kc, vc, ks, vs)]
    out = ops.kv_append_rope(q, k, v, *first, table, lens, freqs(64))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    second = [x.clone() for x in (kc, vc, ks, vs)]
    with torch.cuda.stream(side):
        out2 = ops.kv_append_rope(q, k, v, *second, table, lens, freqs(64))
    side.synchronize()
    assert torch.equal(out, out2) and all(torch.equal(x, y) for x, y in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    third = [x.clone() for x in (kc, vc, ks, vs)]
    with torch.cuda.graph(graph):
        out3 = ops.kv_append_rope(q, k, v, *third, table, lens, freqs(64))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, out3) and all(torch.equal(x, y) for x, y in zip(first, third))
    lens += 1  # lengths may change between replays
    want = [x.clone() for x in third]
    out4 = ops.kv_append_rope(q, k, v, *want, table, lens, freqs(64))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out4, out3) and all(torch.equal(x, y) for x, y in zip(want, third))


def test_empty(ops):
    g = gen(11)
    table, kc, vc, ks, vs = make_cache(g, 1, 2, 1, 16, 64, "e4m3")
    z = torch.empty(0, 1, 64, dtype=H, device="cuda")
    assert ops.kv_append_rope(z, z, z, kc, vc, ks, vs, table, i32([5]), freqs(64)).shape == (0, 1, 64)


@pytest.mark.parametrize("change, message", [
    (dict(inv_freq=torch.ones(4)), "inv_freq must have shape"), (dict(inv_freq=torch.ones(40)), "inv_freq must have shape"),
    (dict(inv_freq=torch.ones(8, dtype=torch.float64)), "inv_freq must be"), (dict(positions=torch.zeros(3, dtype=torch.int32)), "positions must have shape"),
    (dict(positions=torch.zeros(2)), "positions must be"), (dict(rope_scale=float("nan")), "rope_scale"),
    (dict(q=torch.zeros(2, 2, 64)), "q must have k's dtype"), (dict(q=torch.zeros(1, 2, 64, dtype=H)), "q must have shape"),
    (dict(q=None, q_out=torch.zeros(2, 2, 64, dtype=H)), "with q only"), (dict(k=torch.zeros(2, 1, 32, dtype=H)), "k and v must have shape"),
    (dict(fmt="int8"), "fmt must be")])
def test_refuses(ops, change, message):
    g = gen(12)
    table, kc, vc, ks, vs = make_cache(g, 2, 2, 1, 16, 64, "e4m3")
    z = lambda *s: torch.zeros(*s, dtype=H, device="cuda")
    a = dict(q=z(2, 2, 64), k=z(2, 1, 64), v=z(2, 1, 64), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, page_table=table, seq_lens=i32([3, 4]),
             inv_freq=freqs(64))
    a |= {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in change.items()}
    with pytest.raises(RuntimeError, match=message):
        ops.kv_append_rope(**a)


def test_refuses_overlap(ops):
    g = gen(13)
    table, kc, vc, ks, vs = make_cache(g, 2, 2, 1, 16, 64, "e4m3")
    qkv = torch.zeros(2, 4, 64, dtype=H, device="cuda")
    with pytest.raises(RuntimeError, match="q itself or contiguous"):
        ops.kv_append_rope(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], kc, vc, ks, vs, table, i32([3, 4]), freqs(64), q_out=qkv[:, 1:3])
    big = torch.zeros(3, 2, 64, dtype=H, device="cuda")
    with pytest.raises(RuntimeError, match="apart"):
        ops.kv_append_rope(big[:2], qkv[:, 2:3], qkv[:, 3:], kc, vc, ks, vs, table, i32([3, 4]), freqs(64), q_out=big[1:])
