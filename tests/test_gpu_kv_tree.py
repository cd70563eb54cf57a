"""kv_attention_tree on the GPU against 64 bits, within the bound that its roundings give."""
import math

import pytest
import torch

import fp8imma_b200 as F
from layer_ref import ref_tree, tree_mask
from test_gpu_kv_cache import gen, i32, make_cache, offsets

pytestmark = pytest.mark.gpu

H, B = torch.float16, torch.bfloat16


# rows a KV head from which attention runs on tcgen05: never, by the kernel's rule, always
@pytest.fixture(params=[1 << 20, 0, 1], ids=["mma", "default", "tcgen05"])
def ops(cuda, request):
    L = F.lib()
    assert L.fp8imma_set_attention_tc_rows(request.param) == 0
    yield F.ext()
    L.fp8imma_set_attention_tc_rows(0)
    assert L.fp8imma_device_error(1) == 0


def trees(seed, news, words=None):
    """Random trees, one a sequence: (mask rows, depths)."""
    g = torch.Generator().manual_seed(seed)
    masks, depths = [], []
    most = words or max(1, -(-max(news) // 32))
    for n in news:
        parents = [-1] + [int(torch.randint(max(0, i - 4), i, (1,), generator=g)) for i in range(1, n)]
        d = []
        for p in parents[:n]:
            d.append(d[p] + 1 if p >= 0 else 0)
        masks.append(tree_mask(parents[:n], most) if n else torch.zeros(0, most, dtype=torch.int32))
        depths += d
    return torch.cat(masks).cuda(), depths


def queries(g, t, hq, d, dt):
    return (2 * torch.randn(t, hq, d, generator=g, device="cuda")).to(dt)


def check(got, want):
    out, lse = got
    ref, ref_lse, bound, dlse = want
    off = (out.double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-30)).max())
    gone = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(lse), gone) and bool((lse[gone] < 0).all())
    assert bool(((lse.double() - ref_lse).abs()[~gone] <= dlse[~gone]).all())


def attend(ops, q, cache, lens, cu, fmt, mask=None, positions=None, cap=0.0, window=0, scale=None, **kw):
    table, kc, vc, ks, vs = cache
    return ops.kv_attention_tree(q, kc, vc, ks, vs, table, i32(lens), mask, None if cu is None else i32(cu), positions, scale, cap, window, fmt, **kw)


def define(q, cache, lens, cu, fmt, mask=None, positions=None, cap=0.0, window=0, scale=None):
    table, kc, vc, ks, vs = cache
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    return ref_tree(q, kc, vc, ks, vs, table, lens, cu, scale, window, fmt, cap, mask, positions)


STEPS = [
    # lens (counting the step's tokens), tokens of the step, heads, kv heads, dim, page, window, cap
    ([17, 130, 131, 300], [1, 8, 3, 16], 8, 2, 128, 64, 0, 0.0),
    ([40, 7, 129], [7, 7, 5], 4, 1, 64, 16, 0, 30.0),
    ([260, 33], [40, 33], 6, 2, 128, 32, 0, 20.0),        # masks of two words, trees across a tile's border
    ([200, 90, 12], [9, 2, 12], 5, 1, 64, 16, 25, 0.0),   # window
    ([150, 128], [12, 6], 7, 1, 256, 128, 40, 5.0),
    ([70, 64], [70, 64], 4, 4, 64, 16, 0, 2.0),           # nothing before the step
    ([3, 140], [5, 1], 2, 2, 128, 16, 0, 0.0),            # two tokens without a place
]


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dt", [H, B])
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_trees(ops, case, dt, fmt):
    lens, news, hq, hk, d, ps, window, cap = STEPS[case]
    g = gen(case)
    cache = make_cache(g, len(lens), -(-max(lens) // ps), hk, ps, d, fmt)
    cu = offsets(news)
    q = queries(g, cu[-1], hq, d, dt)
    mask, depth = trees(case, news)
    start = [ln - n for ln, n in zip(lens, news) for _ in range(n)]
    pos = i32([s + x for s, x in zip(start, depth)])
    for positions in (pos, None):
        a = dict(mask=mask, positions=positions, cap=cap, window=window)
        check(attend(ops, q, cache, lens, cu, fmt, **a), define(q, cache, lens, cu, fmt, **a))


@pytest.mark.parametrize("dt", [H, B])
@pytest.mark.parametrize("cap", [0.0, 0.5, 50.0])
@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_causal_with_capped_scores(ops, d, window, cap, dt):
    g = gen(d)
    lens, news = [140, 300, 5, 64], [3, 20, 5, 1]
    cache = make_cache(g, 4, 10, 2, 32, d, "e4m3")
    cu = offsets(news)
    q = queries(g, cu[-1], 6, d, dt)
    a = dict(cap=cap, window=window)
    check(attend(ops, q, cache, lens, cu, "e4m3", **a), define(q, cache, lens, cu, "e4m3", **a))


@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
def test_scores_at_the_cap_and_other_scales(ops, scale):
    """Scores far beyond the cap end at it, with either sign; every key then weighs the same."""
    g = gen(1)
    lens, news = [200, 131], [6, 3]
    cache = make_cache(g, 2, 7, 1, 32, 128, "e4m3")
    cu = offsets(news)
    q = queries(g, 9, 16, 128, H)
    mask, _ = trees(1, news)
    a = dict(mask=mask, cap=15.0, scale=scale)
    check(attend(ops, q, cache, lens, cu, "e4m3", **a), define(q, cache, lens, cu, "e4m3", **a))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_that_see_nothing(ops, d):
    g = gen(d + 1)
    lens, news = [6, 100, 0], [6, 4, 0]
    cache = make_cache(g, 3, 7, 1, 16, d, "e4m3")
    cu = offsets(news)
    q = queries(g, 10, 4, d, H)
    mask = torch.zeros(10, 1, dtype=torch.int32, device="cuda")
    mask[1], mask[3], mask[7] = 2, 0b101, 1
    a = dict(mask=mask)
    out, lse = attend(ops, q, cache, lens, cu, "e4m3", **a)
    check((out, lse), define(q, cache, lens, cu, "e4m3", **a))
    for i in (0, 2, 4, 5):
        assert bool((out[i] == 0).all()) and bool((lse[i] == -math.inf).all())


def test_masks_that_are_no_trees(ops):
    """Both directions, documents, bits past the step's tokens and masks narrower than it."""
    g = gen(2)
    lens, news = [150, 45], [45, 45]
    cache = make_cache(g, 2, 10, 2, 16, 64, "e5m2")
    cu = offsets(news)
    q = queries(g, 90, 4, 64, B)
    full = torch.full((90, 2), -1, dtype=torch.int32, device="cuda")
    docs = torch.tensor([[0xFF << (i // 8 * 8) if i < 32 else 0, 0xFF << ((i - 32) // 8 * 8) if i >= 32 else 0] for i in range(45)] * 2)
    docs = torch.where(docs >= 2 ** 31, docs - 2 ** 32, docs).to(torch.int32).cuda()
    narrow = full[:, :1].contiguous()
    wide = torch.cat((full, torch.full((90, 3), -1, dtype=torch.int32, device="cuda")), 1).contiguous()
    for mask in (full, docs, narrow, wide):
        check(attend(ops, q, cache, lens, cu, "e5m2", mask=mask), define(q, cache, lens, cu, "e5m2", mask=mask))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_chain_is_causal(ops, d):
    """A chain's mask gives the causal step: to the bit where both take the same tiles."""
    g = gen(3)
    lens, news = [333, 40], [9, 4]
    cache = make_cache(g, 2, 21, 1, 16, d, "e4m3")
    cu = offsets(news)
    q = queries(g, 13, 4, d, H)
    mask = torch.cat([tree_mask(list(range(-1, n - 1))) for n in news]).cuda()
    check(attend(ops, q, cache, lens, cu, "e4m3", mask=mask), define(q, cache, lens, cu, "e4m3"))


def test_positions_out_of_the_step_count_as_its_ends(ops):
    g = gen(4)
    lens, news = [120, 90], [5, 3]
    cache = make_cache(g, 2, 8, 1, 16, 64, "e4m3")
    cu = offsets(news)
    q = queries(g, 8, 4, 64, H)
    mask, _ = trees(4, news)
    for pos in ([0] * 8, [10 ** 9] * 8, [-(2 ** 31)] * 4 + [2 ** 31 - 1] * 4):
        a = dict(mask=mask, positions=i32(pos), window=30)
        check(attend(ops, q, cache, lens, cu, "e4m3", **a), define(q, cache, lens, cu, "e4m3", **a))


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_nan_in_keys_and_values_that_a_node_does_not_see(ops, d, fmt):
    """What a sibling branch holds does not reach a node."""
    g = gen(d)
    lens, news = [150, 20], [8, 8]
    cache = make_cache(g, 2, 10, 1, 16, d, fmt)
    table, kc, vc, ks, vs = cache
    cu = offsets(news)
    q = queries(g, 16, 4, d, H)
    parents = [-1, 0, 0, 1, 2, 3, 4, 5]
    mask = torch.cat([tree_mask(parents)] * 2).cuda()
    nan = 0x7F if fmt == "e4m3" else 0x7E
    for b, ln in enumerate(lens):
        for node in (1, 3):  # ancestors of 5 and 7
            p = ln - 8 + node
            kc[table[b, p // 16].long(), :, p % 16] = nan
            vc[table[b, p // 16].long(), :, p % 16, 3] = nan
    out, lse = attend(ops, q, cache, lens, cu, fmt, mask=mask, cap=20.0)
    want = define(q, cache, lens, cu, fmt, mask=mask, cap=20.0)
    hit = torch.tensor([node in (1, 3, 5, 7) for node in range(8)] * 2, device="cuda")
    assert bool(torch.isnan(lse[hit]).all())
    check((out[~hit], lse[~hit]), [x[~hit] for x in want])


def test_holes_strides_and_tokens_that_no_sequence_owns(ops):
    g = gen(5)
    lens, news = [200, 60], [5, 7]
    cache = make_cache(g, 2, 13, 2, 16, 64, "e4m3")
    cache[0][0, 3] = -1
    cache[0][0, 12] = 1 << 20
    cu = offsets(news)
    wide = queries(g, 15, 3 * 4, 64, H)
    q = wide[:, 4:8]
    mask, _ = trees(5, news)
    mask = torch.cat((mask, torch.full((3, 1), -1, dtype=torch.int32, device="cuda")))
    out = torch.full((15, 4, 64), 7.0, dtype=H, device="cuda")
    got = attend(ops, q, cache, lens, cu, "e4m3", mask=mask, out=out)
    want = define(q, cache, lens, cu, "e4m3", mask=mask)
    check((got[0][:12], got[1][:12]), [x[:12] for x in want])
    assert bool((out[12:] == 7.0).all())


def test_same_number_each_and_long_contexts(ops):
    g = gen(6)
    lens = [2000, 1, 700, 1400]
    cache = make_cache(g, 4, 2000 // 64 + 1, 1, 64, 128, "e4m3")
    q = queries(g, 4, 8, 128, B)
    mask = torch.ones(4, 1, dtype=torch.int32, device="cuda")
    check(attend(ops, q, cache, lens, None, "e4m3", mask=mask, cap=30.0), define(q, cache, lens, [0, 1, 2, 3, 4], "e4m3", mask=mask, cap=30.0))


def test_repeats_streams_and_graphs_at_once(ops):
    """The same bits from every call; two graphs captured on one stream hold no common workspace."""
    g = gen(7)
    lens, news = [3000, 2500, 40], [12, 16, 9]
    cache = make_cache(g, 3, 3000 // 32 + 1, 2, 32, 128, "e4m3")
    cu = offsets(news)
    q = [queries(g, cu[-1], 16, 128, H) for _ in range(2)]
    mask, _ = trees(7, news)
    lens_d, cu_d = i32(lens), i32(cu)
    table, kc, vc, ks, vs = cache

    def call(x):
        return ops.kv_attention_tree(x, kc, vc, ks, vs, table, lens_d, mask, cu_d, softcap=25.0)

    want = [call(x) for x in q]
    for x, w in zip(q, want):
        for _ in range(3):
            got = call(x)
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
    graphs, outs = [], []
    for x in q:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(x))
        graphs.append(graph)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


def test_sequences_longer_than_their_table(ops):
    """Keys past the table are not read, the step's own among them."""
    g = gen(11)
    lens, news = [70, 64, 500], [10, 5, 7]  # the table holds 64 keys
    cache = make_cache(g, 3, 4, 2, 16, 128, "e4m3")
    cu = offsets(news)
    q = queries(g, cu[-1], 4, 128, H)
    mask, _ = trees(11, news)
    for window in (0, 30):
        a = dict(mask=mask, cap=10.0, window=window)
        check(attend(ops, q, cache, lens, cu, "e4m3", **a), define(q, cache, lens, cu, "e4m3", **a))


def test_two_streams_at_once(ops):
    g = gen(12)
    lens, news = [2600, 1300], [9, 16]
    cache = make_cache(g, 2, 2600 // 64 + 1, 2, 64, 64, "e5m2")
    cu = offsets(news)
    mask, _ = trees(12, news)
    q = [queries(g, cu[-1], 14, 64, B) for _ in range(2)]
    lens_d, cu_d = i32(lens), i32(cu)
    table, kc, vc, ks, vs = cache
    call = lambda x: ops.kv_attention_tree(x, kc, vc, ks, vs, table, lens_d, mask, cu_d, softcap=30.0, fmt="e5m2")  # noqa: E731
    want = [call(x) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(call(q[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(o, want[k][0]) and torch.equal(l, want[k][1]) for o, l in got[k])


def test_descending_offsets_are_refused_on_the_device(ops):
    g = gen(8)
    cache = make_cache(g, 2, 4, 1, 16, 64, "e4m3")
    q = queries(g, 6, 4, 64, H)
    out = torch.full_like(q, 7.0)
    attend(ops, q, cache, [20, 30], [0, 5, 3], "e4m3", mask=torch.ones(6, 1, dtype=torch.int32, device="cuda"), out=out)
    assert F.lib().fp8imma_device_error(1) == 7
    assert bool((out == 7.0).all())


def test_empty(ops):
    g = gen(9)
    cache = make_cache(g, 2, 2, 1, 16, 64, "e4m3")
    out, lse = attend(ops, torch.empty(0, 4, 64, dtype=H, device="cuda"), cache, [5, 6], None, "e4m3", mask=torch.empty(0, 1, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


@pytest.mark.parametrize("change, message", [
    (dict(softcap=-1.0), "softcap"), (dict(softcap=float("inf")), "softcap"), (dict(window=-1), "window"),
    (dict(softmax_scale=float("nan")), "softmax_scale"), (dict(tree_mask=torch.zeros(3, 1, dtype=torch.int32)), "tree_mask must have shape"),
    (dict(tree_mask=torch.zeros(2, 0, dtype=torch.int32)), "tree_mask must have shape"), (dict(tree_mask=torch.zeros(2, 1, dtype=torch.int64)), "tree_mask must be"),
    (dict(positions=torch.zeros(2, dtype=torch.int32)), "with tree_mask only"),
    (dict(tree_mask=torch.zeros(2, 1, dtype=torch.int32), positions=torch.zeros(3, dtype=torch.int32)), "positions must have shape"),
    (dict(q=torch.zeros(2, 3, 64, dtype=H), k_cache=2), "multiple of kv_heads"), (dict(out=torch.zeros(2, 2, 64)), "out must be")])
def test_refuses(ops, change, message):
    g = gen(10)
    hk = change.get("k_cache", 1)
    table, kc, vc, ks, vs = make_cache(g, 2, 2, hk, 16, 64, "e4m3")
    a = dict(q=torch.zeros(2, 2, 64, dtype=H, device="cuda"), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, page_table=table, seq_lens=i32([3, 4]))
    a |= {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in change.items() if k != "k_cache"}
    with pytest.raises(RuntimeError, match=message):
        ops.kv_attention_tree(**a)
