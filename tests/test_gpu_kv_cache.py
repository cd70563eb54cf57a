"""The paged 8-bit KV cache on the GPU: append (bit for bit against the page-by-page definition) and attention
(against 64 bits, within the bound that its roundings give)."""
import math

import pytest
import torch

import fp8imma_b200 as F
from serving_ref import F8, FMAX, ref_append, ref_attention

pytestmark = pytest.mark.gpu


# rows a KV head from which attention runs on tcgen05: never, by the kernel's rule, always
@pytest.fixture(params=[1 << 20, 0, 1], ids=["mma", "default", "tcgen05"])
def ops(cuda, request):
    L = F.lib()
    assert L.fp8imma_set_attention_tc_rows(request.param) == 0
    yield F.ext()
    L.fp8imma_set_attention_tc_rows(0)
    assert L.fp8imma_device_error(1) == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_cache(g, batch, width, hk, ps, d, fmt, spread=0.5, pow2=True, extra=3):
    pages = batch * width + extra
    table = torch.randperm(pages, generator=g, device="cuda")[: batch * width].view(batch, width).to(torch.int32)
    out = []
    for _ in range(2):
        x = torch.randn(pages, hk, ps, d, generator=g, device="cuda")
        x *= torch.exp(spread * torch.randn(pages, hk, 1, 1, generator=g, device="cuda"))
        s = x.abs().amax((2, 3)) / FMAX[fmt]
        s = torch.exp2(torch.ceil(torch.log2(s))) if pow2 else s * 1.01
        out.append(((x / s[:, :, None, None]).clamp(-FMAX[fmt], FMAX[fmt]).to(F8[fmt]).view(torch.uint8), s.contiguous()))
    (kc, ks), (vc, vs) = out
    return table, kc, vc, ks, vs


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def offsets(news):
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    return cu


# -- append ----------------------------------------------------------------

APPEND = [
    # lens (counting the new tokens), new tokens, kv heads, dim, page
    ([1, 16, 17, 40], [1, 1, 1, 1], 2, 64, 16),
    ([5, 64, 65, 128, 200], [5, 64, 1, 3, 150], 1, 128, 64),
    ([300, 0, 7], [130, 0, 7], 3, 256, 128),
    ([33], [33], 8, 128, 32),
    ([2, 30], [4, 2], 1, 64, 16),  # two of the first sequence's tokens have no place
]


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append_matches_definition(ops, case, dtype, fmt):
    lens, news, hk, d, ps = APPEND[case]
    g = gen(case)
    width = max(1, -(-max(lens) // ps))
    table, kc, vc, ks, vs = make_cache(g, len(lens), width, hk, ps, d, fmt)
    cu = offsets(news)
    kv = (torch.randn(cu[-1], 3, hk, d, generator=g, device="cuda") * torch.exp(2 * torch.randn(cu[-1], 1, 1, 1, generator=g, device="cuda"))).to(dtype)
    k, v = kv[:, 1], kv[:, 2]
    want = ref_append(k.cpu(), v.cpu(), kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), table.cpu(), lens, cu, fmt)
    ops.kv_append(k, v, kc, vc, ks, vs, table, i32(lens), i32(cu), fmt)
    for got, ref in zip((kc, vc, ks, vs), want):
        assert torch.equal(got.cpu(), ref)


def test_append_uniform_and_special_values(ops):
    """Without offsets every sequence has the same number of tokens; NaN is kept, Inf saturates and does not count
    for the scale, a zero page takes the smallest scale, rows that are not 16-byte aligned are read as well."""
    hk, d, ps, fmt = 2, 64, 16, "e4m3"
    g = gen(3)
    lens, n = [20, 33, 16], 2
    table, kc, vc, ks, vs = make_cache(g, 3, 3, hk, ps, d, fmt)
    kv = torch.randn(6, 2, hk, d + 1, generator=g, device="cuda").to(torch.float16)[..., 1:]
    k, v = kv[:, 0], kv[:, 1]
    k[0, 0, 3], k[0, 1, 4], k[2, 0, 5] = math.nan, math.inf, -math.inf
    v[4:] = 0
    want = ref_append(k.cpu(), v.cpu(), kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), table.cpu(), lens, [0, 2, 4, 6], fmt)
    ops.kv_append(k, v, kc, vc, ks, vs, table, i32(lens), None, fmt)
    assert torch.equal(ks.cpu(), want[2]) and torch.equal(vs.cpu(), want[3])
    nan = (kc.cpu() & 0x7F) == 0x7F
    assert torch.equal(nan, (want[0] & 0x7F) == 0x7F)
    assert torch.equal(kc.cpu()[~nan], want[0][~nan]) and torch.equal(vc.cpu(), want[1])


def test_append_grows_scale_and_keeps_values(ops):
    """A page filled token by token with growing rows: each earlier value stays within a code's step of what it was."""
    hk, d, ps, fmt = 1, 64, 16, "e4m3"
    g = gen(4)
    table, kc, vc, ks, vs = make_cache(g, 1, 1, hk, ps, d, fmt)
    rows = torch.randn(16, hk, d, generator=g, device="cuda").to(torch.bfloat16) * torch.exp2(torch.arange(16, device="cuda") % 7)[:, None, None].to(torch.bfloat16)
    for i in range(16):
        ops.kv_append(rows[i:i + 1], rows[i:i + 1], kc, vc, ks, vs, table, i32([i + 1]), None, fmt)
    page = int(table[0, 0])
    val = kc[page].view(F8[fmt]).double() * ks[page].double()[:, None, None]
    ref = rows.transpose(0, 1).double()
    step = torch.maximum(ref.abs() * 2.0 ** -4, ks[page].double()[:, None, None] * 2.0 ** -10 * 7)
    assert ((val - ref).abs() <= step).all()


def test_append_skips_holes(ops):
    hk, d, ps, fmt = 1, 64, 16, "e5m2"
    g = gen(5)
    table, kc, vc, ks, vs = make_cache(g, 2, 2, hk, ps, d, fmt)
    table[0, 1], table[1, 0] = -1, kc.shape[0]
    k = torch.randn(2 * 20, hk, d, generator=g, device="cuda").half()
    want = ref_append(k.cpu(), k.cpu(), kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), table.cpu(), [20, 20], [0, 20, 40], fmt)
    ops.kv_append(k, k, kc, vc, ks, vs, table, i32([20, 20]), None, fmt)
    for got, ref in zip((kc, vc, ks, vs), want):
        assert torch.equal(got.cpu(), ref)


# -- attention ---------------------------------------------------------------

ATTEND = [
    # lens, new tokens, heads, kv heads, dim, page, window
    ([1], [1], 1, 1, 64, 16, 0),
    ([1, 2, 15, 16, 17, 127, 128, 129, 400], [1] * 9, 8, 2, 128, 16, 0),
    ([517], [1], 32, 8, 128, 64, 0),
    ([0, 0, 3, 700], [0, 1, 3, 5], 7, 1, 64, 32, 0),
    ([300, 65], [8, 2], 16, 1, 128, 128, 0),
    ([300, 1000, 40], [1, 3, 6], 28, 4, 64, 16, 100),
    ([2, 90], [5, 9], 4, 4, 128, 64, 0),           # more new tokens than the sequence has
    ([1200, 30], [1, 1], 5, 1, 256, 64, 0),
    ([260], [70], 6, 2, 256, 32, 33),
    ([4100], [1], 16, 1, 128, 64, 1),              # a window of one key
    ([128, 384], [128, 200], 4, 2, 64, 128, 0),    # prompts
    ([2500] * 3, [1] * 3, 64, 8, 128, 64, 0),
]


def run_attend(ops, q, cache, lens, cu, window, fmt, scale=None, uniform=False):
    table, kc, vc, ks, vs = cache
    out, lse = ops.kv_attention(q, kc, vc, ks, vs, table, i32(lens), None if uniform else i32(cu), softmax_scale=scale, window=window, fmt=fmt)
    ref = ref_attention(q, kc, vc, ks, vs, table, lens, cu, scale if scale is not None else 1 / math.sqrt(q.shape[2]), window, fmt)
    return out, lse, ref


def check(out, lse, ref):
    o, l, bound = ref
    err = (out.double() - o).abs()
    assert (err <= bound).all(), "worst %.3g of the bound" % float((err / bound.clamp_min(1e-300)).max())
    empty = l == -math.inf
    assert torch.equal(empty, lse == -math.inf)
    assert (out[empty] == 0).all()
    assert ((lse.double() - l)[~empty].abs() <= 2e-5 * (1 + l[~empty].abs())).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention_matches_definition(ops, case, dtype, fmt):
    lens, news, hq, hk, d, ps, window = ATTEND[case]
    g = gen(10 + case)
    width = max(1, -(-max(lens) // ps))
    cache = make_cache(g, len(lens), width, hk, ps, d, fmt)
    cu = offsets(news)
    q = torch.randn(cu[-1], hq, d, generator=g, device="cuda").to(dtype)
    check(*run_attend(ops, q, cache, lens, cu, window, fmt))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_ignores_what_lies_behind_the_end(ops, dtype):
    """NaN codes behind a sequence's end and in pages outside its table, NaN scales of unused pages."""
    g = gen(40)
    lens, hq, hk, d, ps, fmt = [70, 5, 129], 8, 2, 128, 64, "e4m3"
    table, kc, vc, ks, vs = make_cache(g, 3, 3, hk, ps, d, fmt)
    used = torch.zeros(kc.shape[0], dtype=torch.bool, device="cuda")
    for b, ln in enumerate(lens):
        n = -(-ln // ps)
        used[table[b, :n].long()] = True
        kc[int(table[b, n - 1]), :, (ln - 1) % ps + 1:] = 0x7F
        vc[int(table[b, n - 1]), :, (ln - 1) % ps + 1:] = 0xFF
    for x in (kc, vc):
        x[~used] = 0x7F
    for x in (ks, vs):
        x[~used] = math.nan
    q = torch.randn(3, hq, d, generator=g, device="cuda").to(dtype)
    check(*run_attend(ops, q, (table, kc, vc, ks, vs), lens, [0, 1, 2, 3], 0, fmt))


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_nan_in_keys_that_some_rows_do_not_see(ops, d, fmt):
    """A draft token with NaN (and, in E5M2, infinite) keys and values reaches the rows from its own on and no
    earlier one; a key that has left the window reaches only the rows that still see it."""
    g = gen(60)
    lens, n, hq, hk, ps = [150, 40], 6, 14, 2, 32
    table, kc, vc, ks, vs = make_cache(g, 2, 5, hk, ps, d, fmt)
    bad = 0x7F if fmt == "e4m3" else 0x7C

    def at(b, pos):
        return int(table[b, pos // ps]), slice(None), pos % ps

    vc[at(0, 147)][0, 5::16] = bad       # value of a draft token, some channels, head 0
    kc[at(1, 37)][1, 3] = 0x7F           # key of a draft token, one channel, head 1
    vc[at(0, 150 - 6 - 20 + 2)][1] = 0x7F  # leaves the window after the second row
    q = torch.randn(12, hq, d, generator=g, device="cuda").half()
    cu, window, scale = [0, 6, 12], 20, 1 / math.sqrt(d)
    out, lse, _ = run_attend(ops, q, (table, kc, vc, ks, vs), lens, cu, window, fmt)
    o, l, bound = ref_attention(q, kc, vc, ks, vs, table, lens, cu, scale, window, fmt)
    assert torch.isfinite(o).any() and not torch.isfinite(o).all()
    assert torch.equal(torch.isnan(out), torch.isnan(o)) and torch.equal(torch.isnan(lse), torch.isnan(l))
    inf = torch.isinf(o)
    assert torch.equal(torch.isinf(out), inf) and torch.equal(out[inf].double(), o[inf])
    fine = torch.isfinite(o)
    assert ((out.double() - o).abs()[fine] <= bound[fine]).all()


def test_attention_skips_holes(ops):
    """Holes at the front, in the middle, everywhere; holes that hide a whole stretch of pages."""
    g = gen(41)
    lens, hq, hk, d, ps, fmt = [900, 900, 100, 600], 4, 1, 64, 16, "e4m3"
    cache = make_cache(g, 4, 57, hk, ps, d, fmt)
    table = cache[0]
    table[0, 3], table[0, 20:40] = -1, 1 << 30
    table[1, :50] = -5
    table[2] = -1
    q = torch.randn(4, hq, d, generator=g, device="cuda").half()
    check(*run_attend(ops, q, cache, lens, [0, 1, 2, 3, 4], 0, fmt))


def test_attention_value_scales_far_apart(ops):
    """Pages whose value scales differ by many powers of two, zero scales among them, and scales that are no powers
    of two: the weight of a page counts by its scale."""
    g = gen(42)
    lens, hq, hk, d, ps, fmt = [640, 333], 8, 2, 128, 32, "e4m3"
    table, kc, vc, ks, vs = make_cache(g, 2, 20, hk, ps, d, fmt, pow2=False)
    vs *= torch.exp2(torch.randint(-24, 12, vs.shape, generator=g, device="cuda").float())
    vs[int(table[0, 2])] = 0.0
    q = (4 * torch.randn(2, hq, d, generator=g, device="cuda")).bfloat16()
    check(*run_attend(ops, q, (table, kc, vc, ks, vs), lens, [0, 1, 2], 0, fmt))


def test_attention_peaked_rows(ops):
    """Scores of several hundred: one key takes all the weight; scores far below zero."""
    g = gen(43)
    lens, hq, hk, d, ps, fmt = [500], 8, 1, 128, 64, "e4m3"
    cache = make_cache(g, 1, 8, hk, ps, d, fmt)
    q = (30 * torch.randn(1, hq, d, generator=g, device="cuda")).bfloat16()
    for scale in (1.0, -0.5, 0.0):
        check(*run_attend(ops, q, cache, lens, [0, 1], 0, fmt, scale=scale))


@pytest.mark.parametrize("d", [64, 128])
def test_attention_rising_scores(ops, d):
    """Scores that grow along the sequence: the running reference moves again and again, within tiles and between."""
    g = gen(45)
    table, kc, vc, ks, vs = make_cache(g, 1, 60, 2, 32, d, "e4m3")
    for i in range(60):
        ks[table[0, i].long()] *= 2.0 ** (i // 12)
    q = torch.randn(9, 16, d, generator=g, device="cuda").half()
    check(*run_attend(ops, q, (table, kc, vc, ks, vs), [1900], [0, 9], 0, "e4m3", scale=0.5))


@pytest.mark.parametrize("mult", [2.0 ** -30, 2.0 ** 40])
def test_attention_bf16_queries_outside_fp16(ops, mult):
    g = gen(44)
    lens, hq, hk, d, ps, fmt = [200], 4, 1, 128, 64, "e4m3"
    cache = make_cache(g, 1, 4, hk, ps, d, fmt)
    q = (torch.randn(1, hq, d, generator=g, device="cuda") * mult).bfloat16()
    check(*run_attend(ops, q, cache, lens, [0, 1], 0, fmt, scale=0.1 / mult))


def test_attention_strided_queries_and_streams(ops):
    """Queries inside a fused projection (and one that starts at an odd element), uniform runs without offsets, on
    another stream than the default one."""
    g = gen(45)
    lens, n, hq, hk, d, ps, fmt = [100, 64, 9], 3, 4, 2, 64, 16, "e4m3"
    cache = make_cache(g, 3, 7, hk, ps, d, fmt)
    fused = torch.randn(9, 3 * hq * d + 1, generator=g, device="cuda").half()
    st = torch.cuda.Stream()
    for off in (hq * d, 1):
        q = fused[:, off: off + hq * d].unflatten(1, (hq, d))
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got = run_attend(ops, q, cache, lens, [0, 3, 6, 9], 0, fmt, uniform=True)
        torch.cuda.current_stream().wait_stream(st)
        check(*got)


def test_attention_nan_stays_in_its_row(ops):
    g = gen(46)
    lens, hq, hk, d, ps, fmt = [300, 300], 8, 1, 128, 64, "e4m3"
    cache = make_cache(g, 2, 5, hk, ps, d, fmt)
    q = torch.randn(2, hq, d, generator=g, device="cuda").bfloat16()
    q[0, 3, 7] = math.nan
    table, kc, vc, ks, vs = cache
    out, lse = ops.kv_attention(q, kc, vc, ks, vs, table, i32(lens), None)
    bad = torch.isnan(out).any(-1)
    assert bad[0, 3] and torch.isnan(out[0, 3]).all() and torch.isnan(lse[0, 3])
    assert bad.sum() == 1 and torch.isnan(lse).sum() == 1


def test_attention_repeats_bit_for_bit(ops):
    """Work that is split over CTAs is joined in a fixed order; calls on two streams at once do not meet."""
    g = gen(47)
    lens, hq, hk, d, ps, fmt = [30000, 5, 9000], 64, 8, 128, 64, "e4m3"
    cache = make_cache(g, 3, -(-30000 // ps), hk, ps, d, fmt)
    q = torch.randn(3, hq, d, generator=g, device="cuda").half()
    table, kc, vc, ks, vs = cache
    ln = i32(lens)
    first, l0 = ops.kv_attention(q, kc, vc, ks, vs, table, ln, None)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for r in range(6):
        with torch.cuda.stream(streams[r % 2]):
            outs.append(ops.kv_attention(q, kc, vc, ks, vs, table, ln, None))
    torch.cuda.synchronize()
    for o, l in outs:
        assert torch.equal(o, first) and torch.equal(l, l0)


def test_attention_in_a_graph(ops):
    """A captured call reads lengths and table at replay: the sequence may grow between replays."""
    g = gen(48)
    hq, hk, d, ps, fmt = 8, 2, 128, 64, "e4m3"
    table, kc, vc, ks, vs = make_cache(g, 2, 40, hk, ps, d, fmt)
    q = torch.randn(2, hq, d, generator=g, device="cuda").half()
    ln = i32([100, 7])
    out = torch.empty_like(q)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        ops.kv_attention(q, kc, vc, ks, vs, table, ln, None, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        _, lse = ops.kv_attention(q, kc, vc, ks, vs, table, ln, None, out=out)
    for lens in ([100, 7], [2000, 2560], [1, 64]):
        ln.copy_(i32(lens))
        graph.replay()
        torch.cuda.synchronize()
        check(out, lse, ref_attention(q, kc, vc, ks, vs, table, lens, [0, 1, 2], 1 / math.sqrt(d), 0, fmt))


def test_cache_beyond_32_bit_offsets(ops):
    """A pool of more than 4 GB whose last pages are used."""
    hk, d, ps, fmt = 8, 128, 128, "e4m3"
    pages = (1 << 32) // (hk * ps * d) + 8
    kc = torch.zeros(pages, hk, ps, d, dtype=torch.uint8, device="cuda")
    vc = torch.zeros_like(kc)
    ks = torch.ones(pages, hk, device="cuda")
    vs = torch.ones_like(ks)
    table = i32([[pages - 1, pages - 3, 0]])
    g = gen(49)
    k, v = (torch.randn(300, hk, d, generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn(1, 16, d, generator=g, device="cuda").half()
    ops.kv_append(k, v, kc, vc, ks, vs, table, i32([300]), None, fmt)
    assert (kc[pages - 1] != 0).any() and (kc[pages - 2] == 0).all()
    sub = [pages - 1, pages - 3, 0]
    small = [x[sub].contiguous() for x in (kc, vc, ks, vs)]
    out, lse = ops.kv_attention(q, kc, vc, ks, vs, table, i32([300]), None)
    check(out, lse, ref_attention(q, *small, i32([[0, 1, 2]]), [300], [0, 1], 1 / math.sqrt(d), 0, fmt))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens, news, hq, hk, d, ps, window", [
    ([9000, 8000, 1, 700], [17, 30, 1, 64], 16, 2, 128, 64, 0),      # 64 to 512 rows, one sequence of one key
    ([5000, 6000, 130], [40, 1, 129], 24, 4, 64, 16, 700),           # rows that end in every tile, a window
    ([1500, 1290], [1500, 1030], 8, 4, 128, 32, 0),                  # whole prompts, one behind a prefix
])
def test_attention_many_rows(ops, lens, news, hq, hk, d, ps, window, dtype):
    g = gen(90 + d)
    cache = make_cache(g, len(lens), -(-max(lens) // ps), hk, ps, d, "e4m3")
    cu = offsets(news)
    q = torch.randn(cu[-1], hq, d, generator=g, device="cuda").to(dtype)
    check(*run_attend(ops, q, cache, lens, cu, window, "e4m3"))


def test_attention_many_empty_sequences(ops):
    """Runs of sequences without keys between others: each has rows, which see nothing."""
    g = gen(77)
    b, w, hk, ps, d, n = 300, 4, 2, 64, 64, 8
    cache = make_cache(g, b, w, hk, ps, d, "e4m3")
    lens = [0] * b
    for i in (0, 5, 6, 150, 299):
        lens[i] = 8 + 40 * (i % 7)
    q = torch.randn(b * n, 4 * hk, d, generator=g, device="cuda", dtype=torch.float16)
    cu = offsets([n] * b)
    check(*run_attend(ops, q, cache, lens, cu, 0, "e4m3"))


def test_empty_step(ops):
    table, kc, vc, ks, vs = make_cache(gen(50), 2, 1, 1, 16, 64, "e4m3")
    q = torch.empty(0, 4, 64, dtype=torch.float16, device="cuda")
    out, lse = ops.kv_attention(q, kc, vc, ks, vs, table, i32([3, 4]), i32([0, 0, 0]))
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    before = kc.clone()
    ops.kv_append(q[:, :1], q[:, :1], kc, vc, ks, vs, table, i32([3, 4]), i32([0, 0, 0]))
    assert torch.equal(kc, before)


@pytest.mark.parametrize("change, message", [
    (dict(fmt="fp4"), "fmt must be"),
    (dict(window=-1), "window must not be negative"),
    (dict(softmax_scale=math.inf), "softmax_scale must be finite"),
    (dict(q=lambda q: q.float()), "q must be fp16 or bf16"),
    (dict(q=lambda q: q[:, :3]), "heads must be a multiple of kv_heads"),
    (dict(q=lambda q: q[..., :32]), "head_dim"),
    (dict(q=lambda q: q.cpu()), "q must be a CUDA tensor"),
    (dict(q=lambda q: torch.cat([q, q[:1]])), "tokens / batch"),
    (dict(q=lambda q: q.transpose(1, 2).contiguous().transpose(1, 2)), "last dimension of q"),
    (dict(seq_lens=lambda x: x.long()), "seq_lens must be"),
    (dict(seq_lens=lambda x: x[:1]), "seq_lens must have shape"),
    (dict(page_table=lambda x: x[0]), "page_table must have shape"),
    (dict(cu_seqlens=lambda x: i32([0, 1])), "cu_seqlens must have shape"),
    (dict(k_scale=lambda x: x[:, :1].contiguous()), "k_scale / v_scale"),
    (dict(k_cache=lambda x: x[..., :48].contiguous(), v_cache=lambda x: x[..., :48].contiguous(), q=lambda q: q[..., :48]), "head_dim must be"),
    (dict(k_cache=lambda x: x[:, :, :12].contiguous(), v_cache=lambda x: x[:, :, :12].contiguous()), "page_size must be"),
    (dict(out=lambda x: torch.empty(2, 4, 64, device="cuda")), "out must be"),
])
def test_attention_refuses(ops, change, message):
    table, kc, vc, ks, vs = make_cache(gen(51), 2, 2, 2, 16, 64, "e4m3")
    args = dict(q=torch.randn(2, 4, 64, device="cuda").half(), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, page_table=table,
                seq_lens=i32([3, 30]), cu_seqlens=None, softmax_scale=None, window=0, fmt="e4m3", out=None)
    for name, f in change.items():
        args[name] = f(args[name]) if callable(f) else f
    with pytest.raises(RuntimeError, match=message):
        ops.kv_attention(**args)


def test_append_refuses(ops):
    table, kc, vc, ks, vs = make_cache(gen(52), 2, 2, 2, 16, 64, "e4m3")
    k = torch.randn(2, 2, 64, device="cuda").half()
    ln = i32([3, 30])
    with pytest.raises(RuntimeError, match="same dtype"):
        ops.kv_append(k, k.bfloat16(), kc, vc, ks, vs, table, ln)
    with pytest.raises(RuntimeError, match="must have shape"):
        ops.kv_append(k[:, :1], k[:, :1], kc, vc, ks, vs, table, ln)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.kv_append(k.expand(2, 2, 64).transpose(1, 2).contiguous().transpose(1, 2), k, kc, vc, ks, vs, table, ln)
