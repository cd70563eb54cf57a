// What the two kernels of the cache attention share (kv_attention_few.cuh: few
// query rows a KV head; kv_attention_tc.cu: many): the cut of the work into equal
// runs of 128-key tiles, and the join of parts.
#pragma once

#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "sm100_async.cuh"

#include <algorithm>
#include <cstring>

namespace fp8imma_b200 {
namespace attn {

using namespace fp8imma_dev;

constexpr int kKeys = 128;                  // keys of a tile
constexpr float kTinyScale = 7.888609e-31f; // 2^-100: value scales below count as this (values below 2^-91)
constexpr float kRaise = 8.0f;              // M follows the maximum when it lies this far above

// What kv_attention_tree adds; the kernels' TREE variants read it.
struct TreeParams {
  const uint32_t* mask;      // null: the step is causal
  const int32_t* positions;  // null: a token's place
  int words;
  float cap2, by, twice;     // cap log2 e (0: scores as they are), 1 / cap2, 2 log2 e / cap2
  unsigned long long poly[7];  // cap2 times the coefficients below, twice each: pairs for fma.f32x2
};
// Scores are capped in base 2: with x = s log2 e, y = x / cap2,
//   cap tanh(s / cap) log2 e = cap2 tanh y = y cap2 P(y^2)  for |y| <= 1,
// P(w) = tanh(sqrt w) / sqrt w on 0 <= w <= 1 by a minimax fit of degree 6, to 2^-24
// relative (2^-21.8 as 32 bits evaluate it, scaling and all), whatever the cap: no power
// of it enters but the first.
// A cap counts as 2^-30 at least and 2^99 at most: below, all scores lie within 2^-29 of
// one another, and above, tanh changes no score that lies below 2^87.
inline void set_cap(TreeParams& t, float cap) {
  static const double c[7] = {0.9999999403953552, -0.33332839608192444, 0.13325203955173492, -0.05345702916383743,
                              0.020289979875087738, -0.006203379016369581, 0.0010410225950181484};
  const double cap2 = cap > 0.0f ? std::min(std::max((double)cap, 0x1p-30), 0x1p99) * 1.4426950408889634 : 0.0;
  t.cap2 = (float)cap2;
  t.by = cap > 0.0f ? (float)(1.0 / cap2) : 0.0f;
  t.twice = cap > 0.0f ? (float)(2.8853900817779268 / cap2) : 0.0f;
  for (int i = 0; i < 7; ++i) {
    const float d = (float)(c[i] * cap2);
    unsigned int bits;
    static_assert(sizeof(bits) == sizeof(d), "");
    std::memcpy(&bits, &d, sizeof(bits));
    t.poly[i] = (unsigned long long)bits << 32 | bits;
  }
}

struct AttnParams {
  fp8imma_kv_cache c;
  fp8imma_kv_attention_args a;
  int per_seq;   // > 0: every sequence has this many tokens
  int group;     // query heads per KV head
  int vec_q;     // query rows are 16-byte aligned
  int copy;      // pages are copied by lanes instead of TMA
  unsigned int* counters;  // per item: finished parts; zero between calls
  float* parts;            // per (CTA, first / last segment, row warp): M, L, O of a shared item
  TreeParams t;
};

// ---------------------------------------------------------------- helpers --

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// The capped score in base 2 of x = s log2 e beyond the polynomial's range, by
// tanh y = 1 - 2 / (1 + e^2y). It is off by cap2 2^-22 wherever y lies, so what is
// small beside the cap takes the polynomial.
__device__ __forceinline__ float cap_far(const TreeParams& t, float x) {
  return fmaf(-2.0f * t.cap2, __fdividef(1.0f, 1.0f + ex2(x * t.twice)), t.cap2);
}
// near where |y| <= 1; in asm, since the compiler makes a branch of it at which lanes part
__device__ __forceinline__ float cap_pick(float y, float near, float far) {
  float r;
  asm("{\n\t.reg .pred p;\n\tsetp.le.f32 p, %1, 0f3F800000;\n\tselp.f32 %0, %2, %3, p;\n\t}" : "=f"(r) : "f"(fabsf(y)), "f"(near), "f"(far));
  return r;
}
__device__ __forceinline__ float cap_score(const TreeParams& t, float x) {
  const float y = x * t.by, u = y * y;
  float q = __uint_as_float((uint32_t)t.poly[6]);
#pragma unroll
  for (int i = 5; i >= 0; --i) q = fmaf(u, q, __uint_as_float((uint32_t)t.poly[i]));
  return cap_pick(y, y * q, cap_far(t, x));
}
// 16 bytes global -> shared, asynchronously
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// two outputs in the activation type
__device__ __forceinline__ uint32_t out_pair(float lo, float hi, int a_type) {
  if (a_type == FP8IMMA_A_F16) return pack_f16(lo, hi);
  return (uint32_t)f32_to_a16<1>(lo) | ((uint32_t)f32_to_a16<1>(hi) << 16);
}

// NaN or infinite code among the four bytes
template <int FMT>
__device__ __forceinline__ bool nonfinite4(uint32_t w) {
  const uint32_t m = FMT == F8_E4M3 ? 0x7F7F7F7Fu : 0x7C7C7C7Cu;
  return __vcmpeq4(w & m, m) != 0u;
}

// One sequence of the step.
struct Seq {
  int t0, n;      // its packed tokens
  int len;        // as given; the last token's position is len - 1
  int cap;        // keys that the page table holds
  int rows;       // n * group
  int tile0;      // first 128-key tile that any row sees
  int tiles;      // tiles of each item, 1 at least
  int row_tiles;
};

__device__ __forceinline__ Seq load_seq(const AttnParams& p, int b, int rows_per_tile) {
  Seq s;
  if (p.per_seq > 0) {
    s.t0 = b * p.per_seq;
    s.n = p.per_seq;
  } else {
    s.t0 = max(0, __ldg(p.c.cu_new + b));
    s.n = max(0, min(__ldg(p.c.cu_new + b + 1), p.c.tokens) - s.t0);
  }
  s.len = __ldg(p.c.seq_lens + b);
  s.cap = max(0, min(s.len, p.c.max_pages * p.c.page_size));
  s.rows = s.n * p.group;
  s.row_tiles = (s.rows + rows_per_tile - 1) / rows_per_tile;
  s.tile0 = p.a.window > 0 ? (int)max((int64_t)0, (int64_t)s.len - s.n - p.a.window + 1) / kKeys : 0;
  s.tiles = max(1, (s.cap + kKeys - 1) / kKeys - s.tile0);
  return s;
}

// A run of tiles of one item (sequence, row tile, KV head).
struct Segment {
  int b, rt, h;
  int first, count;    // tiles [first, first + count) of the item
  int item0;           // unit index of the item's first tile
  int item;            // item index over all sequences
  int lo, hi;          // keys that some row of the tile sees: [lo, hi)
  int pos_min, pos_max;
};

// Walks the units [u, end) segment by segment.
struct Walk {
  int u, end, base, item_base;  // base: first unit of sequence b, item_base: its first item
  int b;
  Seq s;
  template <bool TREE = false>
  __device__ __forceinline__ bool next(const AttnParams& p, int rows_per_tile, Segment& g) {
    if (u >= end) return false;
    int items = s.row_tiles * p.c.kv_heads;
    while (u - base >= items * s.tiles) {  // u < end <= all units: ends at the last sequence
      base += items * s.tiles;
      item_base += items;
      s = load_seq(p, ++b, rows_per_tile);
      items = s.row_tiles * p.c.kv_heads;
    }
    const int off = u - base, it = off / s.tiles;
    g.b = b;
    g.rt = it / p.c.kv_heads;
    g.h = it % p.c.kv_heads;
    g.first = off - it * s.tiles;
    g.count = min(s.tiles - g.first, end - u);
    g.item0 = base + it * s.tiles;
    g.item = item_base + it;
    const int r0 = g.rt * rows_per_tile, r1 = min(s.rows, r0 + rows_per_tile) - 1;
    g.pos_min = s.len - s.n + r0 / p.group;
    g.pos_max = s.len - s.n + r1 / p.group;
    g.lo = p.a.window > 0 ? (int)max((int64_t)0, (int64_t)g.pos_min - p.a.window + 1) : 0;
    g.hi = min(s.cap, g.pos_max + 1);
    if (TREE && p.t.mask) {
      // any of the step's keys may be seen by any row; all rows see the keys before it, up to the window
      g.pos_min = s.len - s.n - 1;
      g.pos_max = s.len - 1;
      g.lo = p.a.window > 0 ? (int)max((int64_t)0, (int64_t)s.len - s.n - p.a.window + 1) : 0;
      g.hi = s.cap;
    }
    u += g.count;
    return true;
  }
};

// A row's token as the mask sees it.
template <bool TREE>
struct Sight {
  int pos;                // its place, for the window (below all places: no row)
  int start;              // the step's first place
  const uint32_t* mask;   // its mask row, null: causal
  __device__ __forceinline__ void set(const AttnParams& p, const Seq& s, int row) {
    const bool in = row < s.rows;
    const int tok = row / p.group;
    pos = in ? s.len - s.n + tok : TREE ? -(1 << 30) : -1;  // with a mask places below 0 have rows too
    if (TREE) {
      start = s.len - s.n;
      mask = nullptr;
      if (p.t.mask) {
        mask = p.t.mask + (in ? (int64_t)(s.t0 + tok) * p.t.words : 0);
        if (in && p.t.positions) pos = min(max(__ldg(p.t.positions + s.t0 + tok), start), s.len - 1);
      }
    }
  }
  // key j < cap
  __device__ __forceinline__ bool sees(const AttnParams& p, int j) const {
    if (TREE && p.t.mask) {
      const int k = j - start;
      if (k >= 0) return pos >= start && (k >> 5) < p.t.words && ((__ldg(mask + (k >> 5)) >> (k & 31)) & 1u);
      return pos >= start && (p.a.window == 0 || j > pos - p.a.window);
    }
    return j <= pos && (p.a.window == 0 || j > pos - p.a.window);
  }
  // keys j0 .. j0 + 31 as bits, without regard to the cache's end
  __device__ __forceinline__ uint32_t sees32(const AttnParams& p, int j0) const {
    const bool tree = TREE && p.t.mask;
    // before the step (or all of them): first <= j < last
    const int first = p.a.window > 0 ? (int)max((int64_t)0, (int64_t)pos - p.a.window + 1) : 0, last = tree ? (pos >= start ? start : 0) : pos + 1;
    const int a = min(max(first - j0, 0), 32), b = min(max(last - j0, 0), 32);
    uint32_t bits = b > a ? (b == 32 ? 0xffffffffu : (1u << b) - 1u) & ~((1u << a) - 1u) : 0u;
    if (tree && pos >= start && j0 + 31 >= start) {
      const int k = j0 - start, w = k >> 5;  // bit k of the mask row is key j0's
      const uint32_t lo = w >= 0 && w < p.t.words ? __ldg(mask + w) : 0u;
      const uint32_t hi = w + 1 < p.t.words ? __ldg(mask + w + 1) : 0u;
      bits |= __funnelshift_r(lo, hi, k & 31);
    }
    return bits;
  }
};

// CTA c's run of the units: they differ by one in length at most.
struct Runs {
  int per, rem;
  __device__ __forceinline__ Runs(int units, int ctas) : per(units / ctas), rem(units % ctas) {}
  __device__ __forceinline__ int begin(int c) const { return c * per + min(c, rem); }
  __device__ __forceinline__ int of(int u) const {  // the CTA whose run holds unit u
    const int cut = rem * (per + 1);
    return u < cut ? u / (per + 1) : rem + (u - cut) / per;
  }
};

// This CTA's run of units, by a scan of the sequences' units and items; all
// threads of the CTA take part. False: it has none, or the offsets of the step's
// tokens do not ascend (two sequences could own a row, and their items would be
// more than the counters that the host has made room for).
template <int THREADS>
__device__ __forceinline__ bool find_run(const AttnParams& p, int rows_per_tile, Walk& walk, int& units, int& ctas) {
  __shared__ int s_scan[2][THREADS / 32];
  __shared__ int s_start[3];  // sequence, its first unit, its first item
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  units = 0;
  int items = 0, n = 0, ni = 0, at = 0, at_i = 0;
  bool bad = false;
  auto scan = [&](int b0) {  // of sequences b0 .. b0 + THREADS: this thread's start, the running totals
    n = ni = 0;
    if (b0 + tid < p.c.batch) {
      const Seq s = load_seq(p, b0 + tid, rows_per_tile);
      bad |= p.per_seq == 0 && __ldg(p.c.cu_new + b0 + tid + 1) < __ldg(p.c.cu_new + b0 + tid);
      ni = s.row_tiles * p.c.kv_heads;
      n = ni * s.tiles;
    }
    int x = n, xi = ni;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o), yi = __shfl_up_sync(0xffffffffu, xi, o);
      if (lane >= o) {
        x += y;
        xi += yi;
      }
    }
    __syncthreads();
    if (lane == 31) {
      s_scan[0][warp] = x;
      s_scan[1][warp] = xi;
    }
    bad = __syncthreads_or(bad);
    at = units + x - n;
    at_i = items + xi - ni;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) {
        at += s_scan[0][w];
        at_i += s_scan[1][w];
      }
      units += s_scan[0][w];
      items += s_scan[1][w];
    }
  };
  for (int b0 = 0; b0 < p.c.batch; b0 += THREADS) scan(b0);
  if (bad) {
    if (tid == 0) atomicCAS(&g_fp8imma_device_error, 0u, (unsigned int)ERR_BAD_OFFSETS);
    return false;
  }
  if (units == 0) return false;
  ctas = min((int)gridDim.x, units);
  if ((int)blockIdx.x >= ctas) return false;
  const Runs runs(units, ctas);
  walk.u = runs.begin(blockIdx.x);
  walk.end = runs.begin(blockIdx.x + 1);
  const int all = units;
  if (p.c.batch > THREADS) units = items = 0;
  for (int b0 = 0; b0 < p.c.batch; b0 += THREADS) {
    if (p.c.batch > THREADS) scan(b0);
    if (walk.u >= at && walk.u < at + n) {
      s_start[0] = b0 + tid;
      s_start[1] = at;
      s_start[2] = at_i;
    }
  }
  units = all;
  __syncthreads();
  walk.b = s_start[0];
  walk.base = s_start[1];
  walk.item_base = s_start[2];
  walk.s = load_seq(p, walk.b, rows_per_tile);
  return true;
}

// What the output of an item needs to know.
struct Item {
  int t0, rows, rt, h;
};
struct Shared {  // an item that several CTAs worked on
  Item item;
  int index, item0, c0, c1, last;
};

// Parts of a softmax joined: reference, sum and output of two rows. Eight parts
// are asked for at a time, so the join waits for memory once per eight.
struct Joined {
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  template <class ML, class O>
  __device__ __forceinline__ void join(int n, ML ml, O part) {
    constexpr int B = 8;
#pragma unroll 1
    for (int k = 0; k < n; k += B) {
      float4 x[B], y[B];
#pragma unroll
      for (int e = 0; e < B; ++e) {
        x[e] = make_float4(-INFINITY, -INFINITY, 0.0f, 0.0f);
        y[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (k + e < n) {
          x[e] = ml(k + e);
          y[e] = part(k + e);
        }
      }
      float n0 = m0, n1 = m1;
#pragma unroll
      for (int e = 0; e < B; ++e) {
        n0 = fmaxf(n0, x[e].x);
        n1 = fmaxf(n1, x[e].y);
      }
      const float s0 = n0 == -INFINITY ? 0.0f : n0, s1 = n1 == -INFINITY ? 0.0f : n1;
      const float g0 = ex2(m0 - s0), g1 = ex2(m1 - s1);
      m0 = n0;
      m1 = n1;
      l0 *= g0;
      l1 *= g1;
      o = make_float4(o.x * g0, o.y * g1, o.z * g0, o.w * g1);
#pragma unroll
      for (int e = 0; e < B; ++e) {
        const float f0 = ex2(x[e].x - s0), f1 = ex2(x[e].y - s1);
        l0 = fmaf(x[e].z, f0, l0);
        l1 = fmaf(x[e].w, f1, l1);
        o.x = fmaf(y[e].x, f0, o.x);
        o.y = fmaf(y[e].y, f1, o.y);
        o.z = fmaf(y[e].z, f0, o.z);
        o.w = fmaf(y[e].w, f1, o.w);
      }
    }
  }
};

}  // namespace attn

// Many query rows a KV head: products by tcgen05 (kv_attention_tc.cu, kv_attention_tree_tc.cu).
cudaError_t launch_attention_tc(attn::AttnParams& p, cudaStream_t st);
cudaError_t launch_attention_tree_tc(attn::AttnParams& p, cudaStream_t st);
// Whether they take `rows` query rows of a sequence and KV head (kv_attention.cu).
bool attention_tc_pays(const attn::AttnParams& p, int64_t rows);
int attention_tc_forced();  // the number of rows set by fp8imma_set_attention_tc_rows, 0: none

}  // namespace fp8imma_b200
