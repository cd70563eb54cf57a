// Attention of a step's queries over the paged 8-bit KV cache
// (fp8imma_kv_attention).
//
// Mathematics, per sequence and KV head, in base 2 (c = softmax_scale log2 e):
//   x_rj = c <q_r, K_j> ks,   w_rj = 2^(x_rj + log2 vs - M_r),
//   out_r = sum_j w_rj V_j / L_r,   L_r = sum_j w_rj / vs,   lse_r = ln2 (M_r + log2 L_r)
// with K_j, V_j the stored codes (exact in fp16) and ks, vs the scales of
// their page. Taking the value scale into the exponent keeps it out of the
// products: w is rounded to fp16 for the tensor cores relative to the largest
// weight *times scale* of the row so far, so a page with a large scale and a
// small weight is as precise as the other way round. M is a running reference
// that follows the maximum when it is exceeded by more than 2^8; sums, M and L
// are fp32.
//
// Bound: the cache is read once, 2 len D bytes a KV head; at up to ~64 query
// rows a KV head the products are far below the tensor rate, so the kernel is
// built to keep the copies running:
//  * one CTA per SM; a producer warp streams 128-key stages (one TMA box per
//    page for K and for V, 128-byte swizzle) through a 3..6 stage ring, page
//    ids fetched a batch of 32 ahead;
//  * the 128-key tiles of all (sequence, row tile, KV head) items are laid end
//    to end and cut into equal runs, one per CTA, whatever the lengths are
//    (lengths are read on the device). Items that several CTAs share are joined
//    by the last of them to finish, in CTA order, so results do not depend on
//    timing;
//  * K is the 16-row operand of mma.sync m16n8k16 (S^T = K Q^T: 16 keys x 8
//    query rows) and V^T likewise (O^T = V^T P^T), so 8 rows, one group of
//    heads, fill a tile. The order of channels within a product is free, so a
//    lane's operand is bytes that lie together in its key's row; key pairs of V
//    are interleaved with byte permutes; P^T comes from S^T by movmatrix.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

constexpr int kKeys = 128;                  // keys of a stage
constexpr int kConsumers = 8;               // consumer warps
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kSlots = kKeys / 16;          // pages of a stage at most
constexpr float kTinyScale = 7.888609e-31f; // 2^-100: value scales below count as this (values below 2^-91)
constexpr float kRaise = 8.0f;              // M follows the maximum when it lies this far above

struct AttnParams {
  fp8imma_kv_cache c;
  fp8imma_kv_attention_args a;
  int per_seq;   // > 0: every sequence has this many tokens
  int group;     // query heads per KV head
  int vec_q;     // query rows are 16-byte aligned
  int min_units; // tiles a CTA takes at least
  unsigned int* counters;  // per (item, row warp): finished parts; zero between calls
  float* parts;            // per (CTA, first / last segment, row warp): M, L, O of a shared item
};

// ---------------------------------------------------------------- helpers --

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
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
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
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
  int64_t item0;       // unit index of the item's first tile
  int64_t item;        // item index over all sequences
  int lo, hi;          // keys that some row of the tile sees: [lo, hi)
  int pos_min, pos_max;
};

// Walks the units [u, end) segment by segment.
struct Walk {
  int64_t u, end, base, item_base;  // base: first unit of sequence b, item_base: its first item
  int b;
  Seq s;
  __device__ __forceinline__ bool next(const AttnParams& p, int rows_per_tile, Segment& g) {
    if (u >= end) return false;
    int64_t items = (int64_t)s.row_tiles * p.c.kv_heads;
    while (u - base >= items * s.tiles) {  // u < end <= all units: ends at the last sequence
      base += items * s.tiles;
      item_base += items;
      s = load_seq(p, ++b, rows_per_tile);
      items = (int64_t)s.row_tiles * p.c.kv_heads;
    }
    const int64_t off = u - base;
    const int64_t it = off / s.tiles;
    g.b = b;
    g.rt = (int)(it / p.c.kv_heads);
    g.h = (int)(it % p.c.kv_heads);
    g.first = (int)(off - it * s.tiles);
    g.count = (int)min((int64_t)(s.tiles - g.first), end - u);
    g.item0 = base + it * s.tiles;
    g.item = item_base + it;
    const int r0 = g.rt * rows_per_tile, r1 = min(s.rows, r0 + rows_per_tile) - 1;
    g.pos_min = s.len - s.n + r0 / p.group;
    g.pos_max = s.len - s.n + r1 / p.group;
    g.lo = p.a.window > 0 ? (int)max((int64_t)0, (int64_t)g.pos_min - p.a.window + 1) : 0;
    g.hi = min(s.cap, g.pos_max + 1);
    u += g.count;
    return true;
  }
};

__device__ __forceinline__ int64_t run_begin(int64_t units, int ctas, int c) { return units * c / ctas; }
__device__ __forceinline__ int run_of(int64_t units, int ctas, int64_t u) {  // the CTA whose run holds unit u
  int c = (int)(u * ctas / units);
  while (run_begin(units, ctas, c + 1) <= u) ++c;
  while (run_begin(units, ctas, c) > u) --c;
  return c;
}

// Shapes of a variant: head_dim D, NT tiles of 8 query rows a warp, RW warps
// along the rows (8 / RW along the keys).
template <int D, int NT, int RW>
struct Shape {
  static constexpr int kRows = 8 * NT * RW;
  static constexpr int kKeyWarps = kConsumers / RW;
  static constexpr int kHalves = D == 256 ? 2 : 1;        // 128-byte column halves of a tile
  static constexpr int kTileBytes = kKeys * D;            // K (or V) of a stage
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kMT = D / 16;                      // 16-channel tiles of O^T
  static constexpr int kPartFloats = (kMT * NT * 4 + NT * 4) * 32;  // O, M and L of a warp, register by register
  static constexpr int kMergeBytes = kConsumers / 2 * kPartFloats * 4;
  static constexpr int kStages = (227 * 1024 - 2048 - kMergeBytes) / kStageBytes < 6 ? (227 * 1024 - 2048 - kMergeBytes) / kStageBytes : 6;
  static constexpr int kSmem = kStages * kStageBytes + kMergeBytes + 1024;
};

struct StageInfo {
  float ks[kSlots], vs[kSlots];
  int live[kSlots];  // the page exists
};

template <int FMT, int D, int NT, int RW>
__global__ void __launch_bounds__(kThreads, 1)
    kv_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const __grid_constant__ AttnParams p) {
  using S = Shape<D, NT, RW>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_full[S::kStages], s_empty[S::kStages];
  __shared__ StageInfo s_info[S::kStages];
  __shared__ int64_t s_scan[kThreads / 32], s_scan_items[kThreads / 32];
  __shared__ int64_t s_start[3];  // sequence, its first unit, its first item
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* merge = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)) + S::kStages * S::kStageBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], kConsumers);
    }
    fence_barrier_init();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }

  // this CTA's run of units
  int64_t units = 0;
  for (int b0 = 0; b0 < p.c.batch; b0 += kThreads) {
    int64_t n = 0;
    if (b0 + tid < p.c.batch) {
      const Seq s = load_seq(p, b0 + tid, S::kRows);
      n = (int64_t)s.row_tiles * p.c.kv_heads * s.tiles;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    __syncthreads();
    if (lane == 0) s_scan[warp] = n;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) units += s_scan[w];
  }
  if (units == 0) return;
  const int ctas = (int)min((int64_t)gridDim.x, (units + p.min_units - 1) / p.min_units);
  if ((int)blockIdx.x >= ctas) return;
  Walk walk;
  walk.u = run_begin(units, ctas, blockIdx.x);
  walk.end = run_begin(units, ctas, blockIdx.x + 1);
  {
    int64_t base = 0, base_i = 0;
    for (int b0 = 0; b0 < p.c.batch; b0 += kThreads) {
      int64_t n = 0, ni = 0;
      if (b0 + tid < p.c.batch) {
        const Seq s = load_seq(p, b0 + tid, S::kRows);
        ni = (int64_t)s.row_tiles * p.c.kv_heads;
        n = ni * s.tiles;
      }
      int64_t x = n, xi = ni;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o), yi = __shfl_up_sync(0xffffffffu, xi, o);
        if (lane >= o) {
          x += y;
          xi += yi;
        }
      }
      __syncthreads();
      if (lane == 31) {
        s_scan[warp] = x;
        s_scan_items[warp] = xi;
      }
      __syncthreads();
      int64_t before = base, before_i = base_i;
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) {
          before += s_scan[w];
          before_i += s_scan_items[w];
        }
        base += s_scan[w];
        base_i += s_scan_items[w];
      }
      const int64_t at = before + x - n;
      if (walk.u >= at && walk.u < at + n) {
        s_start[0] = b0 + tid;
        s_start[1] = at;
        s_start[2] = before_i + xi - ni;
      }
      if (walk.u < base) break;
    }
    __syncthreads();
    walk.b = (int)s_start[0];
    walk.base = s_start[1];
    walk.item_base = s_start[2];
    walk.s = load_seq(p, walk.b, S::kRows);
  }

  const int ps = p.c.page_size;
  Segment g;

  if (warp == kConsumers) {
    // ---------------------------------------------------------- producer --
    int stage = 0, issued = 0;
    uint32_t phase = 1;  // the ring starts empty
    bool ok = true;
    const int per_stage = kKeys / ps;  // pages of a stage
    const uint32_t page_bytes = (uint32_t)ps * D;
    while (ok && walk.next(p, S::kRows, g)) {
      const int tile_lo = walk.s.tile0 + g.first, tile_hi = tile_lo + g.count;
      const int* table = p.c.page_table + (size_t)g.b * p.c.max_pages;
      // tiles with keys that some row sees
      const int from = max(tile_lo, g.lo / kKeys), to = min(tile_hi, (g.hi + kKeys - 1) / kKeys);
      int ids = -1;
      auto fetch = [&](int tile) {  // ids of the 32 pages from `tile` on
        const int pi = tile * per_stage + lane;
        return pi < p.c.max_pages && pi * ps < g.hi && (pi + 1) * ps > g.lo ? __ldg(table + pi) : -1;
      };
      const int batch = 32 / per_stage;  // tiles of a batch
      int next_ids = from < to ? fetch(from) : -1;
      for (int tile = from; tile < to && ok; ++tile) {
        const int at = (tile - from) % batch * per_stage;
        float ks = 0.0f, vs = 0.0f;
        if (at == 0) {
          ids = next_ids;
          next_ids = tile + batch < to ? fetch(tile + batch) : -1;
        }
        const int page = __shfl_sync(0xffffffffu, ids, at + (lane < per_stage ? lane : 0));
        const bool live = lane < per_stage && (unsigned)page < (unsigned)p.c.num_pages;
        if (live) {
          const size_t ph = (size_t)page * p.c.kv_heads + g.h;
          ks = __ldg(p.c.k_scale + ph);
          vs = __ldg(p.c.v_scale + ph);
        }
        const uint32_t n_live = (uint32_t)__popc(__ballot_sync(0xffffffffu, live));
        ok = mbar_wait(&s_empty[stage], phase, ERR_WAIT_EMPTY);
        if (!ok) break;
        if (lane == 0 && n_live) {
          // one pending arrival stays until the scales are written below
          asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&s_full[stage])), "r"(n_live * 2 * page_bytes) : "memory");
        }
        __syncwarp();
        if (live) {
          uint8_t* dst = smem_raw + (smem_base - smem_u32(smem_raw)) + stage * S::kStageBytes;
          const int row = (page * p.c.kv_heads + g.h) * ps;  // key row of the whole pool
#pragma unroll
          for (int hf = 0; hf < S::kHalves; ++hf) {
            const int off = hf * (kKeys * 128) + lane * (int)(page_bytes / S::kHalves);
            const int y = D == 64 ? row >> 1 : row;
            tma_load_2d(dst + off, &map_k, &s_full[stage], hf * 128, y);
            tma_load_2d(dst + S::kTileBytes + off, &map_v, &s_full[stage], hf * 128, y);
          }
        }
        if (lane < kSlots) {
          s_info[stage].ks[lane] = ks;
          s_info[stage].vs[lane] = vs;
          s_info[stage].live[lane] = live;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_full[stage]);
        ++issued;
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok) {  // a wait ran out: let the copies in flight land before the CTA ends
      for (int i = 0; i < min(issued, S::kStages); ++i) {
        const int k = issued - 1 - i;
        mbar_wait(&s_full[k % S::kStages], (uint32_t)((k / S::kStages) & 1), ERR_WAIT_FULL);
      }
    }
    return;
  }

  // ------------------------------------------------------------ consumers --
  const int q4 = lane >> 2, t4 = lane & 3;  // row / column of the fragments
  const int rw = warp / S::kKeyWarps, kw = warp % S::kKeyWarps;
  // row of the group's 16 keys behind fragment row q4 (and q4 + 8): two keys
  // share a 128-byte line when D = 64, and this order keeps V's reads apart
  const int key_lo = D == 64 ? 4 * (q4 >> 1) + (q4 & 1) : q4;
  const int key_hi = D == 64 ? key_lo + 2 : q4 + 8;
  // V: keys behind this lane's operand pairs
  const int vkey[4] = {D == 64 ? 4 * t4 : 2 * t4, D == 64 ? 4 * t4 + 1 : 2 * t4 + 1, D == 64 ? 4 * t4 + 2 : 2 * t4 + 8,
                       D == 64 ? 4 * t4 + 3 : 2 * t4 + 9};
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  constexpr int QW = D / 8;  // 32-bit words of Q a lane and row: D / 4 channels
  uint32_t q[NT][QW];
  float cq[NT][2];
  int pos[NT][2];
  float o[S::kMT][NT][4], m[NT][2], l[NT][2];

  while (walk.next(p, S::kRows, g)) {
    const Seq s = walk.s;
    // queries of this lane: row q4 of each 8-row tile, channels t4 * 32 .. (D = 64: t4 * 16 ..; D = 256: in both halves)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = g.rt * S::kRows + (rw * NT + nt) * 8 + q4;
      const bool in = row < s.rows;
      const uint16_t* qp = static_cast<const uint16_t*>(p.a.q) +
                           (in ? (int64_t)(s.t0 + row / p.group) * p.a.q_token_stride + (int64_t)(g.h * p.group + row % p.group) * p.a.q_head_stride : 0);
      constexpr int W = D == 64 ? 8 : 16;  // words of a run of channels
#pragma unroll
      for (int hf = 0; hf < S::kHalves; ++hf) {
        const uint16_t* src = qp + hf * 128 + t4 * W * 2;
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) {
            if (p.vec_q) {
              v = __ldg(reinterpret_cast<const uint4*>(src + 2 * i));
            } else {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = (uint32_t)__ldg(src + 2 * (i + k)) | ((uint32_t)__ldg(src + 2 * (i + k) + 1) << 16);
              v = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          q[nt][hf * W + i] = v.x;
          q[nt][hf * W + i + 1] = v.y;
          q[nt][hf * W + i + 2] = v.z;
          q[nt][hf * W + i + 3] = v.w;
        }
      }
      float back = 1.0f;  // what the row was divided by
      if (p.a.a_type == FP8IMMA_A_BF16) {
        // bf16 -> fp16: the row is brought to a largest magnitude of 2^8 .. 2^9 by a power of two, which is exact
        // for everything within 2^22 of the largest
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < QW; ++i)
          big = fmaxf(big, fmaxf(fabsf(__uint_as_float(q[nt][i] << 16)), fabsf(__uint_as_float(q[nt][i] & 0xFFFF0000u))));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int e = (int)(__float_as_uint(big) >> 23) - 127 - 8;
        float f = 1.0f;
        if (big > 0.0f && big < INFINITY) {
          const int ec = max(-126, min(126, e));
          f = __uint_as_float((uint32_t)(127 - ec) << 23);
          back = __uint_as_float((uint32_t)(127 + ec) << 23);
        }
#pragma unroll
        for (int i = 0; i < QW; ++i) q[nt][i] = pack_f16(__uint_as_float(q[nt][i] << 16) * f, __uint_as_float(q[nt][i] & 0xFFFF0000u) * f);
      }
      // the columns 2 * t4, 2 * t4 + 1 of the S^T tiles are rows of this tile
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        cq[nt][c] = p.a.softmax_scale * 1.4426950408889634f * __shfl_sync(0xffffffffu, back, (2 * t4 + c) * 4);
        const int r = g.rt * S::kRows + (rw * NT + nt) * 8 + 2 * t4 + c;
        pos[nt][c] = r < s.rows ? s.len - s.n + r / p.group : -1;
        m[nt][c] = -INFINITY;
        l[nt][c] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < S::kMT; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[i][nt][c] = 0.0f;

    const int tile_lo = s.tile0 + g.first;
    const int from = max(tile_lo, g.lo / kKeys), to = min(tile_lo + g.count, (g.hi + kKeys - 1) / kKeys);
    for (int tile = from; tile < to; ++tile) {
      if (ok) ok = mbar_wait(&s_full[stage], phase, ERR_WAIT_FULL);
      const uint32_t kb = smem_base + stage * S::kStageBytes, vb = kb + S::kTileBytes;
      for (int gi = kw; gi < kKeys / 16; gi += S::kKeyWarps) {
        const int j0 = tile * kKeys + gi * 16, slot = gi * 16 / ps;
        if (!s_info[stage].live[slot] || j0 >= g.hi || j0 + 15 < g.lo) continue;  // warp-uniform: nothing of it is seen
        const float ks = s_info[stage].ks[slot], vs0 = s_info[stage].vs[slot];
        const float vs = vs0 < kTinyScale ? kTinyScale : vs0, lvs = lg2(vs), ivs = __fdividef(1.0f, vs);
        // some row does not see some key of the group
        const bool edge = j0 + 15 > g.pos_min || j0 + 15 >= g.hi || (p.a.window > 0 && j0 <= g.pos_max - p.a.window);

        // S^T = K Q^T, two chains of sums
        float sa[NT][4], sb[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) sa[nt][c] = sb[nt][c] = 0.0f;
        const int r_lo = gi * 16 + key_lo, r_hi = gi * 16 + key_hi;
#pragma unroll
        for (int hf = 0; hf < S::kHalves; ++hf) {
          constexpr int W = D == 64 ? 4 : 8;  // words of K a lane and key (and half)
          uint32_t ka[W], kc[W];
#pragma unroll
          for (int i = 0; i < W; i += 4) {
            uint32_t xa, xc;
            if (D == 64) {
              xa = (uint32_t)((r_lo >> 1) * 128 + (((((r_lo & 1) << 2) + t4) ^ ((r_lo >> 1) & 7)) << 4));
              xc = (uint32_t)((r_hi >> 1) * 128 + (((((r_hi & 1) << 2) + t4) ^ ((r_hi >> 1) & 7)) << 4));
            } else {
              xa = (uint32_t)(hf * (kKeys * 128) + r_lo * 128 + (((2 * t4 + i / 4) ^ (r_lo & 7)) << 4));
              xc = (uint32_t)(hf * (kKeys * 128) + r_hi * 128 + (((2 * t4 + i / 4) ^ (r_hi & 7)) << 4));
            }
            const uint4 a = lds128(kb + xa), c = lds128(kb + xc);
            ka[i] = a.x, ka[i + 1] = a.y, ka[i + 2] = a.z, ka[i + 3] = a.w;
            kc[i] = c.x, kc[i + 1] = c.y, kc[i + 2] = c.z, kc[i + 3] = c.w;
          }
#pragma unroll
          for (int i = 0; i < W; ++i) {
            uint32_t a0, a2, a1, a3;
            f8x4_to_f16x4<FMT>(ka[i], a0, a2);
            f8x4_to_f16x4<FMT>(kc[i], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(i & 1 ? sb[nt] : sa[nt], a0, a1, a2, a3, q[nt][2 * (hf * W + i)], q[nt][2 * (hf * W + i) + 1]);
          }
        }
        bool raise = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float x = fmaf(sa[nt][c] + sb[nt][c], cq[nt][c & 1] * ks, lvs);
            if (edge) {
              const int j = j0 + (c < 2 ? key_lo : key_hi), pc = pos[nt][c & 1];
              if (j > pc || j >= g.hi || (p.a.window > 0 && j <= pc - p.a.window)) x = -INFINITY;
            }
            sa[nt][c] = x;
            raise |= x > m[nt][c & 1] + kRaise;
          }
        }
        if (__any_sync(0xffffffffu, raise)) {  // some row's maximum has moved
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = fmaxf(sa[nt][c], sa[nt][c + 2]);
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
              const float mn = fmaxf(m[nt][c], x);
              const float f = mn == m[nt][c] ? 1.0f : ex2(m[nt][c] - mn);
              m[nt][c] = mn;
              l[nt][c] *= f;
#pragma unroll
              for (int i = 0; i < S::kMT; ++i) {
                o[i][nt][c] *= f;
                o[i][nt][c + 2] *= f;
              }
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 4; ++c) sa[nt][c] = ex2(sa[nt][c] - (m[nt][c & 1] == -INFINITY ? 0.0f : m[nt][c & 1]));
          l[nt][0] = fmaf(sa[nt][0] + sa[nt][2], ivs, l[nt][0]);
          l[nt][1] = fmaf(sa[nt][1] + sa[nt][3], ivs, l[nt][1]);
          pb[nt][0] = transpose_8x8(pack_f16(sa[nt][0], sa[nt][1]));
          pb[nt][1] = transpose_8x8(pack_f16(sa[nt][2], sa[nt][3]));
        }

        // O^T += V^T P^T
        bool odd_values = false;
#pragma unroll
        for (int hf = 0; hf < S::kHalves; ++hf) {
          constexpr int W = D == 64 ? 2 : 4;  // words of V a lane and key (and half): channels q4 * 4 W ..
          uint32_t v[4][W];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = gi * 16 + vkey[k];
            if (D == 64) {
              const uint2 x = lds64(vb + (r >> 1) * 128 + (((((r & 1) << 2) + (q4 >> 1)) ^ ((r >> 1) & 7)) << 4) + (q4 & 1) * 8);
              v[k][0] = x.x, v[k][1] = x.y;
            } else {
              const uint4 x = lds128(vb + hf * (kKeys * 128) + r * 128 + ((q4 ^ (r & 7)) << 4));
              v[k][0] = x.x, v[k][1] = x.y, v[k][W - 2] = x.z, v[k][W - 1] = x.w;
            }
            if (edge) {
              // a key that no row sees may hold anything, a key that some row does not see must not reach it by 0 * NaN
              const int j = j0 + vkey[k];
              const bool gone = j >= g.hi || j < g.lo;
#pragma unroll
              for (int i = 0; i < W; ++i) {
                if (gone) v[k][i] = 0u;
                if (nonfinite4<FMT>(v[k][i])) odd_values = true;
              }
            }
          }
          if (edge && __any_sync(0xffffffffu, odd_values)) {
            // rare: take the non-finite codes out of the product and add them to the rows that see them
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int i = 0; i < W; ++i) {
                const uint32_t mk = FMT == F8_E4M3 ? 0x7F7F7F7Fu : 0x7C7C7C7Cu;
                v[k][i] &= ~__vcmpeq4(v[k][i] & mk, mk);
              }
            for (int k = 0; k < 16; ++k) {
              const int fr = D == 64 ? ((k >> 2) * 2 + (k & 1) + (k & 2) * 4) : k;  // fragment row of key k
              float pv[NT][2];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const float lo = __shfl_sync(0xffffffffu, sa[nt][c], (fr & 7) * 4 + t4), hi = __shfl_sync(0xffffffffu, sa[nt][c + 2], (fr & 7) * 4 + t4);
                  pv[nt][c] = fr < 8 ? lo : hi;
                }
              const int r = gi * 16 + k, j = j0 + k;
              if (j >= g.hi || j < g.lo) continue;
#pragma unroll
              for (int i = 0; i < 2 * W; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int ch = q4 * 4 * W + 2 * i + e;  // channel within the half
                  const uint32_t a = D == 64 ? (r >> 1) * 128 + (((((r & 1) << 2) + (ch >> 4)) ^ ((r >> 1) & 7)) << 4) + (ch & 15)
                                             : hf * (kKeys * 128) + r * 128 + (((ch >> 4) ^ (r & 7)) << 4) + (ch & 15);
                  uint32_t byte;
                  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(byte) : "r"(vb + a));
                  const float val = f8_to_f32<FMT>((uint8_t)byte);
                  if (!(fabsf(val) < INFINITY)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                      for (int c = 0; c < 2; ++c)
                        if (pv[nt][c] != 0.0f) o[hf * 2 * W + i][nt][c + 2 * e] += pv[nt][c] * val;
                  }
                }
            }
          }
#pragma unroll
          for (int i = 0; i < W; ++i) {
            uint32_t a0, a1, a2, a3;
            f8x4_to_f16x4<FMT>(__byte_perm(v[0][i], v[1][i], 0x5140), a0, a1);
            f8x4_to_f16x4<FMT>(__byte_perm(v[2][i], v[3][i], 0x5140), a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[hf * 2 * W + 2 * i][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
            f8x4_to_f16x4<FMT>(__byte_perm(v[0][i], v[1][i], 0x7362), a0, a1);
            f8x4_to_f16x4<FMT>(__byte_perm(v[2][i], v[3][i], 0x7362), a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[hf * 2 * W + 2 * i + 1][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[stage]);
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }

    // ------------------------------------------- join the key warps' parts --
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 4);
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 8);
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 16);
      }
    // a part: O register by register, then M and L, one value a lane; `f` visits each
    auto put = [&](float* dst) {
#pragma unroll
      for (int i = 0; i < S::kMT; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          *reinterpret_cast<float4*>(dst + ((i * NT + nt) * 32 + lane) * 4) = make_float4(o[i][nt][0], o[i][nt][1], o[i][nt][2], o[i][nt][3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        *reinterpret_cast<float4*>(dst + ((S::kMT * NT + nt) * 32 + lane) * 4) = make_float4(m[nt][0], m[nt][1], l[nt][0], l[nt][1]);
    };
    auto add = [&](const float* src, bool global) {  // joins another part to this one
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float4* x = reinterpret_cast<const float4*>(src + ((S::kMT * NT + nt) * 32 + lane) * 4);
        const float4 ml = global ? __ldcg(x) : *x;
        const float m0 = fmaxf(m[nt][0], ml.x), m1 = fmaxf(m[nt][1], ml.y);
        const float a0 = m[nt][0] == m0 ? 1.0f : ex2(m[nt][0] - m0), a1 = m[nt][1] == m1 ? 1.0f : ex2(m[nt][1] - m1);
        const float b0 = ml.x == m0 ? 1.0f : ex2(ml.x - m0), b1 = ml.y == m1 ? 1.0f : ex2(ml.y - m1);
        m[nt][0] = m0;
        m[nt][1] = m1;
        l[nt][0] = l[nt][0] * a0 + ml.z * b0;
        l[nt][1] = l[nt][1] * a1 + ml.w * b1;
#pragma unroll
        for (int i = 0; i < S::kMT; ++i) {
          const float4* y = reinterpret_cast<const float4*>(src + ((i * NT + nt) * 32 + lane) * 4);
          const float4 v = global ? __ldcg(y) : *y;
          o[i][nt][0] = o[i][nt][0] * a0 + v.x * b0;
          o[i][nt][1] = o[i][nt][1] * a1 + v.y * b1;
          o[i][nt][2] = o[i][nt][2] * a0 + v.z * b0;
          o[i][nt][3] = o[i][nt][3] * a1 + v.w * b1;
        }
      }
    };
#pragma unroll
    for (int half = S::kKeyWarps / 2; half > 0; half >>= 1) {
      if (kw >= half && kw < 2 * half) put(merge + (rw * (S::kKeyWarps / 2) + kw - half) * S::kPartFloats);
      named_bar_sync(1, kConsumers * 32);
      if (kw < half) add(merge + (rw * (S::kKeyWarps / 2) + kw) * S::kPartFloats, false);
      named_bar_sync(1, kConsumers * 32);
    }
    if (kw != 0) continue;

    bool write = true;
    if (g.count != s.tiles) {
      // the item is shared by CTAs c0 .. c1: each leaves its part, the last to come joins them in order
      const int c0 = run_of(units, ctas, g.item0), c1 = run_of(units, ctas, g.item0 + s.tiles - 1);
      auto part = [&](int c) {  // a CTA's first segment lies in slot 0, its last in slot 1
        return p.parts + ((int64_t)(c * 2 + (g.item0 > run_begin(units, ctas, c) ? 1 : 0)) * RW + rw) * S::kPartFloats;
      };
      put(part(blockIdx.x));
      __threadfence();
      __syncwarp();
      unsigned int prev = 0;
      unsigned int* ctr = p.counters + g.item * RW + rw;
      if (lane == 0) asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(prev) : "l"(ctr) : "memory");
      prev = __shfl_sync(0xffffffffu, prev, 0);
      write = prev == (unsigned)(c1 - c0);
      if (write) {
        __threadfence();
        if (lane == 0) *ctr = 0;  // ready for the next call
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          m[nt][0] = m[nt][1] = -INFINITY;
          l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
          for (int i = 0; i < S::kMT; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
        }
        for (int c = c0; c <= c1; ++c) add(part(c), true);
      }
    }
    if (!write) continue;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = g.rt * S::kRows + (rw * NT + nt) * 8 + 2 * t4 + c;
        if (row >= s.rows) continue;
        const int64_t at = (int64_t)(s.t0 + row / p.group) * p.a.heads + g.h * p.group + row % p.group;
        const float L = l[nt][c], inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
        uint16_t* out = static_cast<uint16_t*>(p.a.out) + at * D;
        constexpr int W = D == 64 ? 2 : 4;
#pragma unroll
        for (int hf = 0; hf < S::kHalves; ++hf)
#pragma unroll
          for (int i = 0; i < 2 * W; i += 4) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float x = o[hf * 2 * W + i + k][nt][c] * inv, y = o[hf * 2 * W + i + k][nt][c + 2] * inv;
              w[k] = p.a.a_type == FP8IMMA_A_F16 ? pack_f16(x, y)
                                                 : (uint32_t)f32_to_a16<1>(x) | ((uint32_t)f32_to_a16<1>(y) << 16);
            }
            *reinterpret_cast<uint4*>(out + hf * 128 + q4 * 4 * W + 2 * i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        if (p.a.lse && q4 == 0) p.a.lse[at] = L == 0.0f ? -INFINITY : 0.6931471805599453f * (m[nt][c] + log2f(L));
      }
  }
}

template <int FMT, int D, int NT, int RW>
cudaError_t launch(AttnParams& p, cudaStream_t st) {
  using S = Shape<D, NT, RW>;
  static_assert(S::kStages >= 2, "ring too short");
  const auto kern = kv_attention_kernel<FMT, D, NT, RW>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), S::kSmem);
  if (e != cudaSuccess) return e;
  // 128-byte rows: two keys a row when D = 64, half a key when D = 256
  CUtensorMap mk, mv;
  const uint64_t bytes = (uint64_t)p.c.num_pages * p.c.kv_heads * p.c.page_size * D;
  const uint64_t inner = D == 256 ? 256 : 128;
  const uint32_t box_rows = (uint32_t)(D == 64 ? p.c.page_size / 2 : p.c.page_size);
  e = make_tmap_2d_u8(&mk, p.c.k, inner, bytes / inner, inner, 128, box_rows, true);
  if (e == cudaSuccess) e = make_tmap_2d_u8(&mv, p.c.v, inner, bytes / inner, inner, 128, box_rows, true);
  if (e != cudaSuccess) return e;
  const int64_t items = ((int64_t)p.c.tokens * p.group / S::kRows + p.c.batch) * p.c.kv_heads;
  const int64_t tiles = ((int64_t)p.c.max_pages * p.c.page_size + kKeys - 1) / kKeys;
  const int grid = (int)std::min<int64_t>(num_sms_current(), std::max<int64_t>(1, items * tiles));
  const size_t ctr_bytes = (size_t)items * RW * 4, part_bytes = (size_t)grid * 2 * RW * S::kPartFloats * 4;
  ScopedScratch ctr, part;
  e = ctr.get(ctr_bytes, st, kScratchAttn);
  if (e == cudaSuccess && ctr.owned) e = cudaMemsetAsync(ctr.ptr, 0, ctr_bytes, st);
  if (e == cudaSuccess) e = part.get(part_bytes, st, kScratchAttnParts);
  if (e == cudaSuccess) {
    p.counters = static_cast<unsigned int*>(ctr.ptr);
    p.parts = static_cast<float*>(part.ptr);
    kern<<<grid, kThreads, S::kSmem, st>>>(mk, mv, p);
    e = cudaGetLastError();
  }
  const cudaError_t e1 = ctr.release(st), e2 = part.release(st);
  return e != cudaSuccess ? e : e1 != cudaSuccess ? e1 : e2;
}

// Query rows a CTA works on at once: the rows of a sequence and KV head
// (group times its tokens, on average) rounded up, so that few rows do not pay
// for empty ones and many rows read the cache once.
template <int FMT>
cudaError_t launch_d(AttnParams& p, cudaStream_t st) {
  const int64_t rows = ((int64_t)p.c.tokens * p.group + p.c.batch - 1) / p.c.batch;
  if (p.c.head_dim == 256) {
    if (rows <= 8) return launch<FMT, 256, 1, 1>(p, st);
    if (rows <= 16) return launch<FMT, 256, 1, 2>(p, st);
    if (rows <= 32) return launch<FMT, 256, 1, 4>(p, st);
    return launch<FMT, 256, 1, 8>(p, st);
  }
  if (p.c.head_dim == 128) {
    if (rows <= 8) return launch<FMT, 128, 1, 1>(p, st);
    if (rows <= 16) return launch<FMT, 128, 2, 1>(p, st);
    if (rows <= 32) return launch<FMT, 128, 2, 2>(p, st);
    return launch<FMT, 128, 2, 4>(p, st);
  }
  if (rows <= 8) return launch<FMT, 64, 1, 1>(p, st);
  if (rows <= 16) return launch<FMT, 64, 2, 1>(p, st);
  if (rows <= 32) return launch<FMT, 64, 2, 2>(p, st);
  return launch<FMT, 64, 2, 4>(p, st);
}

}  // namespace

unsigned int attn_device_error(bool clear) { return fp8imma_dev::tu_device_error(clear); }
cudaError_t attn_set_wait_limit(unsigned long long ns) { return fp8imma_dev::tu_set_wait_limit(ns); }

}  // namespace fp8imma_b200

using namespace fp8imma_b200;

extern "C" int fp8imma_kv_attention(const fp8imma_kv_cache* c, const fp8imma_kv_attention_args* a, void* stream) {
  FP8IMMA_RANGE("fp8imma_kv_attention");
  const cudaError_t e = kv_cache_check(c);
  if (e != cudaSuccess) return (int)e;
  if (!a || !a->q || !a->out || a->a_type < 0 || a->a_type > 1) return (int)cudaErrorInvalidValue;
  if (a->heads <= 0 || a->heads % c->kv_heads || a->heads > 65535 || a->window < 0) return (int)cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(a->q) & 1u) return (int)cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(a->out) & 15u) return (int)cudaErrorInvalidValue;
  if ((int64_t)c->tokens * (a->heads / c->kv_heads) > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  AttnParams p = {};
  p.c = *c;
  p.a = *a;
  p.per_seq = c->cu_new ? 0 : c->tokens / c->batch;
  p.group = a->heads / c->kv_heads;
  p.vec_q = ((reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)((a->q_token_stride | a->q_head_stride) * 2)) & 15u) == 0;
  p.min_units = 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return (int)(c->format == FP8IMMA_B_E4M3 ? launch_d<F8_E4M3>(p, st) : launch_d<F8_E5M2>(p, st));
}
