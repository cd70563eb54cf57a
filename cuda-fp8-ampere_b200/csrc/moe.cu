// Mixture-of-experts layer with FP8 weights for 1 .. 64 tokens
// (fp8imma_moe_forward), in one launch.
//
// Mathematics: r = x Wr^T (fp32), S_t the top_k experts of token t, p the
// softmax; per chosen (token, expert) slot
//   h = act(sg (x Wg^T)) * (su (x Wu^T)),  out_t = sum_S p sd (h Wd^T).
// FP8 codes are multiplied as fp16 (exact); sums are fp32, scales are applied
// to the sums. x enters as it is when it is fp16; a bf16 row is brought into
// fp16's range by a power of two (exact within 2^22 of the row's largest). h
// is rounded to fp16 (2^-11; 16 bits are what the tensor cores take) as 16
// columns at a time come out of a unit, after a power of two that brings their
// largest magnitude to 2^-1 .. 2^15, where nothing is lost that matters beside
// it (2^-24 of it). These powers lie 16 octaves apart, counted from the one that
// a slot's columns are expected to take: |act(g) u| <= |g| |u|, a gate or up sum
// is at most max_i s_i * fmax * sum |x|, and the largest h of well-spread
// weights lie some 2^16 below that. So the columns of a row nearly always share
// one, and the down product takes them as they are; a unit with a row whose
// columns do not brings them to the row's largest as it reads them. Doing so in
// every unit, with powers one octave apart, took 222 us instead of 197 for 64
// tokens; one power a row, taken from the bound alone, loses small rows beside
// scales that no weight uses.
//
// Bound: a few tokens use each weight byte a few times, so the layer costs the
// bytes of the chosen experts. One cooperative grid, one CTA per SM, keeps
// their stream running through the whole layer:
//  0. router logits (warps over experts x tokens), x to fp16 in operand order,
//     the experts' largest scales; grid barrier; every CTA picks the top_k of
//     all tokens for itself
//  1. gate / up: the chosen experts' row groups are laid end to end and cut
//     into equal runs; a unit is 8 RU gate rows and the same 8 RU up rows, so
//     that both factors of h meet in one fragment; grid barrier
//  2. down: the same over units of 16 RU rows; slot results to scratch; barrier
//  3. out = sum over a token's slots, in their order
// A warp works on units of its own, or a team of 2, 4 or 8 warps shares one
// along the columns. Each warp streams the 128-byte column blocks of its units
// by TMA, one box of 16 RU rows a block, into a ring of its own, across unit
// and phase boundaries: no barrier between warps, and the down weights are
// under way while the grid meets at the barrier before them. A box covers the
// gate and the up rows (a 3-D map over [columns, inter, experts x 2]): copies
// of 4 KB reach 6.6 TB/s, copies of 2 KB 3.8 TB/s, 16-byte asynchronous copies
// of 64-byte row pieces 5.6 TB/s. A team's sums meet in shared memory in a
// fixed order; nothing depends on timing.
//
// Measured: 64 tokens, 4 of 32 experts, 4096 x 2048: 202 us (4.0 TB/s of the
// 806 MB); 8 tokens, 2 of 8 experts, 4096 x 11008: 172 to 198 us by the board and
// the run (4.9 to 5.6 TB/s of 0.97 GB, 75 to 87% of a copy); one token, 6 of 64
// experts, 2048 x 1408: 29 us, of which the bytes are 8: the router's chain and
// three grid barriers come on top.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>
#include <type_traits>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

constexpr int kMaxSlots = FP8IMMA_MOE_MAX_TOKENS * FP8IMMA_MOE_MAX_TOP_K;
constexpr int kLeft = 3, kRouterDone = 64, kSteps = 128, kScaleMax = kSteps + 2 * kMaxSlots, kSyncWords = kScaleMax + 2 * FP8IMMA_MOE_MAX_EXPERTS;
constexpr int kBias = 64;  // above the magnitude of every step of h's powers

struct MoeParams {
  fp8imma_moe_args a;
  // kept zero between calls: three barrier counters, CTAs that have left (kLeft),
  // finished router units of each group of tokens (from kRouterDone on), kBias +
  // the highest and kBias - the lowest step of each slot's columns that are not
  // zero (from kSteps on, [slots, 2]), the experts' largest gate / up scales as
  // bits (from kScaleMax on, [experts, 2])
  unsigned int* sync;
  float* logits;       // [tokens, experts]
  uint16_t* xf;        // [tokens, hidden padded to 128] fp16, operand order
  float* xback;        // [tokens, 2] what a row of xf is to be multiplied by, sum |x|
  int* ids;            // [slots] the choice
  float* weights;      // [slots]
  uint16_t* h;         // [slots, inter padded to 128] fp16, operand order
  signed char* step;   // [slots, a 16th of that] of 16 columns of h: value = h * 2^(base + 16 step - 14), base by slot
  float* part;         // [slots, hidden]
  int hpad, ipad;
};

// ---------------------------------------------------------------- helpers --

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // e: -126 .. 127
// v * 2^e for e of -252 .. 254, in two products
__device__ __forceinline__ float times_pow2(float v, int e) { return v * pow2(e >> 1) * pow2(e - (e >> 1)); }
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float gate_act(float v, int act) {
  if (act == 3) return __fdividef(v, 1.0f + __expf(-v));
  return 0.5f * v * (1.0f + tanhf(0.7978845608028654f * (v + 0.044715f * v * v * v)));
}
// order-preserving integer of a logit: -0 = +0, NaN above everything
__device__ __forceinline__ int order_key(float v) {
  const int k = __float_as_int(v);
  if (isnan(v)) return 0x7fffffff;
  return k < 0 ? (int)(0x80000000u - (unsigned)k) : k;
}
// Power of two that brings a row with the largest magnitude `big` to 2^8 ..
// 2^9 (1 for zero and non-finite rows), and its inverse.
__device__ __forceinline__ void row_factor(float big, float& f, float& back) {
  f = back = 1.0f;
  if (big > 0.0f && big < INFINITY) {
    const int e = max(-126, min(126, (int)(__float_as_uint(big) >> 23) - 127 - 8));
    f = __uint_as_float((uint32_t)(127 - e) << 23);
    back = __uint_as_float((uint32_t)(127 + e) << 23);
  }
}

// All CTAs of the (cooperative) grid meet. False when the wait ran out.
__device__ __forceinline__ bool grid_barrier(unsigned int* ctr) {
  __shared__ int s_ok;
  __syncthreads();
  if (threadIdx.x == 0) {
    // the CTA's writes are ordered before the release by the barrier above
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(ctr) : "memory");
    unsigned int v = 0;
    bool ok = true;
    const unsigned long long t0 = globaltimer_ns();
    for (;;) {
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(ctr) : "memory");
      if (v >= gridDim.x) break;
      const unsigned long long dt = globaltimer_ns() - t0;
      if (dt > kWaitCheckNs && dt > *(volatile unsigned long long*)&g_fp8imma_wait_limit_ns) {
        atomicCAS(&g_fp8imma_device_error, 0u, (unsigned int)ERR_WAIT_GRID);
        ok = false;
        break;
      }
    }
    s_ok = ok;
  }
  __syncthreads();
  return s_ok != 0;
}

// A warp's report that its CTA has read and written the sync words for the last
// time in this call. Every CTA makes it once, whichever of its waits ran out, so
// the last one leaves them zero for the next call also after a failed barrier.
__device__ __forceinline__ void leave(unsigned int* sync, int experts, int slots, int lane) {
  unsigned int before = 0;
  if (lane == 0) asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(sync + kLeft) : "memory");
  before = __shfl_sync(0xffffffffu, before, 0);
  if (before != gridDim.x - 1) return;
  for (int i = lane; i < kSteps + 2 * slots; i += 32) sync[i] = 0u;
  for (int i = lane; i < 2 * experts; i += 32) sync[kScaleMax + i] = 0u;
}

struct Runs {  // CTA c's run of the units: they differ by one in length at most
  int per, rem;
  __device__ __forceinline__ Runs(int units, int ctas) : per(units / ctas), rem(units % ctas) {}
  __device__ __forceinline__ int begin(int c) const { return c * per + min(c, rem); }
};

// 3-D tiled TMA load (no multicast) into this CTA's shared memory
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// NT: 8-token tiles of a unit at most; RU: 16-row tiles of a unit; WARPS a CTA;
// DEPTH: blocks of a warp's ring.
template <int NT, int RU, int WARPS, int DEPTH>
struct Shape {
  static_assert(RU % 2 == 0, "a unit's gate rows are whole groups of 16 columns of h");
  static constexpr int kThreads = WARPS * 32;
  static constexpr int kBlockBytes = 2048 * RU;
  static constexpr int kRing = DEPTH * kBlockBytes;    // of a warp
  static constexpr int kFragFloats = RU * NT * 4 * 32; // a unit's sums of a warp
  static constexpr int kSmem = 1024 + WARPS * (kRing + kFragFloats * 4);
};

// A token's top_k by one warp: rounds of the largest logit not yet taken, the
// lowest index among equal ones. A lane keeps the keys of experts lane + 32 i.
template <int NK>
__device__ __noinline__ void pick(const float* r, int E, int K, int renormalize, int* ids, float* weights, int* ids_out, float* weights_out, int lane) {
  constexpr int kNone = (int)0x80000000;  // below the key of every logit
  int key[NK];
  float z = 0.0f;
#pragma unroll
  for (int i = 0; i < NK; ++i) key[i] = lane + 32 * i < E ? order_key(__ldcg(r + lane + 32 * i)) : kNone;
  auto value = [](int k) { return __int_as_float(k < 0 ? (int)(0x80000000u - (unsigned)k) : k); };
  int mine = 0;  // lane s keeps the s-th choice
  float first = 0.0f, sum = 0.0f, weight = 0.0f;
#pragma unroll 1
  for (int s = 0; s < K; ++s) {
    int best = key[0];
#pragma unroll
    for (int i = 1; i < NK; ++i) best = max(best, key[i]);
    const int top = __reduce_max_sync(0xffffffffu, best);
    int at = 0x7fffffff;
#pragma unroll
    for (int i = NK - 1; i >= 0; --i) at = key[i] == top ? lane + 32 * i : at;
    const int e = __reduce_min_sync(0xffffffffu, at);
    if (s == 0) {
      first = value(top);
      if (!renormalize)
#pragma unroll
        for (int i = 0; i < NK; ++i) z += key[i] == kNone ? 0.0f : __expf(value(key[i]) - first);
    }
#pragma unroll
    for (int i = 0; i < NK; ++i)
      if (lane + 32 * i == e) key[i] = kNone;
    const float w = __expf(value(top) - first);
    sum += w;
    if (lane == s) {
      mine = e;
      weight = w;
    }
  }
  if (!renormalize) sum = warp_sum(z);
  if (lane < K) {
    weight = __fdiv_rn(weight, sum);
    ids[lane] = mine;
    weights[lane] = weight;
    if (ids_out) ids_out[lane] = mine;
    if (weights_out) weights_out[lane] = weight;
  }
}

// Router logits of EX experts x TX tokens a warp; the warp that finishes the
// last of a group of tokens makes their choice.
template <int AT, int EX, int TX>
__device__ __forceinline__ void router(const MoeParams& p, int wid, int nw, int lane, bool vec) {
  const int eu = (p.a.experts + EX - 1) / EX, tu = (p.a.tokens + TX - 1) / TX;
  const uint16_t* X = static_cast<const uint16_t*>(p.a.x);
  const uint16_t* R = static_cast<const uint16_t*>(p.a.router);
  for (int u = wid; u < eu * tu; u += nw) {
    const int e0 = u % eu * EX, t0 = u / eu * TX;
    float s[EX][TX];
#pragma unroll
    for (int e = 0; e < EX; ++e)
#pragma unroll
      for (int t = 0; t < TX; ++t) s[e][t] = 0.0f;
    if (vec) {
#pragma unroll 2
      for (int k = lane * 8; k < p.a.hidden; k += 256) {
        uint4 w[EX], x[TX];
#pragma unroll
        for (int e = 0; e < EX; ++e) w[e] = __ldg(reinterpret_cast<const uint4*>(R + (size_t)min(e0 + e, p.a.experts - 1) * p.a.hidden + k));
#pragma unroll
        for (int t = 0; t < TX; ++t) x[t] = __ldg(reinterpret_cast<const uint4*>(X + min(t0 + t, p.a.tokens - 1) * p.a.x_token_stride + k));
#pragma unroll
        for (int t = 0; t < TX; ++t) {
          const uint32_t xx[4] = {x[t].x, x[t].y, x[t].z, x[t].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x0 = a16_to_f32<AT>((uint16_t)(xx[i] & 0xFFFFu)), x1 = a16_to_f32<AT>((uint16_t)(xx[i] >> 16));
#pragma unroll
            for (int e = 0; e < EX; ++e) {
              const uint32_t ww = i == 0 ? w[e].x : i == 1 ? w[e].y : i == 2 ? w[e].z : w[e].w;
              s[e][t] = fmaf(x0, a16_to_f32<AT>((uint16_t)(ww & 0xFFFFu)), s[e][t]);
              s[e][t] = fmaf(x1, a16_to_f32<AT>((uint16_t)(ww >> 16)), s[e][t]);
            }
          }
        }
      }
    } else {
      for (int k = lane; k < p.a.hidden; k += 32)
#pragma unroll
        for (int t = 0; t < TX; ++t) {
          const float x0 = a16_to_f32<AT>(__ldg(X + min(t0 + t, p.a.tokens - 1) * p.a.x_token_stride + k));
#pragma unroll
          for (int e = 0; e < EX; ++e) s[e][t] = fmaf(x0, a16_to_f32<AT>(__ldg(R + (size_t)min(e0 + e, p.a.experts - 1) * p.a.hidden + k)), s[e][t]);
        }
    }
#pragma unroll
    for (int e = 0; e < EX; ++e)
#pragma unroll
      for (int t = 0; t < TX; ++t) {
        const float v = warp_sum(s[e][t]);
        if (lane == 0 && e0 + e < p.a.experts && t0 + t < p.a.tokens) p.logits[(size_t)(t0 + t) * p.a.experts + e0 + e] = v;
      }
    unsigned int done = 0, *ctr = p.sync + kRouterDone + u / eu;
    if (lane == 0) asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(done) : "l"(ctr) : "memory");
    done = __shfl_sync(0xffffffffu, done, 0);
    __syncwarp();
    if (done == (unsigned)(eu - 1)) {
#pragma unroll 1
      for (int t = t0; t < min(t0 + TX, p.a.tokens); ++t) {
        const int at = t * p.a.top_k;
        const float* r = p.logits + (size_t)t * p.a.experts;
        int* ids_out = p.a.ids ? p.a.ids + at : nullptr;
        float* w_out = p.a.weights ? p.a.weights + at : nullptr;
        if (p.a.experts <= 128) pick<4>(r, p.a.experts, p.a.top_k, p.a.renormalize, p.ids + at, p.weights + at, ids_out, w_out, lane);
        else if (p.a.experts <= 256) pick<8>(r, p.a.experts, p.a.top_k, p.a.renormalize, p.ids + at, p.weights + at, ids_out, w_out, lane);
        else pick<32>(r, p.a.experts, p.a.top_k, p.a.renormalize, p.ids + at, p.weights + at, ids_out, w_out, lane);
      }
    }
  }
}

// Place of element k of a row in operand order: lane t4 of a fragment holds
// bytes 32 t4 .. 32 t4 + 31 of a 128-byte weight block, four bytes a product
// step; eight fp16, two steps, lie together.
__device__ __forceinline__ int place(int k) { return (k & ~127) + (((k & 31) >> 3) << 5) + (((k >> 5) & 3) << 3) + (k & 7); }

// Largest gate / up scales of each expert, a warp 1024 of them at a time.
__device__ __forceinline__ void scale_maxima(const MoeParams& p, int wid, int nw, int lane) {
  const int chunks = (p.a.inter + 1023) >> 10;
#pragma unroll 1
  for (int u = wid; u < p.a.experts * 2 * chunks; u += nw) {
    const int row = u / chunks, c = u - row * chunks;  // row: expert * 2 + (gate, up)
    const float* s = p.a.s_gate_up + (size_t)row * p.a.inter;
    const int hi = min(p.a.inter, c * 1024 + 1024);
    float m = 0.0f;
#pragma unroll 8
    for (int i = c * 1024 + lane; i < hi; i += 32) m = fmaxf(m, fabsf(__ldg(s + i)));
    const unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    if (lane == 0) atomicMax(p.sync + kScaleMax + row, bits);
  }
}

// A token's row as fp16 in operand order, its factor and sum |x|; one CTA.
template <int AT, int THREADS>
__device__ __forceinline__ void convert_row(const MoeParams& p, int t, bool vec) {
  __shared__ float s_big[THREADS / 32], s_sum[THREADS / 32];
  const uint16_t* x = static_cast<const uint16_t*>(p.a.x) + t * p.a.x_token_stride;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto load8 = [&](int k) {
    if (vec) return __ldg(reinterpret_cast<const uint4*>(x + k));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldg(x + k + 2 * i) | ((uint32_t)__ldg(x + k + 2 * i + 1) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  float big = 0.0f, sum = 0.0f;
  for (int k = threadIdx.x * 8; k < p.a.hidden; k += THREADS * 8) {
    const uint4 v = load8(k);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = fabsf(a16_to_f32<AT>((uint16_t)(w[i] & 0xFFFFu))), b = fabsf(a16_to_f32<AT>((uint16_t)(w[i] >> 16)));
      big = fmaxf(big, fmaxf(a, b));
      sum += a + b;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  sum = warp_sum(sum);
  __syncthreads();
  if (lane == 0) {
    s_big[warp] = big;
    s_sum[warp] = sum;
  }
  __syncthreads();
  big = sum = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    big = fmaxf(big, s_big[w]);
    sum += s_sum[w];
  }
  float f = 1.0f, back = 1.0f;
  if (AT == 1) row_factor(big, f, back);
  for (int k = threadIdx.x * 8; k < p.hpad; k += THREADS * 8) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k < p.a.hidden) {
      v = load8(k);
      if (AT == 1) {
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_f16(__uint_as_float(w[i] << 16) * f, __uint_as_float(w[i] & 0xFFFF0000u) * f);
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    *reinterpret_cast<uint4*>(p.xf + (size_t)t * p.hpad + place(k)) = v;
  }
  if (threadIdx.x == 0) {
    p.xback[2 * t] = back;
    p.xback[2 * t + 1] = sum;
  }
}

// An entry is up to 8 NT tokens of a chosen expert.
constexpr int kMaxEntries = FP8IMMA_MOE_MAX_EXPERTS + kMaxSlots / 8;
struct Lists {
  unsigned long long tokens[FP8IMMA_MOE_MAX_EXPERTS];  // tokens that chose the expert
  short first[FP8IMMA_MOE_MAX_EXPERTS];                // an expert's first place in `slot`
  short expert[kMaxEntries];                           // of an entry, ascending
  short start[kMaxEntries + 1];                        // its first place in `slot`
  short slot[kMaxSlots];                               // slots by expert, tokens ascending
  short token[kMaxSlots];                              // and their tokens
  short id[kMaxSlots];                                 // expert of a slot
  float weight[kMaxSlots];                             // p of a slot
  short base[kMaxSlots];                               // exponent that a slot's columns of h are expected to take
  short power[kMaxSlots];                              // the one that its row enters the down product with
  unsigned char mixed[kMaxSlots];                      // its columns do not share it
  float xback[FP8IMMA_MOE_MAX_TOKENS];
  int entries;
  int scan[16];
};

template <int FMT, int NT, int RU, int WARPS, int DEPTH>
__global__ void __launch_bounds__(WARPS * 32, 1)
    moe_kernel(const __grid_constant__ CUtensorMap map_up, const __grid_constant__ CUtensorMap map_down, const __grid_constant__ MoeParams p) {
  using S = Shape<NT, RU, WARPS, DEPTH>;
  constexpr int kThreads = S::kThreads;
  constexpr int CH = NT * RU <= 2 ? 2 : 1;  // chains of dependent products a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ Lists L;
  __shared__ uint64_t s_full[WARPS][DEPTH];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q4 = lane >> 2, t4 = lane & 3;
  uint8_t* const base = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  uint8_t* const ring = base + warp * S::kRing;
  float* const frags = reinterpret_cast<float*>(base + WARPS * S::kRing);
  const int T = p.a.tokens, E = p.a.experts, K = p.a.top_k, H = p.a.hidden, I = p.a.inter;

  if (lane == 0) {
    for (int i = 0; i < DEPTH; ++i) mbar_init(&s_full[warp][i], 1);
    fence_barrier_init();
    prefetch_tensormap(warp & 1 ? &map_down : &map_up);
  }

  // ------------------------------------------------- 0: router, x to fp16 --
  {
    // warps of the grid, CTA by CTA, so that few units spread over many SMs
    const int wid = warp * gridDim.x + blockIdx.x, nw = WARPS * gridDim.x;
    const bool vec = ((reinterpret_cast<uintptr_t>(p.a.x) | reinterpret_cast<uintptr_t>(p.a.router) | (uintptr_t)(p.a.x_token_stride * 2)) & 15u) == 0;
    const bool bf = p.a.a_type == FP8IMMA_A_BF16;
    for (int t = gridDim.x - 1 - blockIdx.x; t < T; t += gridDim.x) {  // the last CTAs: with few router units they have none
      if (bf) convert_row<1, kThreads>(p, t, vec);
      else convert_row<0, kThreads>(p, t, vec);
    }
    // one token and expert a warp while that is one round of the grid's warps; then four experts, then four tokens as well
    if (E * T <= nw) {
      if (bf) router<1, 1, 1>(p, wid, nw, lane, vec);
      else router<0, 1, 1>(p, wid, nw, lane, vec);
    } else if (((E + 3) >> 2) * T <= nw) {
      if (bf) router<1, 4, 1>(p, wid, nw, lane, vec);
      else router<0, 4, 1>(p, wid, nw, lane, vec);
    } else {
      if (bf) router<1, 4, 4>(p, wid, nw, lane, vec);
      else router<0, 4, 4>(p, wid, nw, lane, vec);
    }
    scale_maxima(p, ((warp + WARPS / 2) % WARPS) * gridDim.x + blockIdx.x, nw, lane);  // from the middle warps on: the first have router units
  }
  for (int e = tid; e < E; e += kThreads) L.tokens[e] = 0ull;
  if (!grid_barrier(p.sync)) {
    if (warp == 0) leave(p.sync, E, T * K, lane);
    return;
  }

  // ---------------------------------------------------------------- lists --
  if (tid < T) L.xback[tid] = __ldcg(p.xback + 2 * tid);
  for (int s = tid; s < T * K; s += kThreads) {
    const int t = s / K, e = __ldcg(p.ids + s);
    const float l1 = __ldcg(p.xback + 2 * t + 1);
    L.weight[s] = __ldcg(p.weights + s);
    L.id[s] = (short)e;
    atomicOr(&L.tokens[e], 1ull << t);
    // gate sums are below 2^(eg + 1), up sums below 2^(eu + 1), h is expected 2^16 below their product
    const float fmax_v = FMT == F8_E4M3 ? 448.0f : 57344.0f;
    const uint2 m = __ldcg(reinterpret_cast<const uint2*>(p.sync + kScaleMax) + e);
    const int eg = (int)(__float_as_uint(__uint_as_float(m.x) * fmax_v * l1) >> 23) - 127, eu = (int)(__float_as_uint(__uint_as_float(m.y) * fmax_v * l1) >> 23) - 127;
    L.base[s] = (short)max(-120, min(120, eg + eu - 7));
  }
  __syncthreads();
  {
    int entries = 0, slots = 0;
#pragma unroll 1
    for (int e0 = 0; e0 < E; e0 += kThreads) {
      const int e = e0 + tid;
      const unsigned long long m = e < E ? L.tokens[e] : 0ull;
      const int n = __popcll(m), ne = (n + 8 * NT - 1) / (8 * NT);
      int x = n | (ne << 16);  // slots and entries so far
      const int own = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      __syncthreads();
      if (lane == 31) L.scan[warp] = x;
      __syncthreads();
      int before = slots | (entries << 16), total = 0;
#pragma unroll 1
      for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += L.scan[w];
        total += L.scan[w];
      }
      before += x - own;
      for (int k = 0; k < ne; ++k) {
        L.expert[(before >> 16) + k] = (short)e;
        L.start[(before >> 16) + k] = (short)((before & 0xFFFF) + k * 8 * NT);
      }
      if (e < E) L.first[e] = (short)(before & 0xFFFF);
      slots += total & 0xFFFF;
      entries += total >> 16;
    }
    if (tid == 0) {
      L.entries = entries;
      L.start[entries] = (short)slots;
    }
  }
  __syncthreads();
  for (int s = tid; s < T * K; s += kThreads) {  // slots by expert, tokens ascending
    const int t = s / K, at = L.first[L.id[s]] + __popcll(L.tokens[L.id[s]] & ((1ull << t) - 1ull));
    L.slot[at] = (short)s;
    L.token[at] = (short)t;
  }
  __syncthreads();

  // --------------------------------------------------- the weights' stream --
  // Units of the two phases, this CTA's runs of them, the teams that share one.
  const int entries = L.entries;
  const int per1 = (I + 8 * RU - 1) / (8 * RU), per2 = (H + 16 * RU - 1) / (16 * RU);
  const int nb1 = p.hpad >> 7, nb2 = p.ipad >> 7;
  const Runs runs1(entries * per1, gridDim.x), runs2(entries * per2, gridDim.x);
  const int u1 = runs1.begin(blockIdx.x), n1 = runs1.begin(blockIdx.x + 1) - u1;
  const int u2 = runs2.begin(blockIdx.x), n2 = runs2.begin(blockIdx.x + 1) - u2;
  auto team_of = [](int longest) {  // warps that share a unit: more than one only where each team has one unit
    int ks = 1;
    while (ks < 8 && longest * ks * 2 <= WARPS) ks *= 2;
    return ks;
  };
  const int ks1 = team_of(runs1.per + (runs1.rem > 0)), ks2 = team_of(runs2.per + (runs2.rem > 0));

  // loading side of this warp: the next block to ask for
  int lp = 1, lu = warp / ks1, lb = warp % ks1, issued = 0, used = 0, lost = 0, lrow = 0, lexp = 0;
  bool ok = true;
  auto unit_at = [&]() {
    const int per = lp == 1 ? per1 : per2, u = (lp == 1 ? u1 : u2) + lu, a = u / per;
    lexp = L.expert[a];
    lrow = (u - a * per) * (lp == 1 ? 8 * RU : 16 * RU);
  };
  auto seek = [&]() {  // to the next block when the unit's are done
    if (lp == 1 && lb >= nb1) {
      lb = warp % ks1, lu += WARPS / ks1;
      if (lu < n1) {
        unit_at();
      } else {
        lp = 2, lu = warp / ks2, lb = warp % ks2;
        if (lu < n2 && lb < nb2) unit_at();
        else lp = 3;
      }
    } else if (lp == 2 && lb >= nb2) {
      lb = warp % ks2, lu += WARPS / ks2;
      if (lu < n2) unit_at();
      else lp = 3;
    }
  };
  if (lu < n1 && lb < nb1) {
    unit_at();
  } else {
    lu = n1, lb = nb1;
    seek();
  }
  auto issue = [&]() {
    if (lp == 3 || !ok) return;
    const int st = issued % DEPTH;
    if (lane == 0) {
      mbar_arrive_expect_tx(&s_full[warp][st], S::kBlockBytes);
      tma_load_3d(ring + st * S::kBlockBytes, lp == 1 ? &map_up : &map_down, &s_full[warp][st], lb * 128, lrow, lp == 1 ? 2 * lexp : lexp);
    }
    ++issued;
    lb += lp == 1 ? ks1 : ks2;
    seek();
  };
  auto next_block = [&]() {  // waits for it; after a wait that ran out the rest is passed over
    const int st = used % DEPTH;
    if (ok) {
      ok = mbar_wait(&s_full[warp][st], (uint32_t)((used / DEPTH) & 1), ERR_WAIT_FULL);
      if (!ok) lost = used;
    }
    ++used;
    return ring + st * S::kBlockBytes;
  };
  auto drain = [&]() {  // before an early end: the copies under way land first
    for (int k = ok ? used : lost; k < issued; ++k) mbar_wait(&s_full[warp][k % DEPTH], (uint32_t)((k / DEPTH) & 1), ERR_WAIT_FULL);
  };
#pragma unroll 1
  for (int i = 0; i < DEPTH; ++i) issue();

  float acc[CH][RU][NT][4];
  auto clear = [&]() {
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int r = 0; r < RU; ++r)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[k][r][nt][c] = 0.0f;
  };
  // Sums of the chains, then of the team's warps, in the first warp's
  // registers; false for the others.
  auto gather = [&](int ks) {
    if (CH == 2)
#pragma unroll
      for (int r = 0; r < RU; ++r)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[0][r][nt][c] += acc[CH - 1][r][nt][c];
    if (ks == 1) return true;
    if (warp % ks) {
#pragma unroll
      for (int r = 0; r < RU; ++r)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          *reinterpret_cast<float4*>(frags + warp * S::kFragFloats + ((r * NT + nt) * 32 + lane) * 4) =
              make_float4(acc[0][r][nt][0], acc[0][r][nt][1], acc[0][r][nt][2], acc[0][r][nt][3]);
    }
    named_bar_sync(1 + warp / ks, ks * 32);
    if (warp % ks) {
      named_bar_sync(1 + warp / ks, ks * 32);  // the first warp has read them
      return false;
    }
#pragma unroll 1
    for (int w = warp + 1; w < warp + ks; ++w)
#pragma unroll
      for (int r = 0; r < RU; ++r)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float4 v = *reinterpret_cast<const float4*>(frags + w * S::kFragFloats + ((r * NT + nt) * 32 + lane) * 4);
          acc[0][r][nt][0] += v.x;
          acc[0][r][nt][1] += v.y;
          acc[0][r][nt][2] += v.z;
          acc[0][r][nt][3] += v.w;
        }
    named_bar_sync(1 + warp / ks, ks * 32);
    return true;
  };
  // One block's products: fp16 rows xr (8 NT of them, operand order) times the
  // ring's next block. Mixed rows of h come to their row's power as they are read:
  // half of a lane's places are 16 columns.
  const uint16_t* xr[NT];
  int slot_of[NT];
  auto multiply = [&](int kb, int tiles, auto mixed) {
    char2 st[NT];
    if (mixed)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        st[nt] = xr[nt] ? *reinterpret_cast<const char2*>(p.step + (size_t)slot_of[nt] * (p.ipad >> 4) + kb * 8 + t4 * 2) : make_char2(0, 0);
    auto to_row = [&](uint4 (&v)[2], int nt, int j) {
      if (!mixed || !xr[nt]) return;
      const int top = (L.power[slot_of[nt]] - L.base[slot_of[nt]]) >> 4;
      // columns three steps below the row's are zero beside it
      const float f = pow2(8 * max((j ? st[nt].y : st[nt].x) - top, -3));
      const uint32_t ff = pack_f16(f, f);
      auto scaled = [&](uint32_t w) { return mul_f16x2(mul_f16x2(w, ff), ff); };  // twice: 2^-32 is below fp16's range, the product need not be
#pragma unroll
      for (int i = 0; i < 2; ++i) v[i] = make_uint4(scaled(v[i].x), scaled(v[i].y), scaled(v[i].z), scaled(v[i].w));
    };
    uint4 x[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) x[nt][i] = xr[nt] ? *reinterpret_cast<const uint4*>(xr[nt] + kb * 128 + i * 32) : make_uint4(0, 0, 0, 0);
    const uint8_t* w = next_block();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) to_row(x[nt], nt, 0);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint4 g[RU], b[RU], y[NT][2];
#pragma unroll
      for (int r = 0; r < RU; ++r) {
        const int at = (r * 8 + q4) * 128 + (((2 * t4 + j) ^ q4) << 4);
        g[r] = *reinterpret_cast<const uint4*>(w + at);
        b[r] = *reinterpret_cast<const uint4*>(w + 1024 * RU + at);
      }
      if (j == 0) {  // the second half's operands, while the first half is multiplied
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) y[nt][i] = xr[nt] ? *reinterpret_cast<const uint4*>(xr[nt] + kb * 128 + (2 + i) * 32) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t A[RU][4];
#pragma unroll
        for (int r = 0; r < RU; ++r) {
          f8x4_to_f16x4<FMT>(i == 0 ? g[r].x : i == 1 ? g[r].y : i == 2 ? g[r].z : g[r].w, A[r][0], A[r][2]);
          f8x4_to_f16x4<FMT>(i == 0 ? b[r].x : i == 1 ? b[r].y : i == 2 ? b[r].z : b[r].w, A[r][1], A[r][3]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (nt > 0 && nt >= tiles) break;
          const uint4 v = x[nt][i / 2];
#pragma unroll
          for (int r = 0; r < RU; ++r) mma_f16(acc[i % CH][r][nt], A[r][0], A[r][1], A[r][2], A[r][3], i & 1 ? v.z : v.x, i & 1 ? v.w : v.y);
        }
      }
      if (j == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) x[nt][i] = y[nt][i];
          to_row(x[nt], nt, 1);
        }
      }
    }
    __syncwarp();
    issue();  // into the place of the block just read
  };

  // ------------------------------------------------ 1: gate, up, activation --
#pragma unroll 1
  for (int u = warp / ks1; u < n1; u += WARPS / ks1) {
    const int a = (u1 + u) / per1, i0 = (u1 + u - a * per1) * (8 * RU);
    const int s0 = L.start[a], cnt = min(L.start[a + 1] - s0, 8 * NT), tiles = (cnt + 7) >> 3;
    float sg[RU], su[RU];  // scales of the lane's rows
#pragma unroll
    for (int r = 0; r < RU; ++r) {
      const int i = min(i0 + r * 8 + q4, I - 1);
      const float* sc = p.a.s_gate_up + (size_t)L.expert[a] * 2 * I + i;
      sg[r] = __ldg(sc);
      su[r] = __ldg(sc + I);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) xr[nt] = nt * 8 + q4 < cnt ? p.xf + (size_t)L.token[s0 + nt * 8 + q4] * p.hpad + t4 * 8 : nullptr;
    clear();
#pragma unroll 1
    for (int kb = warp % ks1; kb < nb1; kb += ks1) multiply(kb, tiles, std::false_type());
    if (!gather(ks1)) continue;
    // gate and up of a row lie in one lane
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt >= tiles) break;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int n = nt * 8 + 2 * t4 + c;
        const bool in = n < cnt;
        const int s = in ? L.slot[s0 + n] : 0;
        const float xb = in ? L.xback[L.token[s0 + n]] : 0.0f;
        const int e0 = L.base[s];
        unsigned high = 0, low = 0;
#pragma unroll
        for (int m = 0; m < RU / 2; ++m) {  // 16 columns: two of the lane's rows, those of the eight lanes with this token
          const int i = i0 + m * 16 + q4;   // and i + 8; inter is a multiple of 16
          float hv[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) hv[k] = gate_act(acc[0][2 * m + k][nt][c] * xb * sg[2 * m + k], p.a.act) * (acc[0][2 * m + k][nt][c + 2] * xb * su[2 * m + k]);
          float big = fmaxf(fabsf(hv[0]), fabsf(hv[1]));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 4));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 8));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 16));
          const int e = (int)(__float_as_uint(big) >> 23) - 127, step = (e - e0 + 15) >> 4;  // big * 2^(14 - e0 - 16 step) lies in 2^-1 .. 2^15
          if (in && i < I) {
            const int up = 14 - e0 - 16 * step;
            p.h[(size_t)s * p.ipad + place(i)] = __half_as_ushort(__float2half_rn(times_pow2(hv[0], up)));
            p.h[(size_t)s * p.ipad + place(i + 8)] = __half_as_ushort(__float2half_rn(times_pow2(hv[1], up)));
            if (q4 == 0) p.step[(size_t)s * (p.ipad >> 4) + (i >> 4)] = (signed char)step;
            if (big > 0.0f) {
              high = max(high, (unsigned)(kBias + step));
              low = max(low, (unsigned)(kBias - step));
            }
          }
        }
        if (high && q4 == 0) {
          atomicMax(p.sync + kSteps + 2 * s, high);
          atomicMax(p.sync + kSteps + 2 * s + 1, low);
        }
      }
    }
  }
  // the columns from inter to the padded width are zero
  if (p.ipad > I)
    for (int x = blockIdx.x * kThreads + tid; x < T * K * (p.ipad - I); x += gridDim.x * kThreads) {
      const int s = x / (p.ipad - I), i = I + x % (p.ipad - I);
      p.h[(size_t)s * p.ipad + place(i)] = 0;
      if ((i & 15) == 0) p.step[(size_t)s * (p.ipad >> 4) + (i >> 4)] = -kBias;
    }
  if (!grid_barrier(p.sync + 1)) {
    if (warp == 0) leave(p.sync, E, T * K, lane);
    drain();
    return;
  }

  // the powers of the rows of h, and which have columns of others
  for (int s = tid; s < T * K; s += kThreads) {
    const uint2 m = __ldcg(reinterpret_cast<const uint2*>(p.sync + kSteps) + s);
    L.power[s] = (short)(L.base[s] + (m.x ? 16 * ((int)m.x - kBias) : 0));  // a row of zeros: any
    L.mixed[s] = m.x && m.x + m.y != 2u * kBias;
  }
  __syncthreads();

  // -------------------------------------------------------------- 2: down --
#pragma unroll 1
  for (int u = warp / ks2; u < n2; u += WARPS / ks2) {
    const int a = (u2 + u) / per2, r0 = (u2 + u - a * per2) * (16 * RU);
    const int s0 = L.start[a], cnt = min(L.start[a + 1] - s0, 8 * NT), tiles = (cnt + 7) >> 3;
    float sd[2][RU];
    bool mixed = false;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int r = 0; r < RU; ++r) sd[k][r] = __ldg(p.a.s_down + (size_t)L.expert[a] * H + min(r0 + k * 8 * RU + r * 8 + q4, H - 1));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool in = nt * 8 + q4 < cnt;
      slot_of[nt] = in ? L.slot[s0 + nt * 8 + q4] : 0;
      xr[nt] = in ? p.h + (size_t)slot_of[nt] * p.ipad + t4 * 8 : nullptr;
      mixed |= in && L.mixed[slot_of[nt]];
    }
    clear();
    if (!__any_sync(0xffffffffu, mixed)) {
#pragma unroll 1
      for (int kb = warp % ks2; kb < nb2; kb += ks2) multiply(kb, tiles, std::false_type());
    } else {
#pragma unroll 1
      for (int kb = warp % ks2; kb < nb2; kb += ks2) multiply(kb, tiles, std::true_type());
    }
    if (!gather(ks2)) continue;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt >= tiles) break;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int n = nt * 8 + 2 * t4 + c;
        if (n >= cnt) continue;
        const int s = L.slot[s0 + n];
        const int e = L.power[s] - 14;
        const float wt = L.weight[s] * pow2(e >> 1), back = pow2(e - (e >> 1));
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int r = 0; r < RU; ++r) {
            const int row = r0 + k * 8 * RU + r * 8 + q4;
            if (row < H) p.part[(size_t)s * H + row] = acc[0][r][nt][c + 2 * k] * sd[k][r] * wt * back;
          }
      }
    }
  }
  if (!ok) drain();
  const bool met = grid_barrier(p.sync + 2);
  if (warp == WARPS - 1) leave(p.sync, E, T * K, lane);  // the others' loads of phase 3 are under way meanwhile
  if (!met) return;

  // --------------------------------------------------- 3: a token's slots --
  for (int x = blockIdx.x * kThreads + tid; x < T * (H >> 1); x += gridDim.x * kThreads) {
    const int t = x / (H >> 1), c = x % (H >> 1) * 2;
    const float* src = p.part + (size_t)t * K * H + c;
    float y0 = 0.0f, y1 = 0.0f;
    for (int s = 0; s < K; ++s) {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(src + (size_t)s * H));
      y0 += v.x;
      y1 += v.y;
    }
    uint16_t* out = static_cast<uint16_t*>(p.a.out) + (size_t)t * H + c;
    if (p.a.a_type == FP8IMMA_A_F16) {
      *reinterpret_cast<uint32_t*>(out) = pack_f16(y0, y1);
    } else {
      *reinterpret_cast<uint32_t*>(out) = (uint32_t)f32_to_a16<1>(y0) | ((uint32_t)f32_to_a16<1>(y1) << 16);
    }
  }
}

template <int FMT, int NT, int RU, int WARPS, int DEPTH>
cudaError_t launch(const fp8imma_moe_args& a, cudaStream_t st) {
  using S = Shape<NT, RU, WARPS, DEPTH>;
  const auto kern = moe_kernel<FMT, NT, RU, WARPS, DEPTH>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), S::kSmem);
  if (e != cudaSuccess) return e;
  MoeParams p = {};
  p.a = a;
  CUtensorMap up, down;
  e = make_tmap_3d_u8(&up, a.w_gate_up, a.hidden, a.inter, (uint64_t)a.experts * 2, 128, 8 * RU, 2);
  if (e == cudaSuccess) e = make_tmap_3d_u8(&down, a.w_down, a.inter, a.hidden, a.experts, 128, 16 * RU, 1);
  if (e != cudaSuccess) return e;
  p.hpad = (a.hidden + 127) & ~127;
  p.ipad = (a.inter + 127) & ~127;
  const size_t slots = (size_t)a.tokens * a.top_k;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += (bytes + 255) & ~size_t(255);
    return was;
  };
  const size_t o_logits = take((size_t)a.tokens * a.experts * 4), o_xf = take((size_t)a.tokens * p.hpad * 2), o_back = take((size_t)a.tokens * 8),
               o_ids = take(slots * 4), o_wts = take(slots * 4), o_h = take(slots * p.ipad * 2), o_step = take(slots * (p.ipad >> 4)), o_part = take(slots * a.hidden * 4);
  ScopedScratch sync, work;
  e = sync.get(kSyncWords * 4, st, kScratchMoeSync);
  if (e == cudaSuccess && sync.owned) e = cudaMemsetAsync(sync.ptr, 0, kSyncWords * 4, st);
  if (e == cudaSuccess) e = work.get(at, st, kScratchMoe);
  if (e == cudaSuccess) {
    char* base = static_cast<char*>(work.ptr);
    p.sync = static_cast<unsigned int*>(sync.ptr);
    p.logits = reinterpret_cast<float*>(base + o_logits);
    p.xf = reinterpret_cast<uint16_t*>(base + o_xf);
    p.xback = reinterpret_cast<float*>(base + o_back);
    p.ids = reinterpret_cast<int*>(base + o_ids);
    p.weights = reinterpret_cast<float*>(base + o_wts);
    p.h = reinterpret_cast<uint16_t*>(base + o_h);
    p.step = reinterpret_cast<signed char*>(base + o_step);
    p.part = reinterpret_cast<float*>(base + o_part);
    cudaLaunchConfig_t lc = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;  // the CTAs wait for one another: all of them have to be resident
    attr[0].val.cooperative = 1;
    lc.gridDim = dim3(num_sms_current());
    lc.blockDim = dim3(S::kThreads);
    lc.dynamicSmemBytes = S::kSmem;
    lc.stream = st;
    lc.attrs = attr;
    lc.numAttrs = 1;
    e = cudaLaunchKernelEx(&lc, kern, up, down, p);
  }
  const cudaError_t e1 = sync.release(st), e2 = work.release(st);
  return e != cudaSuccess ? e : e1 != cudaSuccess ? e1 : e2;
}

// Token tiles by the number of tokens, which an expert may all be given; with
// many tokens a unit has more rows, so that the tokens' operands, read again
// for each unit, cost less beside the weights. Measured with 1, 2 and 4 tiles:
// one token, 6 of 64, 2048 x 1408 25 / 27 / 31 us; 8 tokens, 2 of 8, 4096 x 11008
// 197 / 214 / 221; 16 tokens 223 / 245 with 2 and 4; 12 and 16 tokens, 4 of 32,
// 4096 x 2048 141 / 157 and 149 / 162.
template <int FMT>
cudaError_t launch_nt(const fp8imma_moe_args& a, cudaStream_t st) {
  if (a.tokens <= 8) return launch<FMT, 1, 2, 16, 2>(a, st);
  if (a.tokens <= 16) return launch<FMT, 2, 2, 16, 2>(a, st);
  return launch<FMT, 4, 4, 8, 2>(a, st);
}

}  // namespace

unsigned int moe_device_error(bool clear) { return fp8imma_dev::tu_device_error(clear); }
cudaError_t moe_set_wait_limit(unsigned long long ns) { return fp8imma_dev::tu_set_wait_limit(ns); }

}  // namespace fp8imma_b200

using namespace fp8imma_b200;

extern "C" int fp8imma_moe_forward(const fp8imma_moe_args* a, void* stream) {
  FP8IMMA_RANGE("fp8imma_moe_forward");
  if (!a) return (int)cudaErrorInvalidValue;
  if (a->tokens <= 0 || a->experts <= 0 || a->hidden <= 0 || a->inter <= 0) return (int)cudaErrorInvalidConfiguration;
  if (!a->x || !a->router || !a->w_gate_up || !a->s_gate_up || !a->w_down || !a->s_down || !a->out)
    return (int)cudaErrorInvalidValue;
  if (a->a_type < 0 || a->a_type > 1 || a->format < 0 || a->format > 1 || a->act < 2 || a->act > 3)
    return (int)cudaErrorInvalidValue;
  if (a->tokens > FP8IMMA_MOE_MAX_TOKENS || a->experts > FP8IMMA_MOE_MAX_EXPERTS || a->top_k < 1 ||
      a->top_k > FP8IMMA_MOE_MAX_TOP_K || a->top_k > a->experts)
    return (int)cudaErrorInvalidValue;
  if (a->hidden % 16 || a->inter % 16) return (int)cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a->w_gate_up) | reinterpret_cast<uintptr_t>(a->w_down)) & 15u)
    return (int)cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->router)) & 1u) return (int)cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(a->out) & 3u) return (int)cudaErrorInvalidValue;
  // weight rows are indexed with 31 bits
  if ((int64_t)a->experts * 2 * a->inter > 0x7fffffffll || (int64_t)a->experts * a->hidden > 0x7fffffffll)
    return (int)cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return (int)(a->format == FP8IMMA_B_E4M3 ? launch_nt<F8_E4M3>(*a, st) : launch_nt<F8_E5M2>(*a, st));
}
