// Mixture-of-experts layer with FP8 weights for 1 .. 64 tokens
// (fp8imma_moe_forward), in one launch.
//
// Mathematics: r = x Wr^T (fp32), S_t the top_k experts of token t, p the
// softmax; per chosen (token, expert) slot
//   h = act(sg (x Wg^T)) * (su (x Wu^T)),  out_t = sum_S p sd (h Wd^T).
// FP8 codes are multiplied as fp16 (exact); x and h enter as fp16 rows that a
// power of two has brought into fp16's range (exact for fp16 x and for bf16
// values within 2^22 of the row's largest; h is rounded to 2^-11), sums are
// fp32, scales and the powers of two are applied to the sums.
//
// Bound: a few tokens use each weight byte a few times, so the layer costs the
// bytes of the chosen experts. One cooperative grid, one CTA per SM, keeps
// their stream running through the whole layer:
//  0. router logits (warps over experts x tokens), x to fp16 in operand order;
//     grid barrier; every CTA picks the top_k of all tokens for itself
//  1. gate / up: the chosen experts' row groups are laid end to end and cut
//     into equal runs; a unit is 8 RU gate rows and the same 8 RU up rows, so
//     that both factors of h meet in one fragment; grid barrier
//  2. down: the same over units of 16 RU rows; slot results to scratch; barrier
//  3. out = sum over a token's slots, in their order
// A warp takes every eighth 128-byte column block of the flattened (unit,
// block) sequence and streams its blocks by TMA into a ring of its own, across
// unit and phase boundaries: the down weights are under way while the grid
// meets at the barrier before them. The eight warps' partial sums of a unit
// meet in shared memory in a fixed order; nothing depends on timing.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxSlots = FP8IMMA_MOE_MAX_TOKENS * FP8IMMA_MOE_MAX_TOP_K;

struct MoeParams {
  fp8imma_moe_args a;
  unsigned int* sync;  // three barrier counters, zero between calls
  float* logits;       // [tokens, experts]
  uint16_t* xf;        // [tokens, hidden padded to 128] fp16, operand order
  float* xback;        // [tokens] what a row of xf is to be multiplied by
  unsigned int* hmax;  // [slots] bits of the largest |h|
  float* h;            // [slots, inter padded to 128] operand order
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
    __threadfence();
    unsigned int v;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(v) : "l"(ctr) : "memory");
    ++v;
    bool ok = true;
    const unsigned long long t0 = globaltimer_ns();
    while (v < gridDim.x) {
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(ctr) : "memory");
      const unsigned long long dt = globaltimer_ns() - t0;
      if (dt > kWaitCheckNs && dt > *(volatile unsigned long long*)&g_fp8imma_wait_limit_ns) {
        atomicCAS(&g_fp8imma_device_error, 0u, (unsigned int)ERR_WAIT_PEER);
        ok = false;
        break;
      }
    }
    __threadfence();
    s_ok = ok;
  }
  __syncthreads();
  return s_ok != 0;
}

struct Runs {  // CTA c's run of the units: they differ by one in length at most
  int per, rem;
  __device__ __forceinline__ Runs(int units, int ctas) : per(units / ctas), rem(units % ctas) {}
  __device__ __forceinline__ int begin(int c) const { return c * per + min(c, rem); }
};

// NT: 8-token tiles at most; RU: 16-row tiles of a unit.
template <int NT, int RU>
struct Shape {
  static constexpr int kStageBytes = 2048 * RU;
  static constexpr int kStages = RU == 1 ? 8 : NT == 8 ? 4 : 5;
  static constexpr int kRing = kStages * kStageBytes;  // of a warp
  static constexpr int kRedFloats = 16 * RU * 8 * NT;  // of a warp
  static constexpr int kRedBufs = NT <= 2 ? 2 : 1;
  static constexpr int kSmem = 1024 + kWarps * (kRing + kRedBufs * kRedFloats * 4);
};

// Router logits of EX experts x TX tokens a warp, and nothing else.
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
  }
}

// Place of element k of a row in operand order: lane t4 of a fragment reads
// bytes 32 t4 .. 32 t4 + 31 of a 128-byte weight block, four a product step s.
// x keeps eight fp16 (two steps) together, h four fp32 (one step).
__device__ __forceinline__ int x_place(int k) { return (k & ~127) + (((k & 31) >> 3) << 5) + (((k >> 5) & 3) << 3) + (k & 7); }
__device__ __forceinline__ int h_place(int k) { return (k & ~127) + (((k & 31) >> 2) << 4) + (((k >> 5) & 3) << 2) + (k & 3); }

// A token's row as fp16 in operand order; one warp.
template <int AT>
__device__ __forceinline__ void convert_row(const MoeParams& p, int t, int lane, bool vec) {
  const uint16_t* x = static_cast<const uint16_t*>(p.a.x) + t * p.a.x_token_stride;
  float f = 1.0f, back = 1.0f;
  auto load8 = [&](int k) {
    if (vec) return __ldg(reinterpret_cast<const uint4*>(x + k));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldg(x + k + 2 * i) | ((uint32_t)__ldg(x + k + 2 * i + 1) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  if (AT == 1) {
    float big = 0.0f;
#pragma unroll 4
    for (int k = lane * 8; k < p.a.hidden; k += 256) {
      const uint4 v = load8(k);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) big = fmaxf(big, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xFFFF0000u))));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
    row_factor(big, f, back);
  }
#pragma unroll 4
  for (int k = lane * 8; k < p.hpad; k += 256) {
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
    *reinterpret_cast<uint4*>(p.xf + (size_t)t * p.hpad + x_place(k)) = v;
  }
  if (lane == 0) p.xback[t] = back;
}

struct Lists {
  unsigned long long tokens[FP8IMMA_MOE_MAX_EXPERTS];  // tokens that chose the expert
  short expert[FP8IMMA_MOE_MAX_EXPERTS];               // chosen experts, ascending
  short start[FP8IMMA_MOE_MAX_EXPERTS + 1];            // their first entry in `slot`
  short slot[kMaxSlots];                               // slots by expert, tokens ascending
  short id[kMaxSlots];                                 // expert of a slot
  float weight[kMaxSlots];                             // p of a slot
  float scale[kMaxSlots];                              // phase 1: largest |h| bits; phase 2: factor that brings h into fp16's range
  int active;
  int scan[kWarps];
};

// Two tokens' top_k at once by one warp (their chains of reductions overlap).
__device__ __forceinline__ void pick(const MoeParams& p, Lists& L, int t0, int lane) {
  const int E = p.a.experts, K = p.a.top_k;
  unsigned taken[2] = {0u, 0u};
  float first[2] = {0.0f, 0.0f}, sum[2] = {0.0f, 0.0f};
  const float* r[2] = {p.logits + (size_t)t0 * E, p.logits + (size_t)min(t0 + 1, p.a.tokens - 1) * E};
  float keep[2][4];  // the first 128 experts stay in registers
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int i = 0; i < 4; ++i) keep[q][i] = lane + 32 * i < E ? __ldcg(r[q] + lane + 32 * i) : 0.0f;
  for (int s = 0; s < K; ++s) {
    int best[2], at[2];
    float val[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      best[q] = (int)0x80000000;
      at[q] = 0x7fffffff;
      val[q] = 0.0f;
      bool any = false;
      auto look = [&](int i, float v) {
        const int key = order_key(v);
        if (!((taken[q] >> i) & 1u) && (!any || key > best[q])) {
          best[q] = key;
          at[q] = lane + 32 * i;
          val[q] = v;
          any = true;
        }
      };
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < E) look(i, keep[q][i]);
      for (int i = 4; lane + 32 * i < E; ++i) look(i, __ldcg(r[q] + lane + 32 * i));
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int top = __reduce_max_sync(0xffffffffu, best[q]);
      const int e = __reduce_min_sync(0xffffffffu, best[q] == top ? at[q] : 0x7fffffff);
      val[q] = __shfl_sync(0xffffffffu, val[q], e & 31);
      if ((e & 31) == lane) taken[q] |= 1u << (e >> 5);
      if (s == 0) first[q] = val[q];
      const float w = __expf(val[q] - first[q]);
      sum[q] += w;
      if (lane == 0 && t0 + q < p.a.tokens) {
        L.id[(t0 + q) * K + s] = (short)e;
        L.weight[(t0 + q) * K + s] = w;
      }
    }
  }
  if (!p.a.renormalize) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float z = 0.0f;
      for (int i = lane; i < E; i += 32) z += __expf(__ldcg(r[q] + i) - first[q]);
      sum[q] = warp_sum(z);
    }
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 2; ++q)
    if (t0 + q < p.a.tokens && lane < K) L.weight[(t0 + q) * K + lane] = __fdiv_rn(L.weight[(t0 + q) * K + lane], sum[q]);
}

template <int FMT, int NT, int RU>
__global__ void __launch_bounds__(kThreads, 1)
    moe_kernel(const __grid_constant__ CUtensorMap map_up, const __grid_constant__ CUtensorMap map_down, const __grid_constant__ MoeParams p) {
  using S = Shape<NT, RU>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Lists L;
  __shared__ uint64_t s_full[kWarps][S::kStages];
  const uint32_t off = ((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q4 = lane >> 2, t4 = lane & 3;
  uint8_t* const ring = smem_raw + off + warp * S::kRing;
  float* const red = reinterpret_cast<float*>(smem_raw + off + kWarps * S::kRing);
  const int T = p.a.tokens, E = p.a.experts, K = p.a.top_k, H = p.a.hidden, I = p.a.inter;

  if (lane == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&s_full[warp][i], 1);
    fence_barrier_init();
    prefetch_tensormap(warp & 1 ? &map_down : &map_up);
  }

  // ------------------------------------------------- 0: router, x to fp16 --
  {
    // warps of the grid, CTA by CTA, so that few units spread over many SMs
    const int wid = warp * gridDim.x + blockIdx.x, nw = kWarps * gridDim.x;
    const bool vec = ((reinterpret_cast<uintptr_t>(p.a.x) | reinterpret_cast<uintptr_t>(p.a.router) | (uintptr_t)(p.a.x_token_stride * 2)) & 15u) == 0;
    const bool bf = p.a.a_type == FP8IMMA_A_BF16;
    for (int t = nw - 1 - wid; t < T; t += nw) {  // from the last warp on: the first have router units
      if (bf) convert_row<1>(p, t, lane, vec);
      else convert_row<0>(p, t, lane, vec);
    }
    if (NT == 1) {  // 8 tokens at most
      if (T == 1) {
        if (bf) router<1, 1, 1>(p, wid, nw, lane, vec);
        else router<0, 1, 1>(p, wid, nw, lane, vec);
      } else {
        if (bf) router<1, 1, 4>(p, wid, nw, lane, vec);
        else router<0, 1, 4>(p, wid, nw, lane, vec);
      }
    } else {
      if (bf) router<1, 4, 4>(p, wid, nw, lane, vec);
      else router<0, 4, 4>(p, wid, nw, lane, vec);
    }
    if (blockIdx.x == 0)
      for (int s = tid; s < T * K; s += kThreads) p.hmax[s] = 0u;
  }
  if (!grid_barrier(p.sync)) return;  // no copies are under way yet
  if (blockIdx.x == 0 && tid == 0) p.sync[2] = 0u;  // all CTAs of the call before have left its last barrier

  // -------------------------------------------------------- choice, lists --
  for (int e = tid; e < E; e += kThreads) L.tokens[e] = 0ull;
  for (int s = tid; s < T * K; s += kThreads) L.scale[s] = 0.0f;
  for (int t = warp * 2; t < T; t += kWarps * 2) pick(p, L, t, lane);
  __syncthreads();
  for (int s = tid; s < T * K; s += kThreads) {
    atomicOr(&L.tokens[L.id[s]], 1ull << (s / K));
    if (blockIdx.x == 0) {
      if (p.a.ids) p.a.ids[s] = L.id[s];
      if (p.a.weights) p.a.weights[s] = L.weight[s];
    }
  }
  __syncthreads();
  {
    int active = 0, slots = 0;
    for (int e0 = 0; e0 < E; e0 += kThreads) {
      const int e = e0 + tid;
      const int n = e < E ? __popcll(L.tokens[e]) : 0;
      int x = n | ((n > 0) << 16);  // slots and experts so far
      const int own = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      __syncthreads();
      if (lane == 31) L.scan[warp] = x;
      __syncthreads();
      int before = slots | (active << 16), total = 0;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += L.scan[w];
        total += L.scan[w];
      }
      before += x - own;
      if (n > 0) {
        L.expert[before >> 16] = (short)e;
        L.start[before >> 16] = (short)(before & 0xFFFF);
      }
      slots += total & 0xFFFF;
      active += total >> 16;
    }
    if (tid == 0) {
      L.active = active;
      L.start[active] = (short)slots;
    }
  }
  __syncthreads();
  const int active = L.active;
  for (int a = warp; a < active; a += kWarps) {  // slots of each chosen expert, tokens ascending
    const unsigned long long m = L.tokens[L.expert[a]];
    for (int t = lane; t < T; t += 32)
      if ((m >> t) & 1ull) {
        int s = t * K;
        while (L.id[s] != L.expert[a]) ++s;
        L.slot[L.start[a] + __popcll(m & ((1ull << t) - 1ull))] = (short)s;
      }
  }
  __syncthreads();

  // --------------------------------------------------- the weights' stream --
  // Units per expert, column blocks per unit of the two phases; this CTA's runs.
  const int per1 = (I + 8 * RU - 1) / (8 * RU), per2 = (H + 16 * RU - 1) / (16 * RU);
  const int nb1 = p.hpad >> 7, nb2 = p.ipad >> 7;
  const Runs runs1(active * per1, gridDim.x), runs2(active * per2, gridDim.x);
  const int u1 = runs1.begin(blockIdx.x), n1 = runs1.begin(blockIdx.x + 1) - u1;
  const int u2 = runs2.begin(blockIdx.x), n2 = runs2.begin(blockIdx.x + 1) - u2;

  // loading side of this warp: next block to ask for
  int lp = 1, lu = 0, lb = warp, issued = 0, used = 0, lost = 0;
  bool ok = true;
  auto issue = [&]() {
    if (!ok) return;
    // one block further down the flattened sequence, over the phases' ends
    if (lp == 1) {
      while (lb >= nb1) lb -= nb1, ++lu;
      if (lu >= n1) lp = 2, lu = 0, lb = warp;
    }
    if (lp == 2) {
      while (lb >= nb2) lb -= nb2, ++lu;
      if (lu >= n2) lp = 3;
    }
    if (lp == 3) return;
    const int st = issued % S::kStages;
    if (lane == 0) {
      mbar_arrive_expect_tx(&s_full[warp][st], S::kStageBytes);
      uint8_t* dst = ring + st * S::kStageBytes;
      if (lp == 1) {
        const int u = u1 + lu, e = L.expert[u / per1], row = e * 2 * I + u % per1 * (8 * RU);
        tma_load_2d(dst, &map_up, &s_full[warp][st], lb * 128, row);
        tma_load_2d(dst + 1024 * RU, &map_up, &s_full[warp][st], lb * 128, row + I);
      } else {
        const int u = u2 + lu, e = L.expert[u / per2], row = e * H + u % per2 * (16 * RU);
        tma_load_2d(dst, &map_down, &s_full[warp][st], lb * 128, row);
        tma_load_2d(dst + 1024 * RU, &map_down, &s_full[warp][st], lb * 128, row + 8 * RU);
      }
    }
    lb += kWarps;
    ++issued;
  };
  auto wait = [&]() {  // for the next block; after a wait that ran out the rest is passed over
    const int st = used % S::kStages;
    if (ok) {
      ok = mbar_wait(&s_full[warp][st], (uint32_t)((used / S::kStages) & 1), ERR_WAIT_FULL);
      if (!ok) lost = used;
    }
    return ring + st * S::kStageBytes;
  };
  auto drain = [&]() {  // before an early end: the copies under way land first
    for (int k = ok ? used : lost; k < issued; ++k) mbar_wait(&s_full[warp][k % S::kStages], (uint32_t)((k / S::kStages) & 1), ERR_WAIT_FULL);
  };
  for (int i = 0; i < S::kStages; ++i) issue();

  // ------------------------------------------------ 1: gate, up, activation --
  int flip = 0, cb = warp;  // reduction buffer; this warp's next block of the unit
  for (int u = 0; u < n1; ++u) {
    const int a = (u1 + u) / per1, i0 = (u1 + u) % per1 * (8 * RU), e = L.expert[a];
    const int s0 = L.start[a], cnt = L.start[a + 1] - s0;
    const int tiles = (cnt + 7) >> 3;
    const uint16_t* xr[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) xr[nt] = nt * 8 + q4 < cnt ? p.xf + (size_t)(L.slot[s0 + nt * 8 + q4] / K) * p.hpad + t4 * 8 : nullptr;
    float acc[RU][NT][4];
#pragma unroll
    for (int r = 0; r < RU; ++r)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][nt][c] = 0.0f;
    for (; cb < nb1; cb += kWarps) {
      uint4 x0[4];  // the first tile's operands are asked for before the wait
#pragma unroll
      for (int i = 0; i < 4; ++i) x0[i] = xr[0] ? *reinterpret_cast<const uint4*>(xr[0] + cb * 128 + i * 32) : make_uint4(0, 0, 0, 0);
      const uint8_t* w = wait();
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // halves of the lane's 32 bytes a row
        uint32_t g[RU][4], b[RU][4];
#pragma unroll
        for (int r = 0; r < RU; ++r) {
          const int at = (r * 8 + q4) * 128 + (((2 * t4 + j) ^ q4) << 4);
          const uint4 v = *reinterpret_cast<const uint4*>(w + at), z = *reinterpret_cast<const uint4*>(w + 1024 * RU + at);
          g[r][0] = v.x, g[r][1] = v.y, g[r][2] = v.z, g[r][3] = v.w;
          b[r][0] = z.x, b[r][1] = z.y, b[r][2] = z.z, b[r][3] = z.w;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t A[RU][2][4];
#pragma unroll
          for (int r = 0; r < RU; ++r)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              f8x4_to_f16x4<FMT>(g[r][2 * i + s], A[r][s][0], A[r][s][2]);
              f8x4_to_f16x4<FMT>(b[r][2 * i + s], A[r][s][1], A[r][s][3]);
            }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (nt > 0 && nt >= tiles) break;
            const uint4 x = nt == 0 ? x0[2 * j + i] : xr[nt] ? *reinterpret_cast<const uint4*>(xr[nt] + cb * 128 + (2 * j + i) * 32) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < RU; ++r) {
              mma_f16(acc[r][nt], A[r][0][0], A[r][0][1], A[r][0][2], A[r][0][3], x.x, x.y);
              mma_f16(acc[r][nt], A[r][1][0], A[r][1][1], A[r][1][2], A[r][1][3], x.z, x.w);
            }
          }
        }
      }
      ++used;
      __syncwarp();
      issue();
    }
    cb -= nb1;
    // the warps' sums meet: rows 16 r + 0..7 gate, + 8..15 up
    float* mine = red + flip * (kWarps * S::kRedFloats) + warp * S::kRedFloats;
#pragma unroll
    for (int r = 0; r < RU; ++r)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (nt >= tiles) break;
        *reinterpret_cast<float2*>(mine + (r * 16 + q4) * (8 * NT) + nt * 8 + 2 * t4) = make_float2(acc[r][nt][0], acc[r][nt][1]);
        *reinterpret_cast<float2*>(mine + (r * 16 + 8 + q4) * (8 * NT) + nt * 8 + 2 * t4) = make_float2(acc[r][nt][2], acc[r][nt][3]);
      }
    __syncthreads();
    for (int x = tid; x < ((cnt * 8 * RU + 31) & ~31); x += kThreads) {
      const int n = x / (8 * RU), i = x % (8 * RU);
      float hv = 0.0f;
      if (n < cnt && i0 + i < I) {
        const float* src = red + flip * (kWarps * S::kRedFloats) + ((i >> 3) * 16 + (i & 7)) * (8 * NT) + n;
        float gs = 0.0f, us = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          gs += src[w * S::kRedFloats];
          us += src[w * S::kRedFloats + 8 * (8 * NT)];
        }
        const int s = L.slot[s0 + n];
        const float xb = __ldcg(p.xback + s / K);
        const float* sc = p.a.s_gate_up + (size_t)e * 2 * I + i0 + i;
        hv = gate_act(gs * xb * __ldg(sc), p.a.act) * (us * xb * __ldg(sc + I));
        p.h[(size_t)s * p.ipad + h_place(i0 + i)] = hv;
      }
      // largest |h| of the slot so far (as bits, NaN above all)
      unsigned m = __float_as_uint(hv) & 0x7FFFFFFFu;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if ((lane & 7) == 0 && n < cnt) atomicMax(reinterpret_cast<unsigned int*>(&L.scale[L.slot[s0 + n]]), m);
    }
    if (S::kRedBufs == 2) flip ^= 1;
    else __syncthreads();
  }
  __syncthreads();
  for (int s = tid; s < T * K; s += kThreads) {
    const unsigned m = __float_as_uint(L.scale[s]);
    if (m) atomicMax(p.hmax + s, m);
  }
  if (!grid_barrier(p.sync + 1)) {
    drain();
    return;
  }
  if (blockIdx.x == 0 && tid == 0) p.sync[0] = 0u;
  for (int s = tid; s < T * K; s += kThreads) {
    float f, back;
    row_factor(__uint_as_float(__ldcg(p.hmax + s)), f, back);
    L.scale[s] = f;
    // a slot's result is multiplied by its weight and by what undoes the factor
    L.weight[s] = L.weight[s] * back;
  }
  __syncthreads();

  // -------------------------------------------------------------- 2: down --
  cb = warp;
  for (int u = 0; u < n2; ++u) {
    const int a = (u2 + u) / per2, r0 = (u2 + u) % per2 * (16 * RU), e = L.expert[a];
    const int s0 = L.start[a], cnt = L.start[a + 1] - s0;
    const int tiles = (cnt + 7) >> 3;
    const float* hr[NT];
    float hf[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool in = nt * 8 + q4 < cnt;
      const int s = in ? L.slot[s0 + nt * 8 + q4] : 0;
      hr[nt] = in ? p.h + (size_t)s * p.ipad + t4 * 4 : nullptr;
      hf[nt] = in ? L.scale[s] : 0.0f;
    }
    float acc[RU][NT][4];
#pragma unroll
    for (int r = 0; r < RU; ++r)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][nt][c] = 0.0f;
    for (; cb < nb2; cb += kWarps) {
      float4 x0[8];
      const int left = I - cb * 128 - t4 * 32;  // the lane's valid channels of the block
#pragma unroll
      for (int i = 0; i < 8; ++i) x0[i] = hr[0] && 4 * i < left ? *reinterpret_cast<const float4*>(hr[0] + cb * 128 + i * 16) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const uint8_t* w = wait();
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t g[RU][4], b[RU][4];
#pragma unroll
        for (int r = 0; r < RU; ++r) {
          const int at = (r * 8 + q4) * 128 + (((2 * t4 + j) ^ q4) << 4);
          const uint4 v = *reinterpret_cast<const uint4*>(w + at), z = *reinterpret_cast<const uint4*>(w + 1024 * RU + at);
          g[r][0] = v.x, g[r][1] = v.y, g[r][2] = v.z, g[r][3] = v.w;
          b[r][0] = z.x, b[r][1] = z.y, b[r][2] = z.z, b[r][3] = z.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t A[RU][4];
#pragma unroll
          for (int r = 0; r < RU; ++r) {
            f8x4_to_f16x4<FMT>(g[r][i], A[r][0], A[r][2]);
            f8x4_to_f16x4<FMT>(b[r][i], A[r][1], A[r][3]);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (nt > 0 && nt >= tiles) break;
            const float4 x = nt == 0 ? x0[4 * j + i]
                             : hr[nt] && 4 * (4 * j + i) < left ? *reinterpret_cast<const float4*>(hr[nt] + cb * 128 + (4 * j + i) * 16)
                                                                : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const uint32_t b0 = pack_f16(x.x * hf[nt], x.y * hf[nt]), b1 = pack_f16(x.z * hf[nt], x.w * hf[nt]);
#pragma unroll
            for (int r = 0; r < RU; ++r) mma_f16(acc[r][nt], A[r][0], A[r][1], A[r][2], A[r][3], b0, b1);
          }
        }
      }
      ++used;
      __syncwarp();
      issue();
    }
    cb -= nb2;
    // rows 16 r + 0..7: first box, + 8..15: second box (8 RU rows further on)
    float* mine = red + flip * (kWarps * S::kRedFloats) + warp * S::kRedFloats;
#pragma unroll
    for (int r = 0; r < RU; ++r)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (nt >= tiles) break;
        *reinterpret_cast<float2*>(mine + (r * 16 + q4) * (8 * NT) + nt * 8 + 2 * t4) = make_float2(acc[r][nt][0], acc[r][nt][1]);
        *reinterpret_cast<float2*>(mine + (r * 16 + 8 + q4) * (8 * NT) + nt * 8 + 2 * t4) = make_float2(acc[r][nt][2], acc[r][nt][3]);
      }
    __syncthreads();
    for (int x = tid; x < cnt * 16 * RU; x += kThreads) {
      const int n = x / (16 * RU), i = x % (16 * RU);  // i: row of the unit
      if (r0 + i >= H) continue;
      const int box = i / (8 * RU), ri = i % (8 * RU);
      const float* src = red + flip * (kWarps * S::kRedFloats) + ((ri >> 3) * 16 + box * 8 + (ri & 7)) * (8 * NT) + n;
      float y = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) y += src[w * S::kRedFloats];
      const int s = L.slot[s0 + n];
      p.part[(size_t)s * H + r0 + i] = y * __ldg(p.a.s_down + (size_t)e * H + r0 + i) * L.weight[s];
    }
    if (S::kRedBufs == 2) flip ^= 1;
    else __syncthreads();
  }
  if (!ok) drain();
  if (!grid_barrier(p.sync + 2)) return;  // every copy has been waited for
  if (blockIdx.x == 0 && tid == 0) p.sync[1] = 0u;

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

template <int FMT, int NT, int RU>
cudaError_t launch(const fp8imma_moe_args& a, cudaStream_t st) {
  using S = Shape<NT, RU>;
  const auto kern = moe_kernel<FMT, NT, RU>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), S::kSmem);
  if (e != cudaSuccess) return e;
  MoeParams p = {};
  p.a = a;
  p.hpad = (a.hidden + 127) & ~127;
  p.ipad = (a.inter + 127) & ~127;
  CUtensorMap up, down;
  e = make_tmap_2d_u8(&up, a.w_gate_up, (uint64_t)a.hidden, (uint64_t)a.experts * 2 * a.inter, (uint64_t)a.hidden, 128, 8 * RU, true);
  if (e == cudaSuccess) e = make_tmap_2d_u8(&down, a.w_down, (uint64_t)a.inter, (uint64_t)a.experts * a.hidden, (uint64_t)a.inter, 128, 8 * RU, true);
  if (e != cudaSuccess) return e;
  const size_t slots = (size_t)a.tokens * a.top_k;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += (bytes + 255) & ~size_t(255);
    return was;
  };
  const size_t o_logits = take((size_t)a.tokens * a.experts * 4), o_xf = take((size_t)a.tokens * p.hpad * 2), o_back = take((size_t)a.tokens * 4),
               o_max = take(slots * 4), o_h = take(slots * p.ipad * 4), o_part = take(slots * a.hidden * 4);
  ScopedScratch sync, work;
  e = sync.get(256, st, kScratchMoeSync);
  if (e == cudaSuccess && sync.owned) e = cudaMemsetAsync(sync.ptr, 0, 256, st);
  if (e == cudaSuccess) e = work.get(at, st, kScratchMoe);
  if (e == cudaSuccess) {
    char* base = static_cast<char*>(work.ptr);
    p.sync = static_cast<unsigned int*>(sync.ptr);
    p.logits = reinterpret_cast<float*>(base + o_logits);
    p.xf = reinterpret_cast<uint16_t*>(base + o_xf);
    p.xback = reinterpret_cast<float*>(base + o_back);
    p.hmax = reinterpret_cast<unsigned int*>(base + o_max);
    p.h = reinterpret_cast<float*>(base + o_h);
    p.part = reinterpret_cast<float*>(base + o_part);
    cudaLaunchConfig_t lc = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;  // the CTAs wait for one another: all of them have to be resident
    attr[0].val.cooperative = 1;
    lc.gridDim = dim3(num_sms_current());
    lc.blockDim = dim3(kThreads);
    lc.dynamicSmemBytes = S::kSmem;
    lc.stream = st;
    lc.attrs = attr;
    lc.numAttrs = 1;
    e = cudaLaunchKernelEx(&lc, kern, up, down, p);
  }
  const cudaError_t e1 = sync.release(st), e2 = work.release(st);
  return e != cudaSuccess ? e : e1 != cudaSuccess ? e1 : e2;
}

// Token tiles by the number of tokens (an expert can be chosen by all of
// them); with more tokens a unit gets more rows, so that a token's operands,
// read again for each unit, cost less than the weights.
template <int FMT>
cudaError_t launch_nt(const fp8imma_moe_args& a, cudaStream_t st) {
  if (a.tokens <= 8) return launch<FMT, 1, 1>(a, st);
  if (a.tokens <= 16) return launch<FMT, 2, 2>(a, st);
  if (a.tokens <= 32) return launch<FMT, 4, 2>(a, st);
  return launch<FMT, 8, 2>(a, st);
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
