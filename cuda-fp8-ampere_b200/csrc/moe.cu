// Mixture-of-experts layer with FP8 weights for 1 .. 64 tokens
// (fp8imma_moe_forward), in one launch.
//
// Mathematics: r = x Wr^T (fp32), S_t the top_k experts of token t, p the
// softmax; per chosen (token, expert) slot
//   h = act(sg (x Wg^T)) * (su (x Wu^T)),  out_t = sum_S p sd (h Wd^T).
// FP8 codes are multiplied as fp16 (exact); sums are fp32, scales are applied
// to the sums. x enters as it is when it is fp16; a bf16 row is brought into
// fp16's range by a power of two (exact within 2^22 of the row's largest). h
// is rounded to fp16, 2^-11, after a power of two of its slot that keeps it
// below 2^15: |act(g) u| <= |g| |u|, and a gate or up sum is at most
// max_i s_i * fmax * sum |x|. Typical h lie some 2^16 below that bound, well
// inside fp16's normal range, and no largest value has to be agreed on first.
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
// A warp works on units of its own (few units: a team of 2, 4 or 8 warps shares
// one along the columns). Each lane copies the 16-byte pieces of its own
// operand rows asynchronously into a queue of its own in shared memory, some
// 128-byte column blocks ahead, across unit and phase boundaries: no barrier
// between lanes or warps, and the down weights are under way while the grid
// meets at the barrier before them. A team's sums meet in shared memory in a
// fixed order; nothing depends on timing.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

constexpr int kMaxSlots = FP8IMMA_MOE_MAX_TOKENS * FP8IMMA_MOE_MAX_TOP_K;

struct MoeParams {
  fp8imma_moe_args a;
  unsigned int* sync;  // three barrier counters, zero between calls
  float* logits;       // [tokens, experts]
  uint16_t* xf;        // [tokens, hidden padded to 128] fp16, operand order
  float* xback;        // [tokens, 2] what a row of xf is to be multiplied by, sum |x|
  float* smax;         // [experts, 2, chunks] largest gate / up scale of 1024 rows
  uint16_t* h;         // [slots, inter padded to 128] fp16, operand order
  float* part;         // [slots, hidden]
  int hpad, ipad, chunks;
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
        atomicCAS(&g_fp8imma_device_error, 0u, (unsigned int)ERR_WAIT_PEER);
        ok = false;
        break;
      }
    }
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

// 16 bytes global -> shared, asynchronously; zeros when not `in`
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

// NT: 8-token tiles of a unit at most; RU: 16-row tiles of a unit; WARPS a CTA;
// DEPTH: blocks of a lane's queue.
template <int NT, int RU, int WARPS, int DEPTH>
struct Shape {
  static constexpr int kThreads = WARPS * 32;
  static constexpr int kPieces = 4 * RU;               // 16-byte pieces of a block a lane
  static constexpr int kQueue = DEPTH * kPieces * 512; // of a warp
  static constexpr int kFragFloats = RU * NT * 4 * 32; // a unit's sums of a warp
  static constexpr int kSmem = WARPS * (kQueue + kFragFloats * 4);
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

// Place of element k of a row in operand order: lane t4 of a fragment holds
// bytes 16 t4 .. 16 t4 + 15 of both halves of a 128-byte weight block, four
// bytes a product step; eight fp16, two steps, lie together.
__device__ __forceinline__ int place(int k) { return (k & ~127) + (((k >> 5) & 2) + ((k >> 3) & 1)) * 32 + (((k >> 4) & 3) << 3) + (k & 7); }

// Largest gate / up scales by chunks of 1024 rows.
__device__ __forceinline__ void scale_maxima(const MoeParams& p, int wid, int nw, int lane) {
#pragma unroll 1
  for (int u = wid; u < p.a.experts * 2 * p.chunks; u += nw) {
    const int c = u % p.chunks, row = u / p.chunks;  // row: expert * 2 + (gate, up)
    const float* s = p.a.s_gate_up + (size_t)row * p.a.inter;
    const int hi = min(p.a.inter, c * 1024 + 1024);
    float m = 0.0f;
#pragma unroll 8
    for (int i = c * 1024 + lane; i < hi; i += 32) m = fmaxf(m, fabsf(__ldg(s + i)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) p.smax[u] = m;
  }
}

// A token's row as fp16 in operand order; one warp.
template <int AT>
__device__ __forceinline__ void convert_row(const MoeParams& p, int t, int lane, bool vec) {
  const uint16_t* x = static_cast<const uint16_t*>(p.a.x) + t * p.a.x_token_stride;
  float f = 1.0f, back = 1.0f, sum = 0.0f;
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
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += fabsf(a16_to_f32<AT>((uint16_t)(w[i] & 0xFFFFu))) + fabsf(a16_to_f32<AT>((uint16_t)(w[i] >> 16)));
      if (AT == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_f16(__uint_as_float(w[i] << 16) * f, __uint_as_float(w[i] & 0xFFFF0000u) * f);
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    *reinterpret_cast<uint4*>(p.xf + (size_t)t * p.hpad + place(k)) = v;
  }
  sum = warp_sum(sum);
  if (lane == 0) {
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
  float scale[kMaxSlots];                              // factor that brings a slot's h into fp16's range
  float xback[FP8IMMA_MOE_MAX_TOKENS];
  int entries;
  int scan[16];
};

// A token's top_k by one warp: rounds of the largest logit not yet taken.
__device__ __forceinline__ void pick(const MoeParams& p, Lists& L, int t, int lane) {
  const int E = p.a.experts, K = p.a.top_k;
  const float* r = p.logits + (size_t)t * E;
  unsigned taken = 0u;  // expert lane + 32 * bit
  float keep[4], first = 0.0f, sum = 0.0f;  // the first 128 experts stay in registers
#pragma unroll
  for (int i = 0; i < 4; ++i) keep[i] = lane + 32 * i < E ? __ldcg(r + lane + 32 * i) : 0.0f;
#pragma unroll 1
  for (int s = 0; s < K; ++s) {
    int best = (int)0x80000000, at = 0x7fffffff;
    float val = 0.0f;
    auto look = [&](int i, float v) {
      const int key = order_key(v);
      if (!((taken >> i) & 1u) && (at == 0x7fffffff || key > best)) {
        best = key;
        at = lane + 32 * i;
        val = v;
      }
    };
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < E) look(i, keep[i]);
#pragma unroll 1
    for (int i = 4; lane + 32 * i < E; ++i) look(i, __ldcg(r + lane + 32 * i));
    const int top = __reduce_max_sync(0xffffffffu, best);
    const int e = __reduce_min_sync(0xffffffffu, best == top ? at : 0x7fffffff);
    val = __shfl_sync(0xffffffffu, val, e & 31);
    if ((e & 31) == lane) taken |= 1u << (e >> 5);
    if (s == 0) first = val;
    const float w = __expf(val - first);
    sum += w;
    if (lane == 0) {
      L.id[t * K + s] = (short)e;
      L.weight[t * K + s] = w;
    }
  }
  if (!p.a.renormalize) {
    float z = 0.0f;
    for (int i = lane; i < E; i += 32) z += __expf(__ldcg(r + i) - first);
    sum = warp_sum(z);
  }
  __syncwarp();
  if (lane < K) L.weight[t * K + lane] = __fdiv_rn(L.weight[t * K + lane], sum);
}

template <int FMT, int NT, int RU, int WARPS, int DEPTH>
__global__ void __launch_bounds__(WARPS * 32, 1) moe_kernel(const __grid_constant__ MoeParams p) {
  using S = Shape<NT, RU, WARPS, DEPTH>;
  constexpr int kThreads = S::kThreads;
  constexpr int CH = NT * RU <= 2 ? 2 : 1;  // chains of dependent products a tile
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ Lists L;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q4 = lane >> 2, t4 = lane & 3;
  const uint4* const queue = reinterpret_cast<const uint4*>(smem_raw + warp * S::kQueue) + lane;  // pieces 32 apart
  const uint32_t queue_at = smem_u32(queue);
  float* const frags = reinterpret_cast<float*>(smem_raw + WARPS * S::kQueue);
  const int T = p.a.tokens, E = p.a.experts, K = p.a.top_k, H = p.a.hidden, I = p.a.inter;

  // ------------------------------------------------- 0: router, x to fp16 --
  {
    // warps of the grid, CTA by CTA, so that few units spread over many SMs
    const int wid = warp * gridDim.x + blockIdx.x, nw = WARPS * gridDim.x;
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
    scale_maxima(p, nw - 1 - wid, nw, lane);
  }
  for (int e = tid; e < E; e += kThreads) L.tokens[e] = 0ull;
  if (!grid_barrier(p.sync)) return;
  if (blockIdx.x == 0 && tid == 0) p.sync[2] = 0u;  // all CTAs of the call before have left its last barrier

  // -------------------------------------------------------- choice, lists --
  if (tid < T) L.xback[tid] = __ldcg(p.xback + 2 * tid);
#pragma unroll 1
  for (int t = warp; t < T; t += WARPS) pick(p, L, t, lane);
  __syncthreads();
  for (int s = tid; s < T * K; s += kThreads) {
    atomicOr(&L.tokens[L.id[s]], 1ull << (s / K));
    if (blockIdx.x == 0) {
      if (p.a.ids) p.a.ids[s] = L.id[s];
      if (p.a.weights) p.a.weights[s] = L.weight[s];
    }
    // the slot's power of two: gate sums are below 2^(eg + 1), up sums below 2^(eu + 1)
    const float l1 = __ldcg(p.xback + 2 * (s / K) + 1), *m = p.smax + (size_t)L.id[s] * 2 * p.chunks;
    float mg = 0.0f, mu = 0.0f;
#pragma unroll 4
    for (int c = 0; c < p.chunks; ++c) {
      mg = fmaxf(mg, __ldcg(m + c));
      mu = fmaxf(mu, __ldcg(m + p.chunks + c));
    }
    const float fmax_v = FMT == F8_E4M3 ? 448.0f : 57344.0f;
    const int eg = (int)(__float_as_uint(mg * fmax_v * l1) >> 23) - 127, eu = (int)(__float_as_uint(mu * fmax_v * l1) >> 23) - 127;
    const int k = max(-126, min(126, eg + eu - 13));
    L.scale[s] = __uint_as_float((uint32_t)(127 - k) << 23);
    L.weight[s] *= __uint_as_float((uint32_t)(127 + k) << 23);  // a slot's result is multiplied by its weight and by what undoes the factor
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

  // loading side of this warp: the next block to ask for. A lane copies its
  // rows' pieces itself: rows r * 8 + q4 of the gate (first) and up (second)
  // box, bytes 16 t4 of both halves of the block.
  int lp = 1, lu = warp / ks1, lb = warp % ks1, put = 0, got = 0;
  const uint8_t* lrow = nullptr;  // the lane's first row of the unit
  auto unit_row = [&]() {
    const bool up = lp == 1;
    const int per = up ? per1 : per2, u = (up ? u1 : u2) + lu, a = u / per;
    const int row = (u - a * per) * (up ? 8 * RU : 16 * RU) + q4;
    lrow = static_cast<const uint8_t*>(up ? p.a.w_gate_up : p.a.w_down) + ((size_t)L.expert[a] * (up ? 2 * I : H) + row) * (up ? H : I) + t4 * 16;
  };
  auto issue = [&]() {
    bool fresh = put == 0;
    if (lp == 1 && lb >= nb1) lb = warp % ks1, lu += WARPS / ks1, fresh = true;
    if (lp == 1 && (lu >= n1 || lb >= nb1)) lp = 2, lu = warp / ks2, lb = warp % ks2, fresh = true;
    if (lp == 2 && lb >= nb2) lb = warp % ks2, lu += WARPS / ks2, fresh = true;
    if (lp == 2 && (lu >= n2 || lb >= nb2)) lp = 3;
    if (lp < 3) {
      if (fresh) unit_row();
      const bool up = lp == 1;
      const int width = up ? H : I;
      const size_t box = (size_t)(up ? I : 8 * RU) * width;  // from a row of the first box to its row of the second
      // rows past the last one of the matrix (the end of a unit that is not whole) read its last
      const int tail = up ? 0x7fffffff : H - 1 - ((u2 + lu) % per2 * (16 * RU) + q4);
      const uint32_t dst = queue_at + put % DEPTH * (S::kPieces * 512);
#pragma unroll
      for (int r = 0; r < RU; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int step = r * 8 + (up ? 0 : k * 8 * RU);  // rows down from the lane's first, second box of the down weights included
          const uint8_t* src = lrow + (up ? (size_t)(r * 8) * width + k * box : (size_t)max(min(step, tail), 0) * width);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int at = lb * 128 + j * 64;
            const bool in = at + t4 * 16 < width;
            copy16(dst + ((r * 2 + k) * 2 + j) * 512, in ? src + at : static_cast<const uint8_t*>(p.a.w_down), in);
          }
        }
      lb += up ? ks1 : ks2;
      ++put;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto next_block = [&]() {  // the lane's pieces of its next block
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
    return queue + got++ % DEPTH * (S::kPieces * 32);
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
    if (warp % ks) return false;
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
    return true;
  };
  // One block's products: fp16 rows xr (8 NT of them, operand order) times the queue's next block.
  const uint16_t* xr[NT];
  auto multiply = [&](int kb, int tiles) {
    uint4 x[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) x[nt][i] = xr[nt] ? *reinterpret_cast<const uint4*>(xr[nt] + kb * 128 + i * 32) : make_uint4(0, 0, 0, 0);
    const uint4* w = next_block();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint4 g[RU], b[RU], y[NT][2];
#pragma unroll
      for (int r = 0; r < RU; ++r) {
        g[r] = w[((r * 2) * 2 + j) * 32];
        b[r] = w[((r * 2 + 1) * 2 + j) * 32];
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
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) x[nt][i] = y[nt][i];
      }
    }
    issue();  // the lane has read its pieces: their place takes the next block
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
    for (int kb = warp % ks1; kb < nb1; kb += ks1) multiply(kb, tiles);
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
        if (!in) continue;
        const float xb = L.xback[L.token[s0 + n]], f = L.scale[s];
#pragma unroll
        for (int r = 0; r < RU; ++r) {
          const int i = i0 + r * 8 + q4;
          const float hv = gate_act(acc[0][r][nt][c] * xb * sg[r], p.a.act) * (acc[0][r][nt][c + 2] * xb * su[r]);
          if (i < I) p.h[(size_t)s * p.ipad + place(i)] = __half_as_ushort(__float2half_rn(hv * f));
        }
      }
    }
  }
  // the columns from inter to the padded width are zero
  if (p.ipad > I)
    for (int x = blockIdx.x * kThreads + tid; x < T * K * (p.ipad - I); x += gridDim.x * kThreads)
      p.h[(size_t)(x / (p.ipad - I)) * p.ipad + place(I + x % (p.ipad - I))] = 0;
  const bool met = grid_barrier(p.sync + 1);
  if (met && blockIdx.x == 0 && tid == 0) p.sync[0] = 0u;
  if (!met) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  // -------------------------------------------------------------- 2: down --
#pragma unroll 1
  for (int u = warp / ks2; u < n2; u += WARPS / ks2) {
    const int a = (u2 + u) / per2, r0 = (u2 + u - a * per2) * (16 * RU);
    const int s0 = L.start[a], cnt = min(L.start[a + 1] - s0, 8 * NT), tiles = (cnt + 7) >> 3;
    float sd[2][RU];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int r = 0; r < RU; ++r) sd[k][r] = __ldg(p.a.s_down + (size_t)L.expert[a] * H + min(r0 + k * 8 * RU + r * 8 + q4, H - 1));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) xr[nt] = nt * 8 + q4 < cnt ? p.h + (size_t)L.slot[s0 + nt * 8 + q4] * p.ipad + t4 * 8 : nullptr;
    clear();
#pragma unroll 1
    for (int kb = warp % ks2; kb < nb2; kb += ks2) multiply(kb, tiles);
    if (!gather(ks2)) continue;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt >= tiles) break;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int n = nt * 8 + 2 * t4 + c;
        if (n >= cnt) continue;
        const int s = L.slot[s0 + n];
        const float wt = L.weight[s];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int r = 0; r < RU; ++r) {
            const int row = r0 + k * 8 * RU + r * 8 + q4;
            if (row < H) p.part[(size_t)s * H + row] = acc[0][r][nt][c + 2 * k] * sd[k][r] * wt;
          }
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!grid_barrier(p.sync + 2)) return;
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

template <int FMT, int NT, int RU, int WARPS, int DEPTH>
cudaError_t launch(const fp8imma_moe_args& a, cudaStream_t st) {
  using S = Shape<NT, RU, WARPS, DEPTH>;
  const auto kern = moe_kernel<FMT, NT, RU, WARPS, DEPTH>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), S::kSmem);
  if (e != cudaSuccess) return e;
  MoeParams p = {};
  p.a = a;
  p.hpad = (a.hidden + 127) & ~127;
  p.ipad = (a.inter + 127) & ~127;
  p.chunks = (a.inter + 1023) / 1024;
  const size_t slots = (size_t)a.tokens * a.top_k;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += (bytes + 255) & ~size_t(255);
    return was;
  };
  const size_t o_logits = take((size_t)a.tokens * a.experts * 4), o_xf = take((size_t)a.tokens * p.hpad * 2), o_back = take((size_t)a.tokens * 8),
               o_max = take((size_t)a.experts * 2 * p.chunks * 4), o_h = take(slots * p.ipad * 2), o_part = take(slots * a.hidden * 4);
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
    p.smax = reinterpret_cast<float*>(base + o_max);
    p.h = reinterpret_cast<uint16_t*>(base + o_h);
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
    e = cudaLaunchKernelEx(&lc, kern, p);
  }
  const cudaError_t e1 = sync.release(st), e2 = work.release(st);
  return e != cudaSuccess ? e : e1 != cudaSuccess ? e1 : e2;
}

// Token tiles by the number of tokens, which an expert may all be given; with
// many tokens a unit has more rows, so that the tokens' operands, read again
// for each unit, cost less beside the weights.
template <int FMT>
cudaError_t launch_nt(const fp8imma_moe_args& a, cudaStream_t st) {
  if (a.tokens <= 2) return launch<FMT, 1, 1, 16, 4>(a, st);
  if (a.tokens <= 8) return launch<FMT, 1, 2, 16, 2>(a, st);
  if (a.tokens <= 16) return launch<FMT, 2, 2, 16, 2>(a, st);
  return launch<FMT, 4, 2, 8, 4>(a, st);
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
