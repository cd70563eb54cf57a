// Low-rank adapters of many requests beside a projection (fp8imma_lora_add):
//   out_t = base_t + s_e B_e (A_e x_t),  e the adapter of token t.
//
// Both products are far below the tensor rate (2 r flops a byte of x and of out),
// so every call is bound by its bytes: x, base, out, and the adapters' weights.
//  * One launch, no scratch: a cluster of CTAs takes a unit, up to kTile
//    neighbouring tokens of one adapter. Each CTA makes the inner sums of a slice
//    of k, the cluster adds them up in distributed shared memory, and each CTA
//    makes a slice of the outputs. Nothing is kept between calls, sums are in a
//    fixed order.
//  * Units are found on the device from the ids: a token begins one where its id
//    differs from the one before or its place is a multiple of kTile.
//  * Products are mma.sync m16n8k16 with the weights as the 16-row operand and 8
//    tokens as the other. The order of k within a product is free, so a lane takes 8
//    neighbouring elements (16 bytes) of a row for two of them, straight from memory.
//  * The inner sums u enter the second product as two 16-bit numbers, hi + lo, so
//    that they keep 16 (bf16) or 22 (fp16) bits: one rounding to the type would show
//    in outputs whose base cancels the addend. fp16 has no range for u; a token's sums
//    are first brought to a largest magnitude of 1 .. 2 by a power of two.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

constexpr int kThreads = 256, kWarps = 8;
constexpr int kMaxTokens = kThreads * 64;  // tokens of a launch: a thread marks where units begin in 64 bits

struct LoraParams {
  fp8imma_lora_args a;
  int cluster;  // CTAs of a cluster
  int split;    // clusters that share a unit's outputs (each makes the inner sums)
  int vec;      // base and out are 16-byte aligned along their contiguous dimension, their other stride a multiple of 16 bytes
  int col;      // tokens are contiguous
};

template <int AT>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (AT == 0)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 elements of k: the 16-byte pieces of rows q4 and q4 + 8 of the weights, and of token q4
template <int AT>
__device__ __forceinline__ void mma32(float (&d)[4], const uint4& lo, const uint4& hi, const uint4& b) {
  mma16<AT>(d, lo.x, hi.x, lo.y, hi.y, b.x, b.y);
  mma16<AT>(d, lo.z, hi.z, lo.w, hi.w, b.z, b.w);
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 peer_load(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void peer_store(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void copy16(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}

__device__ __forceinline__ float d_to_f32(uint16_t b, int type) { return type == FP8IMMA_OUT_F16 ? a16_to_f32<0>(b) : a16_to_f32<1>(b); }
__device__ __forceinline__ uint16_t f32_to_d(float v, int type) { return type == FP8IMMA_OUT_F16 ? f32_to_a16<0>(v) : f32_to_a16<1>(v); }

// Eight inner sums as 16-bit numbers hi and what they leave, lo.
template <int AT>
__device__ __forceinline__ void split8(const float (&u)[8], float f, uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint16_t hb[2], lb[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float x = u[2 * i + c] * f;
      hb[c] = f32_to_a16<AT>(x);
      const float back = a16_to_f32<AT>(hb[c]);
      lb[c] = fabsf(back) < INFINITY ? f32_to_a16<AT>(x - back) : (uint16_t)0;  // infinities and NaN stand in hi
    }
    h[i] = hb[0] | (uint32_t)hb[1] << 16;
    l[i] = lb[0] | (uint32_t)lb[1] << 16;
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}
// The power of two for a token's sums (1 for bf16), and its inverse.
template <int AT>
__device__ __forceinline__ void range_of(float big, float& f, float& back) {
  f = back = 1.0f;
  if (AT == 0 && big > 0.0f && big < INFINITY) {
    const int e = max(-126, min(126, (int)(__float_as_uint(big) >> 23) - 127));
    f = __uint_as_float((uint32_t)(127 - e) << 23);
    back = __uint_as_float((uint32_t)(127 + e) << 23);
  }
}

// Where the units begin among the launch's tokens, 64 tokens a thread at most.
template <int TILE>
struct Units {
  unsigned long long marks;
  int first, mine, base, total;
  __device__ __forceinline__ static bool begins(const int32_t* ids, int t) { return t % TILE == 0 || __ldg(ids + t) != __ldg(ids + t - 1); }
  __device__ __forceinline__ void scan(const fp8imma_lora_args& a, int* s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, each = (a.tokens + kThreads - 1) / kThreads;
    first = threadIdx.x * each;
    marks = 0;
    for (int i = 0; i < each; ++i)
      if (first + i < a.tokens && begins(a.adapter_ids, first + i)) marks |= 1ull << i;
    mine = __popcll(marks);
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s[warp] = x;
    __syncthreads();
    base = x - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += s[w];
      total += s[w];
    }
    __syncthreads();
  }
  // unit u: its first token and the one after its last
  __device__ __forceinline__ void find(const fp8imma_lora_args& a, int u, int* s, int& t0, int& t1) const {
    if (u >= base && u < base + mine) {
      unsigned long long m = marks;
      for (int i = u - base; i > 0; --i) m &= m - 1;
      s[0] = first + __ffsll((long long)m) - 1;
    }
    __syncthreads();
    t0 = s[0];
    const int t = t0 + 1 + (int)threadIdx.x;
    int len = TILE;
    if (threadIdx.x < TILE && (t >= a.tokens || begins(a.adapter_ids, t))) len = 1 + threadIdx.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) len = min(len, __shfl_xor_sync(0xffffffffu, len, o));
    if ((threadIdx.x & 31) == 0) s[1 + (threadIdx.x >> 5)] = len;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < (TILE + 31) / 32; ++w) len = min(len, s[1 + w]);
    t1 = t0 + len;
    __syncthreads();
  }
};

// ------------------------------------------------------------- few tokens --
// Units of up to 8 tokens. Warps deal out 32-element blocks of the CTA's slice of
// k, then 16-row strips of its outputs; the first strip's weights and base are
// asked for before the cluster meets.
template <int AT, int STRIPS>
__global__ void __launch_bounds__(kThreads, STRIPS >= 8 ? 2 : STRIPS >= 4 ? 3 : 4) lora_few_kernel(const __grid_constant__ LoraParams p) {
  constexpr int kBlocks = (STRIPS + 1) / 2;  // 32-element blocks of the rank
  constexpr int kSums = STRIPS * 16 * 8;     // [token][rank row] inner sums of a unit
  constexpr int kRow = STRIPS * 16;
  __shared__ __align__(16) float s_red[kWarps][kSums];
  __shared__ __align__(16) float s_part[kSums], s_u[8 * (kBlocks * 32 + 4)];
  __shared__ int s_find[kWarps + 1];
  pdl_launch_dependents();
  pdl_wait();
  const fp8imma_lora_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q4 = lane >> 2, t4 = lane & 3;
  const int S = p.cluster, c = (int)cluster_rank(), cid = blockIdx.x / S, clusters = gridDim.x / S;
  Units<8> units;
  units.scan(a, s_find);
  const int R = a.rank, K = a.in_features, N = a.out_features;
  const int kb = (K + 31) / 32, kb0 = (int)((int64_t)kb * c / S), kb1 = (int)((int64_t)kb * (c + 1) / S);
  for (int item = cid; item < units.total * p.split; item += clusters) {
    int t0, t1;
    units.find(a, item / p.split, s_find, t0, t1);
    const int tb = t0 & ~7;  // tokens keep their place within 8
    const int e = __ldg(a.adapter_ids + t0);
    const bool held = (unsigned)e < (unsigned)a.adapters;
    const int share = item % p.split * S + c, shares = p.split * S, strips = (N + 15) / 16;
    const int ns0 = (int)((int64_t)strips * share / shares), ns1 = (int)((int64_t)strips * (share + 1) / shares);
    if (!held && a.out == a.base) continue;
    uint4 hi[kBlocks], lo[kBlocks];
    float f[2] = {0.0f, 0.0f};  // of tokens 2 t4 and 2 t4 + 1

    // a strip's weights and base
    uint4 w[kBlocks][2];
    uint16_t have[4];
    auto at = [&](const void*, int64_t ts, int64_t fs, int ns, int k) {
      return (int64_t)(tb + 2 * t4 + (k & 1)) * ts + (int64_t)(ns * 16 + q4 + (k >> 1) * 8) * fs;
    };
    auto inside = [&](int ns, int k) {
      const int t = tb + 2 * t4 + (k & 1);
      return ns < ns1 && t >= t0 && t < t1 && ns * 16 + q4 + (k >> 1) * 8 < N;
    };
    auto fetch = [&](int ns) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = ns * 16 + q4 + h * 8, r = b * 32 + t4 * 8;
          w[b][h] = make_uint4(0, 0, 0, 0);
          if (held && ns < ns1 && n < N && r < R)
            w[b][h] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.lora_b) + ((int64_t)e * N + n) * R + r));
        }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        have[k] = inside(ns, k) ? static_cast<const uint16_t*>(a.base)[at(a.base, a.base_token_stride, a.base_feature_stride, ns, k)] : (uint16_t)0;
    };

    if (held) {
      float acc[STRIPS][4];
#pragma unroll
      for (int s = 0; s < STRIPS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[s][k] = 0.0f;
      const bool live = tb + q4 >= t0 && tb + q4 < t1;
      const uint16_t* xr = static_cast<const uint16_t*>(a.x) + (int64_t)(tb + q4) * a.x_stride;
      const uint16_t* ar = static_cast<const uint16_t*>(a.lora_a) + (int64_t)e * R * K;
#pragma unroll 2
      for (int blk = kb0 + warp; blk < kb1; blk += kWarps) {
        const int k = blk * 32 + t4 * 8;
        uint4 x = make_uint4(0, 0, 0, 0), m[STRIPS][2];
        if (live && k < K) x = __ldg(reinterpret_cast<const uint4*>(xr + k));
#pragma unroll
        for (int s = 0; s < STRIPS; ++s)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = s * 16 + q4 + h * 8;
            m[s][h] = make_uint4(0, 0, 0, 0);
            if (r < R && k < K) m[s][h] = __ldg(reinterpret_cast<const uint4*>(ar + (int64_t)r * K + k));
          }
#pragma unroll
        for (int s = 0; s < STRIPS; ++s) mma32<AT>(acc[s], m[s][0], m[s][1], x);
      }
#pragma unroll
      for (int s = 0; s < STRIPS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) s_red[warp][(2 * t4 + (k & 1)) * kRow + s * 16 + q4 + (k >> 1) * 8] = acc[s][k];
    }
    fetch(ns0 + warp);
    if (held) {
      __syncthreads();
      for (int i = threadIdx.x; i < kSums; i += kThreads) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) s += s_red[k][i];
        s_part[i] = s;
      }
      cluster_arrive();
      cluster_wait();
      for (int i = threadIdx.x; i < kSums / 4; i += kThreads) {
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < S; ++k) {
          const float4 v = peer_load(peer_addr(s_part + i * 4, k));
          s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
        }
        *reinterpret_cast<float4*>(s_u + i * 4 / kRow * (kBlocks * 32 + 4) + i * 4 % kRow) = s;
      }
      cluster_arrive();  // the parts may be written again once all have read them
      __syncthreads();
      float u[kBlocks][8], big = 0.0f;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = b * 32 + t4 * 8 + i;
          u[b][i] = r < kRow ? s_u[q4 * (kBlocks * 32 + 4) + r] : 0.0f;
          big = fmaxf(big, fabsf(u[b][i]));
        }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      float g, back;
      range_of<AT>(big, g, back);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) split8<AT>(u[b], g, hi[b], lo[b]);
      const float scale = a.scales ? __ldg(a.scales + e) : 1.0f;
#pragma unroll
      for (int k = 0; k < 2; ++k) f[k] = scale * __shfl_sync(0xffffffffu, back, (2 * t4 + k) * 4);
    }
    for (int ns = ns0 + warp; ns < ns1; ns += kWarps) {
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      uint16_t was[4];
      if (held) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          mma32<AT>(acc, w[b][0], w[b][1], lo[b]);
          mma32<AT>(acc, w[b][0], w[b][1], hi[b]);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) was[k] = have[k];
      fetch(ns + kWarps);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (inside(ns, k))
          static_cast<uint16_t*>(a.out)[at(a.out, a.out_token_stride, a.out_feature_stride, ns, k)] =
              held ? f32_to_d(fmaf(f[k & 1], acc[k], d_to_f32(was[k], a.d_type)), a.d_type) : was[k];
    }
    if (held) cluster_wait();
  }
}

// ------------------------------------------------------------ many tokens --
// Units of up to 64 tokens. x and the adapter's slice of A stream through shared
// memory 128 elements of k at a time (asynchronous copies, kStages deep); a warp
// multiplies 32 tokens with a quarter of those. The second product goes 32 outputs x 32
// tokens a warp, results pass through shared memory so that base and out are read
// and written along their contiguous dimension.
constexpr int kTile = 64, kStep = 128, kStages = 3;

template <int STRIPS>
struct Many {
  static constexpr int kRow = STRIPS * 16;                          // rank rows, rounded up
  static constexpr int kBlocks = (STRIPS + 1) / 2;                  // 32-element blocks of the rank
  static constexpr int kStageBytes = (kTile + kRow) * kStep * 2;
  static constexpr int kURow = kBlocks > 1 ? kBlocks * 32 + 32 : 32;  // 16-bit elements of a token's hi (or lo): an odd number of 64 bytes
  static constexpr int kRing = kStages * kStageBytes;               // used again for the 4 parts of the sums,
  static constexpr int kParts = 4 * kTile * kRow * 4;               // and then for
  static constexpr int kOut = kWarps * 32 * 40 * 4;                 // outputs and
  static constexpr int kU = 2 * kTile * kURow * 2;                  // hi and lo
  static constexpr int kPool = kRing > kParts ? (kRing > kOut + kU ? kRing : kOut + kU) : (kParts > kOut + kU ? kParts : kOut + kU);
  static constexpr int kSmem = kPool + kTile * kRow * 4;            // and the unit's sums
};

template <int AT, int STRIPS>
__global__ void __launch_bounds__(kThreads, STRIPS >= 8 ? 1 : 2) lora_many_kernel(const __grid_constant__ LoraParams p) {
  using M = Many<STRIPS>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_find[kWarps + 1];
  __shared__ float s_f[kTile];
  float* const parts = reinterpret_cast<float*>(smem);
  float* const s_sum = reinterpret_cast<float*>(smem + M::kPool);
  uint16_t* const s_hi = reinterpret_cast<uint16_t*>(smem + M::kOut);
  uint16_t* const s_lo = s_hi + kTile * M::kURow;
  pdl_launch_dependents();
  pdl_wait();
  const fp8imma_lora_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q4 = lane >> 2, t4 = lane & 3;
  const int S = p.cluster, c = (int)cluster_rank(), cid = blockIdx.x / S, clusters = gridDim.x / S;
  Units<kTile> units;
  units.scan(a, s_find);
  const int R = a.rank, K = a.in_features, N = a.out_features;
  const int ks = (K + kStep - 1) / kStep, ks0 = (int)((int64_t)ks * c / S), ks1 = (int)((int64_t)ks * (c + 1) / S);
  const int tg = warp & 1, kg = warp >> 1;  // 32 tokens, and a quarter of k (or of the outputs)
  for (int item = cid; item < units.total * p.split; item += clusters) {
    int t0, t1;
    units.find(a, item / p.split, s_find, t0, t1);
    const int tb = t0 & ~(kTile - 1);  // tokens keep their place within 64
    const int i0 = t0 - tb, i1 = t1 - tb;
    const int e = __ldg(a.adapter_ids + t0);
    const bool held = (unsigned)e < (unsigned)a.adapters;
    if (!held && a.out == a.base) continue;
    if (held) {
      const uint16_t* xb = static_cast<const uint16_t*>(a.x);
      const uint16_t* ab = static_cast<const uint16_t*>(a.lora_a) + (int64_t)e * R * K;
      auto load = [&](int i) {
        if (i < ks1) {
          uint8_t* dst = smem + (i - ks0) % kStages * M::kStageBytes;
          // 16-byte pieces of 256-byte rows; a piece's place takes the row's lowest bit, so that two rows' fall on all banks
          for (int v = threadIdx.x; v < (kTile + M::kRow) * 16; v += kThreads) {
            const int row = v >> 4, ch = v & 15, k = i * kStep + ch * 8;
            const bool tok = row < kTile;
            const int r = row - kTile;
            const bool on = k < K && (tok ? row >= i0 && row < i1 : r < R);
            const uint16_t* src = !on ? xb + (int64_t)t0 * a.x_stride : tok ? xb + (int64_t)(tb + row) * a.x_stride + k : ab + (int64_t)r * K + k;
            copy16(dst + row * (kStep * 2) + ((ch ^ ((row & 1) << 2)) << 4), src, on);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      float acc[STRIPS][4][4];
#pragma unroll
      for (int s = 0; s < STRIPS; ++s)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[s][t][k] = 0.0f;
      for (int i = 0; i < kStages - 1; ++i) load(ks0 + i);
      for (int i = ks0; i < ks1; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();  // the stage is there, and the one to be filled has been read
        load(i + kStages - 1);
        const uint8_t* st = smem + (i - ks0) % kStages * M::kStageBytes;
        const int ch = kg * 4 + t4;
        auto piece = [&](int row) { return *reinterpret_cast<const uint4*>(st + row * (kStep * 2) + ((ch ^ ((row & 1) << 2)) << 4)); };
        uint4 x[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = piece(tg * 32 + t * 8 + q4);
#pragma unroll
        for (int s = 0; s < STRIPS; ++s) {
          const uint4 lo = piece(kTile + s * 16 + q4), hi = piece(kTile + s * 16 + q4 + 8);
#pragma unroll
          for (int t = 0; t < 4; ++t) mma32<AT>(acc[s][t], lo, hi, x[t]);
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();  // the ring is free
#pragma unroll
      for (int s = 0; s < STRIPS; ++s)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            parts[(kg * kTile + tg * 32 + t * 8 + 2 * t4 + (k & 1)) * M::kRow + s * 16 + q4 + (k >> 1) * 8] = acc[s][t][k];
      __syncthreads();
      // the unit's tokens only, four sums at a time; each CTA of the cluster adds
      // up its share of them over the CTAs and hands it to all
      const int from = i0 * M::kRow / 4, to = i1 * M::kRow / 4;
      for (int v = from + threadIdx.x; v < to; v += kThreads) {
        float4 s = reinterpret_cast<const float4*>(parts)[v];
#pragma unroll
        for (int k = 1; k < 4; ++k) {
          const float4 x = reinterpret_cast<const float4*>(parts)[k * (kTile * M::kRow / 4) + v];
          s = make_float4(s.x + x.x, s.y + x.y, s.z + x.z, s.w + x.w);
        }
        reinterpret_cast<float4*>(parts)[v] = s;
      }
      cluster_arrive();
      cluster_wait();
      const int each = (to - from + S - 1) / S;
      for (int v = from + c * each + (int)threadIdx.x; v < min(to, from + (c + 1) * each); v += kThreads) {
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < S; ++k) {
          const float4 x = peer_load(peer_addr(parts + v * 4, k));
          s = make_float4(s.x + x.x, s.y + x.y, s.z + x.z, s.w + x.w);
        }
        for (int k = 0; k < S; ++k) peer_store(peer_addr(s_sum + v * 4, k), s);
      }
      cluster_arrive();
      cluster_wait();
      {
        // a warp takes 8 tokens, four lanes a token
        const int i = warp * 8 + q4;
        const bool live = i >= i0 && i < i1;
        float u[M::kBlocks][8], big = 0.0f;
#pragma unroll
        for (int b = 0; b < M::kBlocks; ++b)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int r = b * 32 + t4 * 8 + j;
            u[b][j] = live && r < M::kRow ? s_sum[i * M::kRow + r] : 0.0f;
            big = fmaxf(big, fabsf(u[b][j]));
          }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        float g, back;
        range_of<AT>(big, g, back);
#pragma unroll
        for (int b = 0; b < M::kBlocks; ++b) {
          uint4 hi, lo;
          split8<AT>(u[b], g, hi, lo);
          *reinterpret_cast<uint4*>(s_hi + i * M::kURow + b * 32 + t4 * 8) = hi;
          *reinterpret_cast<uint4*>(s_lo + i * M::kURow + b * 32 + t4 * 8) = lo;
        }
        if (t4 == 0) s_f[i] = back * (a.scales ? __ldg(a.scales + e) : 1.0f);
      }
      __syncthreads();
    }

    const int share = item % p.split * S + c, shares = p.split * S, groups = (N + 31) / 32;
    const int g0 = (int)((int64_t)groups * share / shares), g1 = (int)((int64_t)groups * (share + 1) / shares);
    float* const stage = reinterpret_cast<float*>(smem) + warp * (32 * 40);
    const bool any = tg * 32 < i1 && tg * 32 + 32 > i0;  // the warp's 32 tokens hold some of the unit
    for (int g = g0 + kg; any && g < g1; g += 4) {
      const int n0 = g * 32;
      // what this lane reads and writes: four runs of 8 elements along the contiguous dimension
      auto run = [&](int j, int& i, int& n) {  // first token (within the 64) and output of run j
        const int line = j * 8 + (lane >> 2), at = (lane & 3) * 8;
        i = tg * 32 + (p.col ? at : line);
        n = n0 + (p.col ? line : at);
      };
      auto whole = [&](int i, int n) {
        return p.vec && (p.col ? i >= i0 && i + 8 <= i1 && n < N : i >= i0 && i < i1 && n + 8 <= N);
      };
      uint4 was[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int i, n;
        run(j, i, n);
        if (whole(i, n)) was[j] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.base) + (int64_t)(tb + i) * a.base_token_stride + (int64_t)n * a.base_feature_stride);
      }
      if (held) {
        float acc[2][4][4];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[s][t][k] = 0.0f;
#pragma unroll
        for (int b = 0; b < M::kBlocks; ++b) {
          uint4 w[2][2];
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int n = n0 + s * 16 + h * 8 + q4, r = b * 32 + t4 * 8;
              w[s][h] = make_uint4(0, 0, 0, 0);
              if (n < N && r < R) w[s][h] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.lora_b) + ((int64_t)e * N + n) * R + r));
            }
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int i = tg * 32 + t * 8 + q4;
            const uint4 hi = *reinterpret_cast<const uint4*>(s_hi + i * M::kURow + b * 32 + t4 * 8);
            const uint4 lo = *reinterpret_cast<const uint4*>(s_lo + i * M::kURow + b * 32 + t4 * 8);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              mma32<AT>(acc[s][t], w[s][0], w[s][1], lo);
              mma32<AT>(acc[s][t], w[s][0], w[s][1], hi);
            }
          }
        }
        __syncwarp();
        // row stride 36 (outputs contiguous) or 40 (tokens contiguous): stores fall on all banks
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int n = s * 16 + h * 8 + q4, i = t * 8 + 2 * t4;
              const float x = acc[s][t][2 * h] * s_f[tg * 32 + i], y = acc[s][t][2 * h + 1] * s_f[tg * 32 + i + 1];
              if (p.col) *reinterpret_cast<float2*>(stage + n * 40 + i) = make_float2(x, y);
              else stage[i * 36 + n] = x, stage[(i + 1) * 36 + n] = y;
            }
        __syncwarp();
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int i, n;
        run(j, i, n);
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.0f;
        if (held) {
          const float4* s = reinterpret_cast<const float4*>(stage + (j * 8 + (lane >> 2)) * (p.col ? 40 : 36) + (lane & 3) * 8);
          const float4 x = s[0], y = s[1];
          v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
        }
        uint16_t* const dst = static_cast<uint16_t*>(a.out) + (int64_t)(tb + i) * a.out_token_stride + (int64_t)n * a.out_feature_stride;
        if (whole(i, n)) {
          uint32_t w[4] = {was[j].x, was[j].y, was[j].z, was[j].w};
          if (held) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = (uint32_t)f32_to_d(d_to_f32((uint16_t)w[k], a.d_type) + v[2 * k], a.d_type) |
                     (uint32_t)f32_to_d(d_to_f32((uint16_t)(w[k] >> 16), a.d_type) + v[2 * k + 1], a.d_type) << 16;
          }
          *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
          const uint16_t* src = static_cast<const uint16_t*>(a.base) + (int64_t)(tb + i) * a.base_token_stride + (int64_t)n * a.base_feature_stride;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int ii = i + (p.col ? k : 0), nn = n + (p.col ? 0 : k);
            if (ii >= i0 && ii < i1 && nn < N) {
              const uint16_t b = src[k];
              dst[k] = held ? f32_to_d(d_to_f32(b, a.d_type) + v[k], a.d_type) : b;
            }
          }
        }
      }
    }
    __syncthreads();  // outputs' places are the next unit's ring
  }
  // no CTA leaves while another may still write its sums: each has passed the last
  // barrier after those writes, so nothing is left to wait for
}

template <class Kern>
cudaError_t launch_clusters(Kern kern, const LoraParams& p, int clusters, int smem, cudaStream_t st) {
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  lc.gridDim = dim3((unsigned)(clusters * p.cluster));
  lc.blockDim = dim3(kThreads);
  lc.dynamicSmemBytes = (size_t)smem;
  lc.stream = st;
  lc.attrs = attr;
  lc.numAttrs = api_pdl() ? 2 : 1;
  return cudaLaunchKernelEx(&lc, kern, p);
}

template <int AT, int STRIPS>
cudaError_t launch(LoraParams& p, cudaStream_t st) {
  const int sms = num_sms_current(), T = p.a.tokens;
  p.cluster = 8;
  if (T <= 128) {
    // a unit of its own for each token at most: as many clusters share a unit's
    // outputs as the SMs have room for, each with a strip a warp or so
    const int strips = (p.a.out_features + 15) / 16;
    p.split = std::max(1, std::min(sms / (T * p.cluster), (strips + p.cluster * kWarps - 1) / (p.cluster * kWarps)));
    return launch_clusters(lora_few_kernel<AT, STRIPS>, p, T * p.split, 0, st);
  }
  p.split = 1;
  return launch_clusters(lora_many_kernel<AT, STRIPS>, p, std::min(T, 2 * sms / p.cluster), Many<STRIPS>::kSmem, st);
}

}  // namespace
}  // namespace fp8imma_b200

using namespace fp8imma_b200;

extern "C" int fp8imma_lora_add(const fp8imma_lora_args* a, void* stream) {
  FP8IMMA_RANGE("fp8imma_lora_add");
  if (!a) return (int)cudaErrorInvalidValue;
  if (a->tokens <= 0 || a->in_features <= 0 || a->out_features <= 0 || a->rank <= 0 || a->adapters <= 0) return (int)cudaErrorInvalidConfiguration;
  if (a->a_type < 0 || a->a_type > 1 || a->d_type < 0 || a->d_type > 1) return (int)cudaErrorInvalidValue;
  if (a->rank > FP8IMMA_LORA_MAX_RANK || a->rank % 8 || a->in_features % 8) return (int)cudaErrorInvalidValue;
  if (!a->x || !a->lora_a || !a->lora_b || !a->adapter_ids || !a->base || !a->out) return (int)cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->lora_a) | reinterpret_cast<uintptr_t>(a->lora_b)) & 15u) return (int)cudaErrorInvalidValue;
  if (a->x_stride < 0 || a->x_stride % 8) return (int)cudaErrorInvalidValue;
  const int64_t bt = a->base_token_stride, bf = a->base_feature_stride, ot = a->out_token_stride, of = a->out_feature_stride;
  if (bt < 0 || bf < 0 || ot < 0 || of < 0) return (int)cudaErrorInvalidValue;
  const bool row = bf == 1 && of == 1, col = !row && bt == 1 && ot == 1;
  if (!row && !col) return (int)cudaErrorInvalidValue;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a->base) | reinterpret_cast<uintptr_t>(a->out) | (uintptr_t)((row ? bt | ot : bf | of) * 2);
  if (bits & 1u) return (int)cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int t = 0; t < a->tokens; t += kMaxTokens) {
    LoraParams p = {};
    p.a = *a;
    p.a.tokens = std::min(a->tokens - t, kMaxTokens);
    p.a.x = static_cast<const uint16_t*>(a->x) + t * a->x_stride;
    p.a.adapter_ids = a->adapter_ids + t;
    p.a.base = static_cast<const uint16_t*>(a->base) + t * bt;
    p.a.out = static_cast<uint16_t*>(a->out) + t * ot;
    p.vec = (bits & 15u) == 0;
    p.col = col;
    cudaError_t e;
    const int strips = (a->rank + 15) / 16;
    if (a->a_type == FP8IMMA_A_F16) e = strips <= 1 ? launch<0, 1>(p, st) : strips <= 2 ? launch<0, 2>(p, st) : strips <= 4 ? launch<0, 4>(p, st) : launch<0, 8>(p, st);
    else e = strips <= 1 ? launch<1, 1>(p, st) : strips <= 2 ? launch<1, 2>(p, st) : strips <= 4 ? launch<1, 4>(p, st) : launch<1, 8>(p, st);
    if (e != cudaSuccess) return (int)e;
  }
  return 0;
}
