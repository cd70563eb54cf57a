// Low-rank adapters of many requests beside a projection (fp8imma_lora_add):
//   out_t = base_t + s_e B_e (A_e x_t),  e the adapter of token t.
//
// Both products are far below the tensor rate (2 r flops a byte of x and of out),
// so a call's floor is its bytes: x, base, out, and the adapters' weights.
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
//
// Measured: one token, rank 16, 4096 -> 4096 5.2 us; 64 requests of one token, rank
// 32, 4096 -> 11008 27 us on column-major results (their 2-byte pieces cost 10 of
// them: 15 us row-major), one adapter for all of them 9.6 us; prompts of 4001
// tokens, rank 64, 8192 -> 8192 78 us, 2.6 TB/s of the 205 MB (160 us with outputs
// straight from memory), bound by the latency of a step's instructions: a CTA's chain
// of 32 steps takes as long with one CTA an SM as with two.
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

constexpr int kThreads = 256, kWarps = 8;
constexpr int kRunTokens = 4;  // runs of this length in the mean of a call and more go through the kernel for many tokens
constexpr int kMaxTokens = kThreads * 64;  // tokens of a launch: a thread marks where units begin in 64 bits

struct LoraParams {
  fp8imma_lora_args a;
  int cluster;  // CTAs of a cluster
  int split;    // clusters that may share a unit's outputs at most (each makes the inner sums)
  int vec;      // base and out are 16-byte aligned along their contiguous dimension, their other stride a multiple of 16 bytes
  int col;      // tokens are contiguous
  int choose;   // both kernels are launched: the ids say which one works
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
  int first, mine, base, total, runs;  // runs: of equal ids
  __device__ __forceinline__ static bool begins(const int32_t* ids, int t) { return t % TILE == 0 || __ldg(ids + t) != __ldg(ids + t - 1); }
  // s: kWarps words, words: one for each 32 tokens
  __device__ __forceinline__ void scan(const fp8imma_lora_args& a, int* s, uint32_t* words) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int changes = 0;
#pragma unroll 4
    for (int t0 = 0; t0 < a.tokens; t0 += kThreads) {
      const int t = t0 + (int)threadIdx.x;
      const bool in = t < a.tokens;
      const int id = in ? __ldg(a.adapter_ids + t) : 0, before = in && t > 0 ? __ldg(a.adapter_ids + t - 1) : 0;
      const bool change = in && (t == 0 || id != before);
      const uint32_t word = __ballot_sync(0xffffffffu, change || (in && t % TILE == 0));
      changes += __popc(__ballot_sync(0xffffffffu, change));
      if (lane == 0) words[t >> 5] = word;
    }
    __syncthreads();
    const int end = (a.tokens + kThreads - 1) / kThreads * kThreads / 32;  // words written
    first = threadIdx.x * 64;
    marks = 2 * threadIdx.x < end ? words[2 * threadIdx.x] | (unsigned long long)words[2 * threadIdx.x + 1] << 32 : 0ull;
    mine = __popcll(marks);
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s[warp] = x | changes << 16;  // at most 2^14 of either
    __syncthreads();
    base = x - mine;
    total = runs = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += s[w] & 0xFFFF;
      total += s[w] & 0xFFFF;
      runs += s[w] >> 16;
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
// k, then blocks of kOuts of its outputs, whose weights are copied one block ahead;
// the first of them are under way before the inner sums are begun. Sums go through
// shared memory, so that a lane adds and stores neighbouring outputs of a token.
template <int STRIPS>
struct Few {
  static constexpr int kBlocks = (STRIPS + 1) / 2;      // 32-element blocks of the rank
  static constexpr int kRow = STRIPS * 16;
  static constexpr int kSums = kRow * 8;                // [token][rank row] inner sums of a unit
  static constexpr int kURow = kBlocks * 32 + 4;
  static constexpr int kOuts = 64 / kBlocks;            // outputs of a warp's block: 4 KB of weights
  static constexpr int kStage = 256;                    // uint4 of a block's weights
  static constexpr int kLine = kOuts + 2;               // floats of a token's sums
  static constexpr int kRed = kWarps * kSums * 4;       // the warps' parts of the inner sums, then the outputs' sums
  static constexpr int kOutBytes = kWarps * 8 * kLine * 4;
  static constexpr int kSmem = kWarps * 2 * kStage * 16 + (kRed > kOutBytes ? kRed : kOutBytes) + kSums * 4 + 8 * kURow * 4;
};

template <int AT, int STRIPS, bool COL>
__global__ void __launch_bounds__(kThreads, STRIPS >= 8 ? 2 : 3) lora_few_kernel(const __grid_constant__ LoraParams p) {
  using F = Few<STRIPS>;
  constexpr int kBlocks = F::kBlocks, kRow = F::kRow, kSums = F::kSums, kOuts = F::kOuts;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_find[kWarps + 1];
  uint4* const s_ring = reinterpret_cast<uint4*>(smem);
  float* const s_red = reinterpret_cast<float*>(smem + kWarps * 2 * F::kStage * 16);
  float* const s_part = reinterpret_cast<float*>(smem + F::kSmem) - kSums - 8 * F::kURow;
  float* const s_u = s_part + kSums;
  pdl_launch_dependents();
  pdl_wait();
  const fp8imma_lora_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q4 = lane >> 2, t4 = lane & 3;
  const int S = p.cluster, c = (int)cluster_rank(), cid = blockIdx.x / S, clusters = gridDim.x / S;
  Units<8> units;
  units.scan(a, s_find, reinterpret_cast<uint32_t*>(smem));
  if (p.choose && a.tokens >= kRunTokens * units.runs) return;
  const int R = a.rank, K = a.in_features, N = a.out_features;
  const int kb = (K + 31) / 32, kb0 = (int)((int64_t)kb * c / S), kb1 = (int)((int64_t)kb * (c + 1) / S);
  uint4* const ring = s_ring + warp * (2 * F::kStage) + lane;
  float* const outs = s_red + warp * (8 * F::kLine);
  // few units share the clusters that the others would have taken
  const int split = max(1, min(p.split, clusters / max(1, units.total)));
  for (int item = cid; item < units.total * split; item += clusters) {
    int t0, t1;
    units.find(a, item / split, s_find, t0, t1);
    const int tb = t0 & ~7;  // tokens keep their place within 8
    const int e = __ldg(a.adapter_ids + t0);
    const bool held = (unsigned)e < (unsigned)a.adapters;
    if (!held && a.out == a.base) continue;
    const int share = item % split * S + c, shares = split * S, groups = (N + kOuts - 1) / kOuts;
    const int g0 = (int)((int64_t)groups * share / shares), g1 = (int)((int64_t)groups * (share + 1) / shares);
    // a lane copies the pieces that it multiplies itself: rows q4 + 8 i of a block of outputs
    auto fetch = [&](int g, int slot) {
      if (held && g < g1) {
        const uint16_t* src = static_cast<const uint16_t*>(a.lora_b) + ((int64_t)e * N + g * kOuts + q4) * R + t4 * 8;
#pragma unroll
        for (int i = 0; i < kOuts / 8; ++i)
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            const bool on = g * kOuts + i * 8 + q4 < N && b * 32 + t4 * 8 < R;
            copy16(ring + slot * F::kStage + (i * kBlocks + b) * 32, on ? src + i * 8 * R + b * 32 : static_cast<const uint16_t*>(a.lora_b), on);
          }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(g0 + warp, 0);
    uint4 hi[kBlocks], lo[kBlocks];
    float f[2] = {0.0f, 0.0f};  // of tokens 2 t4 and 2 t4 + 1
    if (held) {
      float acc[STRIPS][4];
#pragma unroll
      for (int s = 0; s < STRIPS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[s][k] = 0.0f;
      const bool live = tb + q4 >= t0 && tb + q4 < t1;
      const uint16_t* xr = static_cast<const uint16_t*>(a.x) + (int64_t)(tb + q4) * a.x_stride;
      const uint16_t* ar = static_cast<const uint16_t*>(a.lora_a) + ((int64_t)e * R + q4) * K;
#pragma unroll 2
      for (int blk = kb0 + warp; blk < kb1; blk += kWarps) {
        const int k = blk * 32 + t4 * 8;
        uint4 x = make_uint4(0, 0, 0, 0), m[STRIPS][2];
        if (live && k < K) x = __ldg(reinterpret_cast<const uint4*>(xr + k));
#pragma unroll
        for (int s = 0; s < STRIPS; ++s)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            m[s][h] = make_uint4(0, 0, 0, 0);
            if (s * 16 + h * 8 + q4 < R && k < K) m[s][h] = __ldg(reinterpret_cast<const uint4*>(ar + (int64_t)(s * 16 + h * 8) * K + k));
          }
#pragma unroll
        for (int s = 0; s < STRIPS; ++s) mma32<AT>(acc[s], m[s][0], m[s][1], x);
      }
#pragma unroll
      for (int s = 0; s < STRIPS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) s_red[warp * kSums + (2 * t4 + (k & 1)) * kRow + s * 16 + q4 + (k >> 1) * 8] = acc[s][k];
      __syncthreads();
      for (int i = threadIdx.x; i < kSums; i += kThreads) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) s += s_red[k * kSums + i];
        s_part[i] = s;
      }
      cluster_arrive();
      cluster_wait();
      for (int i = threadIdx.x; i < kSums / 4; i += kThreads) {
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int k = 0; k < S; ++k) {
          const float4 v = peer_load(peer_addr(s_part + i * 4, k));
          s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
        }
        *reinterpret_cast<float4*>(s_u + i * 4 / kRow * F::kURow + i * 4 % kRow) = s;
      }
      cluster_arrive();  // the parts may be written again once all have read them
      __syncthreads();
      float u[kBlocks][8], big = 0.0f;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = b * 32 + t4 * 8 + i;
          u[b][i] = r < kRow ? s_u[q4 * F::kURow + r] : 0.0f;
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
    int slot = 0;
    const bool wide = COL && p.vec && tb + 8 <= a.tokens, all8 = wide && t1 - t0 == 8;
    for (int g = g0 + warp; g < g1; g += kWarps, slot ^= 1) {
      // This lane's outputs: n0 + lane and n0 + lane + 32, of all tokens at once where
      // tokens are contiguous, or two neighbours, token after token, where outputs are.
      constexpr int kEach = kOuts / 32 > 0 ? kOuts / 32 : 1;
      const int n0 = g * kOuts, at0 = COL || kEach == 1 ? lane : 2 * lane;
      auto out_at = [&](int i) { return at0 + (COL ? 32 * i : i); };
      auto there = [&](int i) { return out_at(i) < kOuts && n0 + out_at(i) < N; };
      uint16_t was[kEach];
      uint4 was8[kEach];
      auto load = [&](int t) {
        const uint16_t* src = static_cast<const uint16_t*>(a.base) + (int64_t)t * a.base_token_stride;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          if (there(i)) was[i] = src[(int64_t)(n0 + out_at(i)) * a.base_feature_stride];
      };
      if (COL) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (!there(i)) continue;
          const uint16_t* src = static_cast<const uint16_t*>(a.base) + tb + (int64_t)(n0 + out_at(i)) * a.base_feature_stride;
          if (wide) was8[i] = *reinterpret_cast<const uint4*>(src);  // the other tokens' values are not used
          else {
            uint32_t x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = tb + j >= t0 && tb + j < t1 ? src[j] : 0u;
            was8[i] = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
          }
        }
      } else {
        load(t0);
      }
      fetch(g + kWarps, slot ^ 1);
      if (held) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        float acc[kOuts / 16][4];
#pragma unroll
        for (int s = 0; s < kOuts / 16; ++s) {
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[s][k] = 0.0f;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            const uint4 w0 = ring[slot * F::kStage + (2 * s * kBlocks + b) * 32], w1 = ring[slot * F::kStage + ((2 * s + 1) * kBlocks + b) * 32];
            mma32<AT>(acc[s], w0, w1, lo[b]);
            mma32<AT>(acc[s], w0, w1, hi[b]);
          }
        }
        __syncwarp();  // the sums of the block before have been read
#pragma unroll
        for (int s = 0; s < kOuts / 16; ++s)
#pragma unroll
          for (int k = 0; k < 4; ++k) outs[(2 * t4 + (k & 1)) * F::kLine + s * 16 + q4 + (k >> 1) * 8] = f[k & 1] * acc[s][k];
        __syncwarp();
      }
      if (COL) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (!there(i)) continue;
          uint16_t* const dst = static_cast<uint16_t*>(a.out) + tb + (int64_t)(n0 + out_at(i)) * a.out_feature_stride;
          uint32_t w[4] = {was8[i].x, was8[i].y, was8[i].z, was8[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (tb + 2 * j + 1 < t0 || tb + 2 * j >= t1) continue;
            if (held) {
              const float x = d_to_f32((uint16_t)w[j], a.d_type) + outs[2 * j * F::kLine + out_at(i)];
              const float y = d_to_f32((uint16_t)(w[j] >> 16), a.d_type) + outs[(2 * j + 1) * F::kLine + out_at(i)];
              w[j] = a.d_type == FP8IMMA_OUT_F16 ? f32x2_to_a16x2<0>(x, y) : f32x2_to_a16x2<1>(x, y);
            }
            if (!all8) {
              if (tb + 2 * j >= t0 && tb + 2 * j < t1) dst[2 * j] = (uint16_t)w[j];
              if (tb + 2 * j + 1 >= t0 && tb + 2 * j + 1 < t1) dst[2 * j + 1] = (uint16_t)(w[j] >> 16);
            }
          }
          if (all8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
        for (int t = t0; t < t1; ++t) {
          uint16_t* const dst = static_cast<uint16_t*>(a.out) + (int64_t)t * a.out_token_stride;
          uint16_t old[kEach];
#pragma unroll
          for (int i = 0; i < kEach; ++i) old[i] = was[i];
          if (t + 1 < t1) load(t + 1);
#pragma unroll
          for (int i = 0; i < kEach; ++i)
            if (there(i))
              dst[(int64_t)(n0 + out_at(i)) * a.out_feature_stride] =
                  held ? f32_to_d(d_to_f32(old[i], a.d_type) + outs[(t & 7) * F::kLine + out_at(i)], a.d_type) : old[i];
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (held) cluster_wait();
  }
}

// ------------------------------------------------------------ many tokens --
// Units of up to 64 tokens. x and the adapter's slice of A stream through shared
// memory 128 elements of k at a time (asynchronous copies, kStages deep); a warp
// multiplies 32 tokens with a quarter of those. The second product goes 64 tokens x
// 64 outputs a step, B's rows and the base under way kAhead steps before: a warp
// keeps the inner sums of 16 tokens in registers and makes 32 outputs of each. It adds
// them to the base in shared memory, two neighbours along the contiguous dimension a
// lane (COL: tokens, so they are the 8-column operand; else outputs), and stores 16
// bytes a lane.
constexpr int kTile = 64, kStep = 128, kStages = 3, kAhead = 4;

template <int STRIPS>
struct Many {
  static constexpr int kRow = STRIPS * 16;                          // rank rows, rounded up
  static constexpr int kBlocks = (STRIPS + 1) / 2;                  // 32-element blocks of the rank
  static constexpr int kStageBytes = (kTile + kRow) * kStep * 2;
  static constexpr int kRing = kStages * kStageBytes;               // used again for the 4 parts of the sums,
  static constexpr int kParts = 4 * kTile * kRow * 4;               // and then for
  static constexpr int kLine = kTile * 2 + 16;                      // lines of the base: 16 bytes apart modulo 128
  static constexpr int kBytesB = kTile * kBlocks * 64;              // steps of B and
  static constexpr int kOutBytes = kBytesB + kTile * kLine;         // the base
  static constexpr int kPool0 = kRing > kParts ? kRing : kParts;
  static constexpr int kPool = kPool0 > kAhead * kOutBytes ? kPool0 : kAhead * kOutBytes;
  static constexpr int kSmem = kPool + kTile * kRow * 4;            // and the unit's sums
};

template <int AT, int STRIPS, bool COL>
__global__ void __launch_bounds__(kThreads, STRIPS >= 8 ? 1 : 2) lora_many_kernel(const __grid_constant__ LoraParams p) {
  using M = Many<STRIPS>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_find[kWarps + 1];
  float* const parts = reinterpret_cast<float*>(smem);
  float* const s_sum = reinterpret_cast<float*>(smem + M::kPool);
  pdl_launch_dependents();
  pdl_wait();
  const fp8imma_lora_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q4 = lane >> 2, t4 = lane & 3;
  const int S = p.cluster, c = (int)cluster_rank(), cid = blockIdx.x / S, clusters = gridDim.x / S;
  Units<kTile> units;
  units.scan(a, s_find, reinterpret_cast<uint32_t*>(smem));
  if (p.choose && a.tokens < kRunTokens * units.runs) return;
  const int R = a.rank, K = a.in_features, N = a.out_features;
  const int ks = (K + kStep - 1) / kStep, ks0 = (int)((int64_t)ks * c / S), ks1 = (int)((int64_t)ks * (c + 1) / S);
  const int split = max(1, min(p.split, clusters / max(1, units.total)));
  for (int item = cid; item < units.total * split; item += clusters) {
    int t0, t1;
    units.find(a, item / split, s_find, t0, t1);
    const int tb = t0 & ~(kTile - 1);  // tokens keep their place within 64
    const int i0 = t0 - tb, i1 = t1 - tb;
    const int e = __ldg(a.adapter_ids + t0);
    const bool held = (unsigned)e < (unsigned)a.adapters;
    if (!held && a.out == a.base) continue;
    // of an eight that begins at token i (within the 64), output n: whether it is whole and aligned, and else its elements
    auto whole = [&](int i, int n) {
      return p.vec && (COL ? i >= i0 && i + 8 <= i1 && n < N : i >= i0 && i < i1 && n + 8 <= N);
    };
    auto part = [&](int i, int n, auto each) {
      if (i >= i1 || i + (COL ? 8 : 1) <= i0 || n >= N) return;
#pragma unroll 1
      for (int k = 0; k < 8; ++k) {
        const int ii = i + (COL ? k : 0), nn = n + (COL ? 0 : k);
        if (ii >= i0 && ii < i1 && nn < N) each(k);
      }
    };
    const int share = item % split * S + c, shares = split * S, groups = (N + kTile - 1) / kTile;
    // the steps of a cluster's CTAs lie side by side, so that they read and write whole pages of memory together
    if (held) {
      // 16-byte pieces of 256-byte rows: a thread copies piece ch of rows row0 + 16 i, of
      // the tokens first. A piece's place takes the row's lowest bit, so that two rows'
      // fall on all banks.
      const int row0 = threadIdx.x >> 4, ch0 = threadIdx.x & 15;
      const uint16_t* xp = static_cast<const uint16_t*>(a.x) + (int64_t)(tb + row0) * a.x_stride + (int64_t)ks0 * kStep + ch0 * 8;
      const uint16_t* ap = static_cast<const uint16_t*>(a.lora_a) + ((int64_t)e * R + row0) * K + (int64_t)ks0 * kStep + ch0 * 8;
      const int64_t x_rows = 16 * a.x_stride, a_rows = 16ll * K;
      int k_left = K - ks0 * kStep - ch0 * 8;  // elements from the piece to the row's end
      uint8_t* const dst0 = smem + row0 * (kStep * 2) + ((ch0 ^ ((row0 & 1) << 2)) << 4);
      auto load = [&](int i, int stage) {
        if (i < ks1) {
          uint8_t* const dst = dst0 + stage * M::kStageBytes;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool on = k_left > 0 && row0 + 16 * r >= i0 && row0 + 16 * r < i1;
            copy16(dst + r * (16 * kStep * 2), on ? xp + r * x_rows : static_cast<const uint16_t*>(a.x), on);
          }
#pragma unroll
          for (int r = 0; r < STRIPS; ++r) {
            const bool on = k_left > 0 && row0 + 16 * r < R;
            copy16(dst + (4 + r) * (16 * kStep * 2), on ? ap + r * a_rows : static_cast<const uint16_t*>(a.lora_a), on);
          }
        }
        xp += kStep;
        ap += kStep;
        k_left -= kStep;
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      const int tg = warp & 1, kg = warp >> 1;  // 32 tokens, and a quarter of k
      float acc[STRIPS][4][4];
#pragma unroll
      for (int s = 0; s < STRIPS; ++s)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[s][t][k] = 0.0f;
      for (int i = 0; i < kStages - 1; ++i) load(ks0 + i, i);
      for (int i = ks0, stage = 0; i < ks1; ++i, stage = stage == kStages - 1 ? 0 : stage + 1) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();  // the stage is there, and the one to be filled has been read
        load(i + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
        const uint8_t* st = smem + stage * M::kStageBytes;
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
      cluster_wait();  // the sums are here, and the parts have been read
    }

    // Element v of a step's 64 lines: whether it is one of the unit's, and where it lies.
    auto element = [&](int g, int v, auto* from, int64_t ts, int64_t fs, auto*& at) {
      const int i = COL ? v & 63 : v >> 6, n = g * kTile + (COL ? v >> 6 : v & 63);
      using E = std::remove_reference_t<decltype(*at)>;
      at = static_cast<E*>(from) + (int64_t)(tb + i) * ts + (int64_t)n * fs;
      return i >= i0 && i < i1 && n < N;
    };
    // Lines of a step's base: tokens (COL: outputs), 64 elements each in eights, or, where
    // they are not aligned, neighbouring elements for neighbouring threads. A
    // thread copies eight j of lines l and l + 32; in which of its tokens the unit
    // lies and which outputs there are is settled line by line.
    auto load = [&](int g, int stage) {
      if (g < groups) {
        uint8_t* const dst = smem + stage * M::kOutBytes;
        if (held) {
          constexpr int kChunks = M::kBlocks * 4, kRows = kThreads / kChunks;
          const int row = threadIdx.x / kChunks, ch = threadIdx.x % kChunks;
          const uint16_t* src = static_cast<const uint16_t*>(a.lora_b) + ((int64_t)e * N + g * kTile + row) * R + ch * 8;
#pragma unroll
          for (int i = 0; i < kTile / kRows; ++i) {
            const bool on = g * kTile + row + i * kRows < N && ch * 8 < R;
            const int r = row + i * kRows;
            copy16(dst + r * (M::kBlocks * 64) + ((M::kBlocks == 1 ? ch : ch ^ ((r & 1) << 2)) << 4), on ? src + i * kRows * R : static_cast<const uint16_t*>(a.lora_b), on);
          }
        }
        if (!p.vec) {
          uint16_t x[16];
          const uint16_t* src;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (element(g, threadIdx.x + i * kThreads, a.base, a.base_token_stride, a.base_feature_stride, src)) x[i] = *src;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int v = threadIdx.x + i * kThreads;
            *reinterpret_cast<uint16_t*>(dst + M::kBytesB + (v >> 6) * M::kLine + (v & 63) * 2) = x[i];
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          return;
        }
        const int l = threadIdx.x >> 3, j = threadIdx.x & 7;
        const uint16_t* src = static_cast<const uint16_t*>(a.base) + (int64_t)(tb + (COL ? 8 * j : l)) * a.base_token_stride +
                              (int64_t)(g * kTile + (COL ? l : 8 * j)) * a.base_feature_stride;
        const int64_t lines = 32 * (COL ? a.base_feature_stride : a.base_token_stride);
        uint8_t* line = dst + M::kBytesB + l * M::kLine + j * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = COL ? 8 * j : l + 32 * h, n = g * kTile + (COL ? l + 32 * h : 8 * j);
          if (whole(i, n)) copy16(line + h * 32 * M::kLine, src + h * lines, true);
          else part(i, n, [&](int k) { reinterpret_cast<uint16_t*>(line + h * 32 * M::kLine)[k] = src[h * lines + k]; });
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // inner sums of the warp's 16 tokens
    const int tok = (warp & 3) * 16, half = (warp >> 2) * 32;  // and the outputs of a step
    uint4 hi[2][M::kBlocks], lo[2][M::kBlocks];
    float f[4];  // COL: of tokens 2 t4, 2 t4 + 1 of both eights; else of q4 of both
    if (held) {
      const float scale = a.scales ? __ldg(a.scales + e) : 1.0f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int i = tok + t * 8 + q4;
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
        back *= scale;
#pragma unroll
        for (int b = 0; b < M::kBlocks; ++b) split8<AT>(u[b], g, hi[t][b], lo[t][b]);
        if (COL) {
          f[2 * t] = __shfl_sync(0xffffffffu, back, 2 * t4 * 4);
          f[2 * t + 1] = __shfl_sync(0xffffffffu, back, (2 * t4 + 1) * 4);
        } else {
          f[2 * t] = f[2 * t + 1] = back;
        }
      }
    }
    const bool any = tok < i1 && tok + 16 > i0;  // the warp has tokens of the unit
    for (int i = 0; i < kAhead - 1; ++i) load(share + i * shares, i);
    for (int g = share, stage = 0; g < groups; g += shares, stage = stage == kAhead - 1 ? 0 : stage + 1) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 2) : "memory");
      __syncthreads();  // the step is there, and the one to be filled has been stored
      load(g + (kAhead - 1) * shares, stage == 0 ? kAhead - 1 : stage - 1);
      if (!any) continue;
      uint8_t* const step = smem + stage * M::kOutBytes;
      uint8_t* const lines = step + M::kBytesB;
      if (held) {
        // rows q4 and q4 + 8 of the 16-row operand, columns 2 t4 and 2 t4 + 1 of the other
        uint8_t* const mine = lines + (COL ? half + q4 : tok + q4) * M::kLine + ((COL ? tok : half) + 2 * t4) * 2;
        auto two = [&](int k, int h) { return reinterpret_cast<uint32_t*>(mine + (COL ? k / 2 * 16 + h * 8 : h * 8) * M::kLine + (COL ? (k & 1) * 8 : k * 8) * 2); };
        uint32_t was[4][2];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) was[k][h] = *two(k, h);
        // COL: [strip of 16 outputs][eight of tokens]; else [eight of outputs] x 16 tokens
        float acc[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[k][j] = 0.0f;
        auto piece = [&](int row, int b) {
          return *reinterpret_cast<const uint4*>(step + row * (M::kBlocks * 64) + ((M::kBlocks == 1 ? t4 : (b * 4 + t4) ^ ((row & 1) << 2)) << 4));
        };
#pragma unroll
        for (int b = 0; b < M::kBlocks; ++b) {
          uint4 w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = piece(half + k * 8 + q4, b);
#pragma unroll
          for (int p = 0; p < 2; ++p)  // the small parts first
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (COL) mma32<AT>(acc[k], w[k / 2 * 2], w[k / 2 * 2 + 1], (p ? hi : lo)[k & 1][b]);  // strip k / 2, eight of tokens k % 2
              else mma32<AT>(acc[k], (p ? hi : lo)[0][b], (p ? hi : lo)[1][b], w[k]);
            }
        }
        auto add = [&](auto type) {
          constexpr int DT = decltype(type)::value;
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float f0 = COL ? f[2 * (k & 1)] : f[2 * h], f1 = COL ? f[2 * (k & 1) + 1] : f[2 * h];
              const uint32_t b = was[k][h];
              const float b0 = a16_to_f32<DT>((uint16_t)b), b1 = DT == 0 ? a16_to_f32<0>((uint16_t)(b >> 16)) : __uint_as_float(b & 0xFFFF0000u);
              *two(k, h) = f32x2_to_a16x2<DT>(fmaf(f0, acc[k][2 * h], b0), fmaf(f1, acc[k][2 * h + 1], b1));
            }
        };
        if (a.d_type == FP8IMMA_OUT_F16) add(std::integral_constant<int, 0>());
        else add(std::integral_constant<int, 1>());
        __syncwarp();
      }
      if (!p.vec) {
        // the warp's elements, half a line's neighbours a time
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
          const int l = COL ? half + 2 * i + (lane >> 4) : tok + i, at = COL ? tok + (lane & 15) : half + lane;
          uint16_t* to;
          if (element(g, l * kTile + at, a.out, a.out_token_stride, a.out_feature_stride, to)) *to = *reinterpret_cast<const uint16_t*>(lines + l * M::kLine + at * 2);
        }
        continue;
      }
      // the warp's 16 x 32 (COL: 32 x 16) elements, 16 bytes a lane
      const int l = COL ? half + (lane >> 1) : tok + (lane >> 2), j = COL ? tok / 8 + (lane & 1) : half / 8 + (lane & 3);
      constexpr int kNext = COL ? 16 : 8;  // lines to the lane's second eight
      uint16_t* const dst = static_cast<uint16_t*>(a.out) + (int64_t)(tb + (COL ? 8 * j : l)) * a.out_token_stride +
                            (int64_t)(g * kTile + (COL ? l : 8 * j)) * a.out_feature_stride;
      const int64_t next = kNext * (COL ? a.out_feature_stride : a.out_token_stride);
      const uint8_t* const line = lines + l * M::kLine + j * 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = COL ? 8 * j : l + kNext * h, n = g * kTile + (COL ? l + kNext * h : 8 * j);
        if (whole(i, n)) *reinterpret_cast<uint4*>(dst + h * next) = *reinterpret_cast<const uint4*>(line + h * kNext * M::kLine);
        else part(i, n, [&](int k) { dst[h * next + k] = reinterpret_cast<const uint16_t*>(line + h * kNext * M::kLine)[k]; });
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the steps' places are the next unit's ring
  }
  // no CTA leaves while another may still write its sums: each has passed the last
  // barrier after those writes, so nothing is left to wait for
}

template <class Kern>
cudaError_t launch_clusters(Kern kern, const LoraParams& p, int clusters, int smem, cudaStream_t st) {
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), smem + 1024);  // static shared memory counts too
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

// Up to 128 tokens take the kernel for few, more than 1024 the one for many. Between
// them, where a decode batch as well as a prompt may lie, both are launched, and the
// ids say which of them returns at once (5 to 10 us). Measured, rank 32, 4096 -> 11008,
// column-major, 150 requests of one token: 56 to 63 us, 476 in the kernel for many alone.
// Where the mean of the runs belongs to none of them, and above 1024 tokens, short runs
// pay for a tile of 64 tokens each: one prompt of 900 tokens beside 124 requests of one
// 484 us, 1025 requests of one token 3350 (1024 of them 402, one prompt of 1024 36).
template <int AT, int STRIPS>
cudaError_t launch(LoraParams& p, cudaStream_t st) {
  const int sms = num_sms_current(), T = p.a.tokens;
  p.choose = T > 128 && T <= 1024;
  if (T <= 1024) {
    // a unit of its own for each token at most: clusters small enough to run all at
    // once, and more of them where there are few tokens, each with a block a warp or so
    using F = Few<STRIPS>;
    p.cluster = 8;
    while (p.cluster > 4 && T * p.cluster > 3 * sms) p.cluster /= 2;
    const int groups = (p.a.out_features + F::kOuts - 1) / F::kOuts;
    p.split = std::max(1, (groups + p.cluster * kWarps - 1) / (p.cluster * kWarps));
    const int clusters = std::min(3 * sms / p.cluster, std::max(T, std::min(T * p.split, sms / p.cluster)));
    const cudaError_t e = p.col ? launch_clusters(lora_few_kernel<AT, STRIPS, true>, p, clusters, F::kSmem, st)
                                : launch_clusters(lora_few_kernel<AT, STRIPS, false>, p, clusters, F::kSmem, st);
    if (e != cudaSuccess || !p.choose) return e;
  }
  // As large a cluster as lets about T / 64 units run at once, so that a unit's
  // weights cross few SMs' links.
  const int room = sms * (STRIPS >= 8 ? 95 : 190) / 100, units = (T + kTile - 1) / kTile;  // clusters leave some SMs out
  p.cluster = 8;
  while (p.cluster > 1 && units * p.cluster > room) p.cluster /= 2;
  const int groups = (p.a.out_features + kTile - 1) / kTile;
  p.split = std::max(1, groups / (2 * p.cluster));
  const int clusters = (int)std::min<int64_t>((int64_t)T * p.split, room / p.cluster);
  return p.col ? launch_clusters(lora_many_kernel<AT, STRIPS, true>, p, clusters, Many<STRIPS>::kSmem, st)
               : launch_clusters(lora_many_kernel<AT, STRIPS, false>, p, clusters, Many<STRIPS>::kSmem, st);
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
  if (a->x_stride < 0 || a->x_stride % 8 || !aligned4({a->adapter_ids, a->scales})) return (int)cudaErrorInvalidValue;
  const int64_t bt = a->base_token_stride, bf = a->base_feature_stride, ot = a->out_token_stride, of = a->out_feature_stride;
  if (bt < 0 || bf < 0 || ot < 0 || of < 0) return (int)cudaErrorInvalidValue;
  const bool row = bf == 1 && of == 1, col = !row && bt == 1 && ot == 1;
  if (!row && !col) return (int)cudaErrorInvalidValue;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a->base) | reinterpret_cast<uintptr_t>(a->out) | (uintptr_t)((row ? bt | ot : bf | of) * 2);
  if (bits & 1u) return (int)cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int64_t t = 0; t < a->tokens; t += kMaxTokens) {
    LoraParams p = {};
    p.a = *a;
    p.a.tokens = (int)std::min<int64_t>(a->tokens - t, kMaxTokens);
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
