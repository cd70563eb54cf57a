// What the appends to the paged 8-bit cache share (kv_cache.cu, kv_rope.cu):
// rows as 16-byte pieces, a page's scale, codes.
#pragma once

#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "sm100_async.cuh"

namespace fp8imma_b200 {
namespace kv {

using namespace fp8imma_dev;

template <int AT>
__device__ __forceinline__ uint4 load_row8(const uint16_t* p, bool vec) {
  if (vec) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldg(p + 2 * i) | ((uint32_t)__ldg(p + 2 * i + 1) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int AT>
__device__ __forceinline__ float absmax8(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = fabsf(a16_to_f32<AT>((uint16_t)(w[i] & 0xFFFFu))), b = fabsf(a16_to_f32<AT>((uint16_t)(w[i] >> 16)));
    m = fmaxf(m, a < INFINITY ? a : 0.0f);
    m = fmaxf(m, b < INFINITY ? b : 0.0f);
  }
  return m;
}

template <int AT, int FMT>
__device__ __forceinline__ uint2 to_codes(uint4 v, float s, float inv) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  // a page's scale that the caller set to something else than a power of two takes the division
  const bool pow2 = (__float_as_uint(s) & 0x7FFFFFu) == 0u;
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = a16_to_f32<AT>((uint16_t)(w[i] & 0xFFFFu)), b = a16_to_f32<AT>((uint16_t)(w[i] >> 16));
    o[i] = pow2 ? f32x2_to_f8x2<FMT>(a * inv, b * inv) : f32x2_to_f8x2<FMT>(__fdiv_rn(a, s), __fdiv_rn(b, s));
  }
  return make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
}

// The smallest power of two, 2^-126 at least, that brings amax within the format's range:
// amax = 1.m * 2^e <= 1.75 * 2^(8|15) * 2^k  <=>  k >= e - (8|15), one more when 1.m > 1.75
template <int FMT>
__device__ __forceinline__ float needed_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - (FMT == F8_E4M3 ? 8 : 15) + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

// 16 codes under a scale larger by 1 / ratio
template <int FMT>
__device__ __forceinline__ uint4 moved_codes(uint4 c, float ratio) {
  uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a, bb;
    f8x4_to_f16x4<FMT>(w[i], a, bb);
    const float2 fa = __half22float2(*reinterpret_cast<__half2*>(&a)), fb = __half22float2(*reinterpret_cast<__half2*>(&bb));
    w[i] = (uint32_t)f32x2_to_f8x2<FMT>(fa.x * ratio, fa.y * ratio) | ((uint32_t)f32x2_to_f8x2<FMT>(fb.x * ratio, fb.y * ratio) << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// sequence b's packed token range, clamped to the packed axis
__device__ __forceinline__ void token_range(const fp8imma_kv_cache& c, int per_seq, int b, int& t0, int& n) {
  if (per_seq > 0) {
    t0 = b * per_seq;
    n = per_seq;
  } else {
    t0 = max(0, __ldg(c.cu_new + b));
    n = max(0, min(__ldg(c.cu_new + b + 1), c.tokens) - t0);
  }
}

// The page that CTA blockIdx.x works on: sequence b, and the pi-th of the pages
// that its new tokens touch, the first of them being `first`. count(b, first)
// gives their number. False: none, or offsets that do not ascend (the error word
// is set). All threads of the CTA take part.
template <int THREADS, class Count>
__device__ __forceinline__ bool find_page(const fp8imma_kv_cache& c, int per_seq, int pages_seq, Count count, int& b, int& first, int& pi) {
  constexpr int kWarps = THREADS / 32;
  __shared__ int s_pick[3];
  __shared__ int s_scan[2][kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (per_seq > 0) {
    b = blockIdx.x / pages_seq;
    pi = blockIdx.x % pages_seq;
    return pi < count(b, first);
  }
  // unit blockIdx.x of the sequences' touched pages laid end to end
  if (threadIdx.x == 0) s_pick[0] = -1;
  int base = 0, turn = 0;
  bool bad = false;
  for (int b0 = 0; b0 < c.batch; b0 += THREADS) {
    const int mine = b0 + (int)threadIdx.x;
    int f = 0;
    const int n = mine < c.batch ? max(0, count(mine, f)) : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_scan[turn][warp] = x;
    // Offsets that do not ascend would give a token to two sequences. Every CTA
    // looks at all of them first, so that none of them stores anything.
    if (b0 == 0)
      for (int i = mine; i < c.batch; i += THREADS) bad |= __ldg(c.cu_new + i + 1) < __ldg(c.cu_new + i);
    if (__syncthreads_or(bad)) {
      if (threadIdx.x == 0) atomicCAS(&g_fp8imma_device_error, 0u, (unsigned int)ERR_BAD_OFFSETS);
      return false;
    }
    int before = base;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_scan[turn][w];
      base += s_scan[turn][w];
    }
    turn ^= 1;  // the other one has been read by all: they have met since
    const int lo = before + x - n;
    if ((int)blockIdx.x >= lo && (int)blockIdx.x < lo + n) {
      s_pick[0] = mine;
      s_pick[1] = f;
      s_pick[2] = (int)blockIdx.x - lo;
    }
    if ((int)blockIdx.x < base) break;
  }
  __syncthreads();
  b = s_pick[0];
  if (b < 0) return false;
  first = s_pick[1];
  pi = s_pick[2];
  return true;
}

}  // namespace kv
}  // namespace fp8imma_b200
