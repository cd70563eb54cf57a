// The residual connection between two blocks with the norms on both sides of it
// (fp8imma_residual_norm). Per token, o = weight_offset:
//   b = y, or rms(y) (post + o);  r' = r + alpha gate b;  h = rms(r') (pre + o)
//   rms(x) = x / sqrt(mean x^2 + eps)
// in fp32; r' and h are rounded once, h is made from the unrounded r'.
//
// Bound: every tensor is read or written once. A row stays in registers of the
// threads that share it (up to 32 elements each) from its load to its last store,
// so the two sums over the row cost no further pass. A team of 1 .. 32 warps owns
// a row; a CTA holds as many teams as 256 threads make.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

constexpr int kCta = 256;

struct NormParams {
  fp8imma_residual_norm_args a;
  int team;  // threads of a row
};

// Eight elements as fp32: the vector form takes neighbours, the other one every
// team-th element from `at` on (loads of a warp are contiguous either way).
template <int VEC>
struct Eight {
  float v[8];
  __device__ __forceinline__ void load(const void* p, int type, int64_t row, int at, int step, int n) {
    if (VEC) {
      if (at >= n) return;
      if (type == FP8IMMA_L_F32) {
        const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + row + at);
        const float4 a = s[0], b = s[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + row + at);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = type == FP8IMMA_L_F16 ? a16_to_f32<0>((uint16_t)(w[i] & 0xFFFFu)) : __uint_as_float(w[i] << 16);
          v[2 * i + 1] = type == FP8IMMA_L_F16 ? a16_to_f32<0>((uint16_t)(w[i] >> 16)) : __uint_as_float(w[i] & 0xFFFF0000u);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = at + i * step;
        if (e >= n) continue;
        if (type == FP8IMMA_L_F32) v[i] = static_cast<const float*>(p)[row + e];
        else {
          const uint16_t b = static_cast<const uint16_t*>(p)[row + e];
          v[i] = type == FP8IMMA_L_F16 ? a16_to_f32<0>(b) : a16_to_f32<1>(b);
        }
      }
    }
  }
  __device__ __forceinline__ void store(void* p, int type, int64_t row, int at, int step, int n) const {
    if (VEC) {
      if (at >= n) return;
      if (type == FP8IMMA_L_F32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + row + at);
        d[0] = make_float4(v[0], v[1], v[2], v[3]);
        d[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = type == FP8IMMA_L_F16 ? (uint32_t)f32_to_a16<0>(v[2 * i]) | (uint32_t)f32_to_a16<0>(v[2 * i + 1]) << 16
                                       : (uint32_t)f32_to_a16<1>(v[2 * i]) | (uint32_t)f32_to_a16<1>(v[2 * i + 1]) << 16;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + row + at) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = at + i * step;
        if (e >= n) continue;
        if (type == FP8IMMA_L_F32) static_cast<float*>(p)[row + e] = v[i];
        else static_cast<uint16_t*>(p)[row + e] = type == FP8IMMA_L_F16 ? f32_to_a16<0>(v[i]) : f32_to_a16<1>(v[i]);
      }
    }
  }
};

// Sum over the row's team: every thread gets it, in one order.
__device__ __forceinline__ float team_sum(float x, float* s, int team, int warp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (team == 32) return x;
  if ((threadIdx.x & 31) == 0) s[warp] = x;
  __syncthreads();
  const int w0 = warp & ~(team / 32 - 1);
  float t = 0.0f;
  for (int w = 0; w < team / 32; ++w) t += s[w0 + w];
  return t;
}

// V: eights of a thread.
template <int VEC, int V>
__global__ void __launch_bounds__(1024) residual_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float s_sum[2][32];
  pdl_launch_dependents();
  pdl_wait();
  const fp8imma_residual_norm_args& a = p.a;
  const int warp = threadIdx.x >> 5, tid = threadIdx.x & (p.team - 1), n = a.hidden;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / p.team) + threadIdx.x / p.team;
  const int lim = row < a.tokens ? n : 0;  // teams past the last row only meet at the barriers
  // element of the v-th eight, and the step within it
  auto at = [&](int v) { return VEC ? (v * p.team + tid) * 8 : v * 8 * p.team + tid; };
  Eight<VEC> x[V], r[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[v].v[i] = r[v].v[i] = 0.0f;
    x[v].load(a.y, a.a_type, row * a.y_stride, at(v), p.team, lim);
    if (a.residual) r[v].load(a.residual, a.r_type, row * a.residual_stride, at(v), p.team, lim);
  }
  float scale = a.alpha;
  if (a.post_weight) {
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(x[v].v[i], x[v].v[i], s);
    s = team_sum(s, s_sum[0], p.team, warp);
    const float f = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(s, (float)n) + a.eps));
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Eight<VEC> w;
#pragma unroll
      for (int i = 0; i < 8; ++i) w.v[i] = 0.0f;
      w.load(a.post_weight, a.w_type, 0, at(v), p.team, lim);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[v].v[i] *= f * (w.v[i] + a.weight_offset);
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Eight<VEC> g;
#pragma unroll
    for (int i = 0; i < 8; ++i) g.v[i] = 1.0f;
    if (a.gate) g.load(a.gate, a.g_type, row * a.gate_stride, at(v), p.team, lim);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r[v].v[i] = fmaf(scale, g.v[i] * x[v].v[i], r[v].v[i]);
      s = fmaf(r[v].v[i], r[v].v[i], s);
    }
    if (a.residual_out) r[v].store(a.residual_out, a.r_type, row * n, at(v), p.team, lim);
  }
  if (!a.pre_weight) return;
  s = team_sum(s, s_sum[1], p.team, warp);
  const float f = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(s, (float)n) + a.eps));
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Eight<VEC> w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w.v[i] = 0.0f;
    w.load(a.pre_weight, a.w_type, 0, at(v), p.team, lim);
#pragma unroll
    for (int i = 0; i < 8; ++i) w.v[i] = r[v].v[i] * f * (w.v[i] + a.weight_offset);
    w.store(a.out, a.a_type, row * n, at(v), p.team, lim);
  }
}

template <int VEC, int V>
cudaError_t launch(const NormParams& p, cudaStream_t st) {
  const int cta = std::max(p.team, kCta);
  const int64_t rows = cta / p.team;
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.gridDim = dim3((unsigned)((p.a.tokens + rows - 1) / rows));
  lc.blockDim = dim3(cta);
  lc.stream = st;
  lc.attrs = attr;
  lc.numAttrs = api_pdl() ? 1 : 0;
  return cudaLaunchKernelEx(&lc, residual_norm_kernel<VEC, V>, p);
}

}  // namespace
}  // namespace fp8imma_b200

using namespace fp8imma_b200;

extern "C" int fp8imma_residual_norm(const fp8imma_residual_norm_args* a, void* stream) {
  FP8IMMA_RANGE("fp8imma_residual_norm");
  if (!a) return (int)cudaErrorInvalidValue;
  if (a->tokens <= 0 || a->hidden <= 0) return (int)cudaErrorInvalidConfiguration;
  if (a->hidden > FP8IMMA_NORM_MAX_HIDDEN || a->a_type < 0 || a->a_type > 1 || a->r_type < 0 || a->r_type > 2 || a->w_type < 0 || a->w_type > 2 ||
      a->g_type < 0 || a->g_type > 2 || a->y_stride < 0 || a->residual_stride < 0 || a->gate_stride < 0)
    return (int)cudaErrorInvalidValue;
  if (!a->y || (!a->residual_out && !a->pre_weight) || (a->pre_weight != nullptr) != (a->out != nullptr)) return (int)cudaErrorInvalidValue;
  if (!(a->eps >= 0.0f && a->eps < 3.4e38f)) return (int)cudaErrorInvalidValue;
  // addresses and strides in bytes of each tensor: a whole number of elements, and of 16 bytes for the vector form
  auto bits = [](const void* q, int64_t stride, int type) {
    return q ? reinterpret_cast<uintptr_t>(q) | (uintptr_t)(stride * (type == FP8IMMA_L_F32 ? 4 : 2)) : (uintptr_t)0;
  };
  const uintptr_t res = bits(a->residual, a->residual_stride, a->r_type) | bits(a->residual_out, a->hidden, a->r_type);
  const uintptr_t w = bits(a->post_weight, 0, a->w_type) | bits(a->pre_weight, 0, a->w_type), g = bits(a->gate, a->gate_stride, a->g_type);
  const uintptr_t all = bits(a->y, a->y_stride, a->a_type) | bits(a->out, a->hidden, a->a_type) | res | w | g;
  if (all & 1u) return (int)cudaErrorInvalidValue;
  if ((a->r_type == FP8IMMA_L_F32 && (res & 3u)) || (a->w_type == FP8IMMA_L_F32 && (w & 3u)) || (a->g_type == FP8IMMA_L_F32 && (g & 3u)))
    return (int)cudaErrorInvalidValue;
  const bool vec = (all & 15u) == 0 && a->hidden % 8 == 0;
  NormParams p = {};
  p.a = *a;
  // A thread takes one eight while that fills 256 threads at most, then two, so
  // that small rows meet few warps at a barrier and large ones fit in 1024 threads.
  const int eights = (a->hidden + 7) / 8;
  const int v = eights <= 256 ? 1 : eights <= 2048 ? 2 : 4;
  p.team = 32;
  while (p.team * v < eights) p.team *= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (vec) return (int)(v == 1 ? launch<1, 1>(p, st) : v == 2 ? launch<1, 2>(p, st) : launch<1, 4>(p, st));
  return (int)(v == 1 ? launch<0, 1>(p, st) : v == 2 ? launch<0, 2>(p, st) : launch<0, 4>(p, st));
}
