// Mixture-of-experts layer with FP8 weights for a few tokens
// (fp8imma_moe_forward).
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <cuda_runtime.h>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float gate_act(float v, int act) {
  if (act == 3) return v / (1.0f + __expf(-v));
  return 0.5f * v * (1.0f + tanhf(0.7978845608028654f * (v + 0.044715f * v * v * v)));
}

// one warp per (token, expert)
template <int AT>
__global__ void moe_router_kernel(fp8imma_moe_args a, float* logits) {
  const int e = blockIdx.x * 4 + (threadIdx.x >> 5), t = blockIdx.y, lane = threadIdx.x & 31;
  if (e >= a.experts) return;
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + t * a.x_token_stride;
  const uint16_t* w = static_cast<const uint16_t*>(a.router) + (size_t)e * a.hidden;
  float s = 0.0f;
  for (int i = lane; i < a.hidden; i += 32) s += a16_to_f32<AT>(x[i]) * a16_to_f32<AT>(w[i]);
  s = warp_sum(s);
  if (lane == 0) logits[(size_t)t * a.experts + e] = s;
}

// one warp per token: k rounds of the largest not yet taken
__global__ void moe_topk_kernel(fp8imma_moe_args a, const float* logits, int* ids, float* wts) {
  const int t = blockIdx.x, lane = threadIdx.x;
  const float* r = logits + (size_t)t * a.experts;
  unsigned taken = 0;  // expert lane + 32 * bit
  float first = 0.0f, sum = 0.0f;
  for (int s = 0; s < a.top_k; ++s) {
    long long best = -0x7fffffffffffffffll;
    for (int i = 0; lane + 32 * i < a.experts; ++i) {
      if (taken >> i & 1) continue;
      const float v = r[lane + 32 * i];
      int key = __float_as_int(v);
      key = isnan(v) ? 0x7fffffff : (key < 0 ? (int)(0x80000000u - (unsigned)key) : key);
      best = max(best, ((long long)key << 32) - (lane + 32 * i));
    }
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    const int e = (int)(-(best & 0xffffffffll) & 0x7ff);
    if ((e & 31) == lane) taken |= 1u << (e >> 5);
    const float v = r[e];
    if (s == 0) first = v;
    sum += __expf(v - first);
    if (lane == 0) {
      ids[t * a.top_k + s] = e;
      wts[t * a.top_k + s] = __expf(v - first);
    }
  }
  if (!a.renormalize) {
    sum = 0.0f;
    for (int i = lane; i < a.experts; i += 32) sum += __expf(r[i] - first);
    sum = warp_sum(sum);
  }
  __syncwarp();
  for (int s = lane; s < a.top_k; s += 32) {
    const float p = wts[t * a.top_k + s] / sum;
    wts[t * a.top_k + s] = p;
    if (a.ids) a.ids[t * a.top_k + s] = ids[t * a.top_k + s];
    if (a.weights) a.weights[t * a.top_k + s] = p;
  }
}

// one warp per (slot, inner channel)
template <int AT, int FMT>
__global__ void moe_up_kernel(fp8imma_moe_args a, const int* ids, float* hbuf) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), slot = blockIdx.y, lane = threadIdx.x & 31;
  if (i >= a.inter) return;
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + (slot / a.top_k) * a.x_token_stride;
  const int e = ids[slot];
  const uint8_t* w = static_cast<const uint8_t*>(a.w_gate_up) + ((size_t)e * 2 * a.inter + i) * a.hidden;
  float g = 0.0f, u = 0.0f;
  for (int k = lane; k < a.hidden; k += 32) {
    const float v = a16_to_f32<AT>(x[k]);
    g += v * f8_to_f32<FMT>(w[k]);
    u += v * f8_to_f32<FMT>(w[(size_t)a.inter * a.hidden + k]);
  }
  g = warp_sum(g) * a.s_gate_up[(size_t)e * 2 * a.inter + i];
  u = warp_sum(u) * a.s_gate_up[(size_t)e * 2 * a.inter + a.inter + i];
  if (lane == 0) hbuf[(size_t)slot * a.inter + i] = gate_act(g, a.act) * u;
}

// one warp per (token, output channel)
template <int AT, int FMT>
__global__ void moe_down_kernel(fp8imma_moe_args a, const int* ids, const float* wts, const float* hbuf) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), t = blockIdx.y, lane = threadIdx.x & 31;
  if (i >= a.hidden) return;
  float y = 0.0f;
  for (int s = 0; s < a.top_k; ++s) {
    const int slot = t * a.top_k + s, e = ids[slot];
    const uint8_t* w = static_cast<const uint8_t*>(a.w_down) + ((size_t)e * a.hidden + i) * a.inter;
    float d = 0.0f;
    for (int k = lane; k < a.inter; k += 32) d += hbuf[(size_t)slot * a.inter + k] * f8_to_f32<FMT>(w[k]);
    y += wts[slot] * (warp_sum(d) * a.s_down[(size_t)e * a.hidden + i]);
  }
  if (lane == 0) static_cast<uint16_t*>(a.out)[(size_t)t * a.hidden + i] = f32_to_a16<AT>(y);
}

template <int AT, int FMT>
cudaError_t run_moe(const fp8imma_moe_args& a, cudaStream_t st) {
  const size_t slots = (size_t)a.tokens * a.top_k;
  ScopedScratch sc;
  cudaError_t e = sc.get((size_t)a.tokens * a.experts * 4 + slots * 8 + slots * a.inter * 4, st, kScratchMoe);
  if (e != cudaSuccess) return e;
  float* logits = static_cast<float*>(sc.ptr);
  int* ids = reinterpret_cast<int*>(logits + (size_t)a.tokens * a.experts);
  float* wts = reinterpret_cast<float*>(ids + slots);
  float* hbuf = wts + slots;
  moe_router_kernel<AT><<<dim3((a.experts + 3) / 4, a.tokens), 128, 0, st>>>(a, logits);
  moe_topk_kernel<<<a.tokens, 32, 0, st>>>(a, logits, ids, wts);
  moe_up_kernel<AT, FMT><<<dim3((a.inter + 3) / 4, (unsigned)slots), 128, 0, st>>>(a, ids, hbuf);
  moe_down_kernel<AT, FMT><<<dim3((a.hidden + 3) / 4, a.tokens), 128, 0, st>>>(a, ids, wts, hbuf);
  e = cudaGetLastError();
  const cudaError_t e2 = sc.release(st);
  return e != cudaSuccess ? e : e2;
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
  if ((reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->router) | reinterpret_cast<uintptr_t>(a->out)) & 1u)
    return (int)cudaErrorInvalidValue;
  // weight rows are indexed with 31 bits
  if ((int64_t)a->experts * 2 * a->inter > 0x7fffffffll || (int64_t)a->experts * a->hidden > 0x7fffffffll)
    return (int)cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->a_type == FP8IMMA_A_F16)
    return (int)(a->format == FP8IMMA_B_E4M3 ? run_moe<0, F8_E4M3>(*a, st) : run_moe<0, F8_E5M2>(*a, st));
  return (int)(a->format == FP8IMMA_B_E4M3 ? run_moe<1, F8_E4M3>(*a, st) : run_moe<1, F8_E5M2>(*a, st));
}
