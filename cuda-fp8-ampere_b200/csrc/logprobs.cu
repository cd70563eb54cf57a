// Log probabilities of given tokens, entropy and top alternatives of logits
// (fp8imma_token_logprobs).
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"

#include <cuda_runtime.h>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

constexpr int kThreads = 256;

template <int LT>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  if (LT == FP8IMMA_L_F32) return static_cast<const float*>(p)[i];
  return a16_to_f32<LT>(static_cast<const uint16_t*>(p)[i]);
}

// order-preserving integer of a logit: -0 = +0, NaN above everything
__device__ __forceinline__ int order_key(float v) {
  const int k = __float_as_int(v);
  if (isnan(v)) return 0x7fffffff;
  return k < 0 ? (int)(0x80000000u - (unsigned)k) : k;
}

template <class T, class F>
__device__ __forceinline__ T block_reduce(T v, T* red, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < kThreads / 32; ++i) v = f(v, red[i]);
  return v;
}

// one CTA per row, several passes
template <int LT>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(fp8imma_logprobs_args a) {
  __shared__ float redf[kThreads / 32];
  __shared__ long long redl[kThreads / 32];
  const int t = blockIdx.x;
  const int64_t base = (int64_t)t * a.token_stride;
  const float it = 1.0f / a.temperature;
  auto z = [&](int j) { return load_logit<LT>(a.logits, base + (int64_t)j * a.vocab_stride) * it; };
  float m = -INFINITY;
  bool nan = false;
  for (int j = threadIdx.x; j < a.vocab; j += kThreads) {
    const float v = z(j);
    nan |= isnan(v);
    m = fmaxf(m, v);
  }
  m = block_reduce(m, redf, [](float x, float y) { return fmaxf(x, y); });
  nan = __syncthreads_or(nan);
  float l = 0.0f, s = 0.0f;
  for (int j = threadIdx.x; j < a.vocab; j += kThreads) {
    const float d = z(j) - m, e = expf(d);
    l += e;
    if (d > -INFINITY) s += e * d;
  }
  l = block_reduce(l, redf, [](float x, float y) { return x + y; });
  s = block_reduce(s, redf, [](float x, float y) { return x + y; });
  const bool bad = nan || !(fabsf(m) < INFINITY);
  const float lse = bad ? NAN : m + logf(l);
  if (threadIdx.x == 0) {
    const int id = a.token_ids[t];
    a.logprobs[t] = (unsigned)id < (unsigned)a.vocab ? z(id) - lse : NAN;
    a.entropy[t] = bad ? NAN : logf(l) - s / l;
  }
  long long last = 0x7fffffffffffffffll;
  for (int k = 0; k < a.top; ++k) {
    long long best = -0x7fffffffffffffffll - 1;
    for (int j = threadIdx.x; j < a.vocab; j += kThreads) {
      const long long key = ((long long)order_key(load_logit<LT>(a.logits, base + (int64_t)j * a.vocab_stride)) << 32) - j;
      if (key < last && key > best) best = key;
    }
    best = block_reduce(best, redl, [](long long x, long long y) { return x > y ? x : y; });
    last = best;
    const int id = (int)(-(best & 0xffffffffll) & 0x7fffffff);
    if (threadIdx.x == 0) {
      a.top_ids[(int64_t)t * a.top + k] = id;
      a.top_logprobs[(int64_t)t * a.top + k] = z(id) - lse;
    }
  }
}

}  // namespace
}  // namespace fp8imma_b200

using namespace fp8imma_b200;

extern "C" int fp8imma_token_logprobs(const fp8imma_logprobs_args* a, void* stream) {
  FP8IMMA_RANGE("fp8imma_token_logprobs");
  if (!a) return (int)cudaErrorInvalidValue;
  if (a->tokens <= 0 || a->vocab <= 0) return (int)cudaErrorInvalidConfiguration;
  if (!a->logits || !a->token_ids || !a->logprobs || !a->entropy) return (int)cudaErrorInvalidValue;
  if (a->top < 0 || a->top > FP8IMMA_LOGPROBS_MAX_TOP || a->top > a->vocab) return (int)cudaErrorInvalidValue;
  if (a->top > 0 && (!a->top_ids || !a->top_logprobs)) return (int)cudaErrorInvalidValue;
  if (a->l_type < 0 || a->l_type > 2 || !(a->temperature > 0.0f) || !(a->temperature < INFINITY))
    return (int)cudaErrorInvalidValue;
  if (a->vocab_stride != 1 && a->token_stride != 1) return (int)cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(a->logits) & (a->l_type == FP8IMMA_L_F32 ? 3u : 1u)) return (int)cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->l_type == FP8IMMA_L_F16) logprobs_kernel<FP8IMMA_L_F16><<<a->tokens, kThreads, 0, st>>>(*a);
  else if (a->l_type == FP8IMMA_L_BF16) logprobs_kernel<FP8IMMA_L_BF16><<<a->tokens, kThreads, 0, st>>>(*a);
  else logprobs_kernel<FP8IMMA_L_F32><<<a->tokens, kThreads, 0, st>>>(*a);
  return (int)cudaGetLastError();
}
