// Attention of a step's queries over the paged 8-bit KV cache
// (fp8imma_kv_attention).
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"

#include <cuda_runtime.h>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

struct AttnParams {
  fp8imma_kv_cache c;
  fp8imma_kv_attention_args a;
  int per_seq;
};

constexpr int kWarps = 4;

// One CTA per (token, query head): each warp takes every fourth key, a lane
// D / 32 channels of it, with a running maximum and sum.
template <int AT, int FMT, int D>
__global__ void __launch_bounds__(kWarps * 32) kv_attention_kernel(const __grid_constant__ AttnParams p) {
  constexpr int E = D / 32;
  __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][D];
  const int t = blockIdx.x, h = blockIdx.y, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int b, t0, n;
  if (p.per_seq > 0) {
    b = t / p.per_seq;
    t0 = b * p.per_seq;
    n = p.per_seq;
  } else {
    int lo = 0, hi = p.c.batch - 1;  // last b with cu_new[b] <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(p.c.cu_new + mid) <= t) lo = mid; else hi = mid - 1;
    }
    b = lo;
    t0 = __ldg(p.c.cu_new + b);
    n = __ldg(p.c.cu_new + b + 1) - t0;
  }
  const int hk = h / (p.a.heads / p.c.kv_heads);
  const int len = min(__ldg(p.c.seq_lens + b), p.c.max_pages * p.c.page_size);
  const int pos = __ldg(p.c.seq_lens + b) - n + (t - t0);
  const int j0 = p.a.window > 0 ? max(0, pos - p.a.window + 1) : 0, j1 = min(pos + 1, len);
  float q[E];
  const uint16_t* qp = static_cast<const uint16_t*>(p.a.q) + (int64_t)t * p.a.q_token_stride + (int64_t)h * p.a.q_head_stride + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) q[i] = a16_to_f32<AT>(qp[i]) * p.a.softmax_scale;
  float m = -INFINITY, l = 0.0f, o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.0f;
  for (int j = j0 + w; j < j1; j += kWarps) {
    const int page = __ldg(p.c.page_table + (size_t)b * p.c.max_pages + j / p.c.page_size);
    if ((unsigned)page >= (unsigned)p.c.num_pages) continue;
    const size_t ph = (size_t)page * p.c.kv_heads + hk;
    const size_t at = (ph * p.c.page_size + j % p.c.page_size) * D + lane * E;
    const uint8_t* kp = static_cast<const uint8_t*>(p.c.k) + at;
    const uint8_t* vp = static_cast<const uint8_t*>(p.c.v) + at;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += q[i] * f8_to_f32<FMT>(kp[i]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= p.c.k_scale[ph];
    const float mn = fmaxf(m, s), keep = m == mn ? 1.0f : __expf(m - mn), e = __expf(s - mn);
    l = l * keep + e;
    const float ev = e * p.c.v_scale[ph];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = o[i] * keep + ev * f8_to_f32<FMT>(vp[i]);
    m = mn;
  }
  if (lane == 0) {
    s_m[w] = m;
    s_l[w] = l;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) s_o[w][lane * E + i] = o[i];
  __syncthreads();
  float mm = -INFINITY, ll = 0.0f;
  for (int i = 0; i < kWarps; ++i) mm = fmaxf(mm, s_m[i]);
  float f[kWarps];
  for (int i = 0; i < kWarps; ++i) {
    f[i] = s_m[i] == -INFINITY ? 0.0f : __expf(s_m[i] - mm);
    ll += f[i] * s_l[i];
  }
  uint16_t* op = static_cast<uint16_t*>(p.a.out) + ((int64_t)t * p.a.heads + h) * D;
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float v = 0.0f;
    for (int i = 0; i < kWarps; ++i) v += f[i] * s_o[i][d];
    op[d] = f32_to_a16<AT>(ll == 0.0f ? 0.0f : v / ll);
  }
  if (p.a.lse && threadIdx.x == 0) p.a.lse[(int64_t)t * p.a.heads + h] = ll == 0.0f ? -INFINITY : mm + logf(ll);
}

template <int AT, int FMT>
cudaError_t launch_d(const AttnParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)p.c.tokens, (unsigned)p.a.heads);
  if (p.c.head_dim == 64) kv_attention_kernel<AT, FMT, 64><<<grid, kWarps * 32, 0, st>>>(p);
  else if (p.c.head_dim == 128) kv_attention_kernel<AT, FMT, 128><<<grid, kWarps * 32, 0, st>>>(p);
  else kv_attention_kernel<AT, FMT, 256><<<grid, kWarps * 32, 0, st>>>(p);
  return cudaGetLastError();
}
template <int AT>
cudaError_t launch_f(const AttnParams& p, cudaStream_t st) {
  return p.c.format == FP8IMMA_B_E4M3 ? launch_d<AT, F8_E4M3>(p, st) : launch_d<AT, F8_E5M2>(p, st);
}

}  // namespace
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
  AttnParams p = {};
  p.c = *c;
  p.a = *a;
  p.per_seq = c->cu_new ? 0 : c->tokens / c->batch;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return (int)(a->a_type == FP8IMMA_A_F16 ? launch_f<0>(p, st) : launch_f<1>(p, st));
}
