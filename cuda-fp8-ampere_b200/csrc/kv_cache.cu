// Appending key and value rows to the paged 8-bit KV cache (fp8imma_kv_append).
//
// Per page and KV head, over the new rows x of the page:
//   need = 2^e, the smallest power of two >= 2^-126 with absmax_finite(x) <= fmax * 2^e
//   s'   = max(s, need) when the page holds earlier tokens, else need
//   earlier codes c -> rne(c * (s / s')), only when s' > s;  new codes = rne_sat(x / s')
// An FP8 code carries its own exponent, so a scale finer than a power of two
// would not make the codes more precise, and with powers of two a growing
// scale only shifts exponents: codes move exactly until they drop below the
// format's smallest step. Division by s' is an exact product as well, so each
// stored value is rounded once.
//
// A team of 1 .. 8 warps owns one (page, head, K or V), so scales and codes of
// a page have one writer and no atomics are needed. A CTA's teams share a page:
// finding it (a scan of the sequences' lengths) is what a small append spends
// its time on. Rows stay in registers between the pass for the scale and the one
// for the codes, as far as kKeep pieces a thread go.
//
// Measured: 64 sequences of one token, 8 heads of 128: 4.8 us (6.0 with a page
// lookup a warp), a chain of latencies: lengths, page id, row and scale, store.
// Prompts of 9200 tokens, rows from HBM: 22.6 us, 2.5 TB/s of the 57 MB read and
// written (24.6 with two CTAs a SM, 39 us with a page lookup a warp as well); the
// look at all offsets is 0.8 of them.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>
#include <cuda_runtime.h>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kKeep = 8;  // 16-byte vectors of a page that a thread keeps between the two passes

struct AppendParams {
  fp8imma_kv_cache c;
  const uint16_t* src[2];
  int64_t ts[2], hs[2];
  int vec;         // rows are 16-byte aligned
  int per_seq;     // > 0: every sequence appends this many tokens
  int pages_seq;   // then: pages a sequence can touch
  int team;        // warps of a (page, head, K or V)
};

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

// sequence b's packed token range, clamped to the packed axis
__device__ __forceinline__ void token_range(const AppendParams& p, int b, int& t0, int& n) {
  if (p.per_seq > 0) {
    t0 = b * p.per_seq;
    n = p.per_seq;
  } else {
    t0 = max(0, __ldg(p.c.cu_new + b));
    n = max(0, min(__ldg(p.c.cu_new + b + 1), p.c.tokens) - t0);
  }
}

// pages that sequence b's new tokens touch: first page index and count
__device__ __forceinline__ int touched(const AppendParams& p, int b, int& first) {
  int t0, n;
  token_range(p, b, t0, n);
  const int len = __ldg(p.c.seq_lens + b), start = max(0, len - n);
  first = start / p.c.page_size;
  return (n > 0 && len > start) ? min((len - 1) / p.c.page_size, p.c.max_pages - 1) - first + 1 : 0;
}

template <int AT, int FMT, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS) kv_append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ int s_pick[3];
  __shared__ int s_scan[2][kWarps];
  __shared__ float s_max[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  int b = 0, first = 0, pi = 0;
  if (p.per_seq > 0) {
    b = blockIdx.x / p.pages_seq;
    pi = blockIdx.x % p.pages_seq;
    if (pi >= touched(p, b, first)) return;
  } else {
    // unit blockIdx.x of the sequences' touched pages laid end to end
    if (threadIdx.x == 0) s_pick[0] = -1;
    int base = 0, turn = 0;
    bool bad = false;
    for (int b0 = 0; b0 < p.c.batch; b0 += kThreads) {
      const int mine = b0 + (int)threadIdx.x;
      int f = 0;
      const int n = mine < p.c.batch ? max(0, touched(p, mine, f)) : 0;
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
        for (int i = mine; i < p.c.batch; i += kThreads) bad |= __ldg(p.c.cu_new + i + 1) < __ldg(p.c.cu_new + i);
      if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) atomicCAS(&g_fp8imma_device_error, 0u, (unsigned int)ERR_BAD_OFFSETS);
        return;
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
    if (b < 0) return;
    first = s_pick[1];
    pi = s_pick[2];
  }
  const int ps = p.c.page_size, D = p.c.head_dim;
  pi += first;
  if (pi >= p.c.max_pages) return;
  const int page = __ldg(p.c.page_table + (size_t)b * p.c.max_pages + pi);
  if ((unsigned)page >= (unsigned)p.c.num_pages) return;
  int t0, n;
  token_range(p, b, t0, n);
  const int len = __ldg(p.c.seq_lens + b);
  const int start = len - n;  // position of token t0 (may be negative: those tokens have no place)
  const int lo = max(max(start, 0), pi * ps), hi = min(len, (pi + 1) * ps);
  const int slot0 = lo - pi * ps, rows = hi - lo;
  if (rows <= 0) return;
  // this team's head and tensor; teams past the last one only take part in the barrier
  const int item = blockIdx.y * (kWarps / p.team) + warp / p.team;
  const bool on = item < 2 * p.c.kv_heads;
  const int h = item >> 1, which = item & 1;
  const int tid = warp % p.team * 32 + lane, step = p.team * 32;
  const uint16_t* src = p.src[which] + (int64_t)(t0 + lo - start) * p.ts[which] + (int64_t)h * p.hs[which];
  const size_t ph = (size_t)page * p.c.kv_heads + h;
  uint8_t* dst = static_cast<uint8_t*>(which ? p.c.v : p.c.k) + ph * ps * D;
  float* scale = (which ? p.c.v_scale : p.c.k_scale) + ph;
  const float s_old = on && slot0 > 0 ? *scale : 0.0f;

  const int vr = __ffs(D) - 4, nv = on ? rows << vr : 0;  // 8-element vectors of a row (log2), of the page's new rows
  auto vec_at = [&](int v) { return src + (int64_t)(v >> vr) * p.ts[which] + (v & ((1 << vr) - 1)) * 8; };
  uint4 keep[kKeep];
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int v = tid + i * step;
    if (v < nv) keep[i] = load_row8<AT>(vec_at(v), p.vec);
  }
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (tid + i * step < nv) amax = fmaxf(amax, absmax8<AT>(keep[i]));
  for (int v = tid + kKeep * step; v < nv; v += step)
    amax = fmaxf(amax, absmax8<AT>(load_row8<AT>(vec_at(v), p.vec)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (lane == 0) s_max[warp] = amax;
  __syncthreads();
  if (!on) return;
  for (int w = 0; w < p.team; ++w) amax = fmaxf(amax, s_max[warp / p.team * p.team + w]);

  // amax = 1.m * 2^e <= 1.75 * 2^(8|15) * 2^k  <=>  k >= e - (8|15), one more when 1.m > 1.75
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - (FMT == F8_E4M3 ? 8 : 15) + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  const float need = __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
  const float s_new = fmaxf(s_old, need);
  const float inv = __fdiv_rn(1.0f, s_new);
  if (slot0 > 0 && s_new != s_old) {  // uniform: the page's earlier codes move to the larger scale
    const float ratio = __fdiv_rn(s_old, s_new);
    for (int v = tid; v < slot0 * (D >> 4); v += step) {
      uint4 c = reinterpret_cast<uint4*>(dst)[v];
      uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a, bb;
        f8x4_to_f16x4<FMT>(w[i], a, bb);
        const float2 fa = __half22float2(*reinterpret_cast<__half2*>(&a)), fb = __half22float2(*reinterpret_cast<__half2*>(&bb));
        w[i] = (uint32_t)f32x2_to_f8x2<FMT>(fa.x * ratio, fa.y * ratio) |
               ((uint32_t)f32x2_to_f8x2<FMT>(fb.x * ratio, fb.y * ratio) << 16);
      }
      reinterpret_cast<uint4*>(dst)[v] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  uint2* out = reinterpret_cast<uint2*>(dst + (size_t)slot0 * D);
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int v = tid + i * step;
    if (v < nv) out[v] = to_codes<AT, FMT>(keep[i], s_new, inv);
  }
  for (int v = tid + kKeep * step; v < nv; v += step)
    out[v] = to_codes<AT, FMT>(load_row8<AT>(vec_at(v), p.vec), s_new, inv);
  if (tid == 0) *scale = s_new;
}

// CTAS: CTAs a SM that registers have to leave room for. Two (86 registers) have
// all loads of a page in flight at once; more than two a SM at hand, and four
// take the waves faster. Measured with 1 and 4 in the bounds: 16 prompts of 200
// tokens, 4 heads of 64, 6.2 / 8.2 us; 64 single tokens, 8 heads of 128, 3.9 /
// 5.1; 256 single tokens 7.7 / 6.1; 6 prompts of 1536 tokens 24.3 / 18.0.
template <int AT, int CTAS>
cudaError_t launch_append(const AppendParams& p, dim3 grid, cudaStream_t st) {
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.gridDim = grid;
  lc.blockDim = dim3(kThreads);
  lc.stream = st;
  lc.attrs = attr;
  lc.numAttrs = api_pdl() ? 1 : 0;
  return p.c.format == FP8IMMA_B_E4M3 ? cudaLaunchKernelEx(&lc, kv_append_kernel<AT, F8_E4M3, CTAS>, p)
                                      : cudaLaunchKernelEx(&lc, kv_append_kernel<AT, F8_E5M2, CTAS>, p);
}

}  // namespace

unsigned int kv_append_device_error(bool clear) { return fp8imma_dev::tu_device_error(clear); }

cudaError_t kv_cache_check(const fp8imma_kv_cache* c) {
  if (!c) return cudaErrorInvalidValue;
  if (c->tokens <= 0 || c->batch <= 0 || c->num_pages <= 0 || c->max_pages <= 0 || c->kv_heads <= 0)
    return cudaErrorInvalidConfiguration;
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->page_table || !c->seq_lens) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u) return cudaErrorInvalidValue;
  if (c->format < 0 || c->format > 1) return cudaErrorInvalidValue;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return cudaErrorInvalidValue;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return cudaErrorInvalidValue;
  if (!c->cu_new && c->tokens % c->batch) return cudaErrorInvalidValue;
  // row indexes of the cache stay within 31 bits
  if ((int64_t)c->num_pages * c->kv_heads * c->page_size > 0x7fffffffll) return cudaErrorInvalidValue;
  if ((int64_t)c->max_pages * c->page_size > 0x7fffffffll) return cudaErrorInvalidValue;
  return cudaSuccess;
}

}  // namespace fp8imma_b200

using namespace fp8imma_b200;

extern "C" int fp8imma_kv_append(const fp8imma_kv_cache* c, const fp8imma_kv_append_args* a, void* stream) {
  FP8IMMA_RANGE("fp8imma_kv_append");
  const cudaError_t e = kv_cache_check(c);
  if (e != cudaSuccess) return (int)e;
  if (!a || !a->k || !a->v || a->a_type < 0 || a->a_type > 1) return (int)cudaErrorInvalidValue;
  AppendParams p = {};
  p.c = *c;
  p.src[0] = static_cast<const uint16_t*>(a->k);
  p.src[1] = static_cast<const uint16_t*>(a->v);
  p.ts[0] = a->k_token_stride;
  p.hs[0] = a->k_head_stride;
  p.ts[1] = a->v_token_stride;
  p.hs[1] = a->v_head_stride;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
                         (uintptr_t)((p.ts[0] | p.hs[0] | p.ts[1] | p.hs[1]) * 2);
  if (bits & 1u) return (int)cudaErrorInvalidValue;
  p.vec = (bits & 15u) == 0;
  int64_t units;
  if (!c->cu_new) {
    p.per_seq = c->tokens / c->batch;
    p.pages_seq = (p.per_seq + c->page_size - 2) / c->page_size + 1;
    units = (int64_t)c->batch * p.pages_seq;
  } else {
    units = c->tokens / c->page_size + 2ll * c->batch;  // sum over b of ceil((n_b - 1) / page) + 1 at most
  }
  // a team keeps its rows in registers: kKeep vectors a lane
  const int64_t rows = std::min<int64_t>(c->page_size, ((int64_t)c->tokens + c->batch - 1) / c->batch);
  p.team = 1;
  while (p.team < kWarps && rows * (c->head_dim / 8) > (int64_t)p.team * 32 * kKeep) p.team *= 2;
  const int64_t rows_y = (2ll * c->kv_heads * p.team + kWarps - 1) / kWarps;
  if (units > 0x7fffffffll || rows_y > 65535) return (int)cudaErrorInvalidValue;
  const dim3 grid((unsigned)units, (unsigned)rows_y);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (units * rows_y > 2ll * num_sms_current())
    return (int)(a->a_type == FP8IMMA_A_F16 ? launch_append<0, 4>(p, grid, st) : launch_append<1, 4>(p, grid, st));
  return (int)(a->a_type == FP8IMMA_A_F16 ? launch_append<0, 1>(p, grid, st) : launch_append<1, 1>(p, grid, st));
}
