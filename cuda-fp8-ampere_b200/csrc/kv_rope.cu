// Append to the paged 8-bit KV cache with the position rotation on the way
// (fp8imma_kv_append_rope). Scales and codes are those of kv_cache.cu; a key pair
// (x, y) of channels enters as, and a query pair leaves as,
//   (x cos a - y sin a, y cos a + x sin a) * rope_scale,  a = position * inv_freq
// in fp32. The angle is formed in turns, position * (inv_freq / 2 pi) in 64 bits,
// and brought to half a turn there: in 32 bits a position of 10^6 leaves angles off by
// 0.06 and more.
//
// Bound: rows are read and written once; a small step is a chain of latencies.
//  * a CTA takes one page's new tokens, all of its heads and queries among them
//    (in blockIdx.y shares): their cosines and sines are made once, into shared
//    memory, for all heads;
//  * a thread takes two 16-byte pieces of a row that turn together, so the
//    rotation needs no exchange between threads;
//  * a team of 1 .. 8 warps owns one (page, head, K or V) as in kv_cache.cu, its
//    rows in registers between the pass for the scale and the one for the codes.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "kv_cache.cuh"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>
#include <cmath>
#include <cuda_runtime.h>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;
using namespace kv;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kKeep = 4;  // pairs of pieces of a page that a thread keeps between the two passes
constexpr int kQ = 4;     // pairs of query pieces that a thread has in flight

struct RopeParams {
  fp8imma_kv_cache c;
  fp8imma_kv_append_rope_args a;
  int vec;         // rows of k and v are 16-byte aligned
  int vec_q;       // those of q and q_out
  int per_seq;     // > 0: every sequence appends this many tokens
  int pages_seq;   // then: pages a sequence can touch
  int team;        // warps of a (page, head, K or V)
  int table_rows;  // rows that the table of cosines and sines has room for
};

__device__ __forceinline__ int length(const RopeParams& p, int b) { return max(0, __ldg(p.c.seq_lens + b)); }

// Pages that sequence b's new tokens fall into, those before the first place and
// past the table among them (their queries turn all the same).
__device__ __forceinline__ int touched(const RopeParams& p, int b, int& first) {
  int t0, n;
  token_range(p.c, p.per_seq, b, t0, n);
  const int len = length(p, b), pl = __ffs(p.c.page_size) - 1;
  first = (len - n) >> pl;
  return n > 0 ? ((len - 1) >> pl) - first + 1 : 0;
}

// position * inv_freq / 2 pi without its whole turns, in -0.5 .. 0.5. 1 / 2 pi and the
// products are held as two 64-bit numbers: one alone would leave 2^-21 of an angle at
// a position of 2^31.
__device__ __forceinline__ float turn_fraction(int position, float inv_freq) {
  constexpr double kHi = 0.15915494309189535, kLo = -9.839338337591243e-18;  // 1 / 2 pi
  const double f = inv_freq, at = position;
  const double hi = f * kHi, lo = fma(f, kHi, -hi) + f * kLo;
  const double t = at * hi, rest = fma(at, hi, -t) + at * lo;
  return (float)((t - rint(t)) + rest);
}

template <int AT>
__device__ __forceinline__ void unpack8(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = a16_to_f32<AT>((uint16_t)(w[i] & 0xFFFFu));
    x[2 * i + 1] = a16_to_f32<AT>((uint16_t)(w[i] >> 16));
  }
}

template <int FMT>
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float s, float inv) {
  const bool pow2 = (__float_as_uint(s) & 0x7FFFFFu) == 0u;  // as in to_codes()
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = pow2 ? f32x2_to_f8x2<FMT>(x[2 * i] * inv, x[2 * i + 1] * inv) : f32x2_to_f8x2<FMT>(__fdiv_rn(x[2 * i], s), __fdiv_rn(x[2 * i + 1], s));
  return make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
}

__device__ __forceinline__ float absmax8(const float (&x)[8], float m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : 0.0f);
  return m;
}

// Pair j of a row's pieces: two that turn together (j < turning, the number of
// turning pieces halved), or two neighbours of those that stay.
struct PairAt {
  int a, b;
  __device__ __forceinline__ PairAt(int j, int turning) {
    a = j < turning ? j : 2 * j;
    b = j < turning ? j + turning : a + 1;
  }
};

// Turns pair j (j < turning); cos and sin: the row's.
__device__ __forceinline__ void turn(float (&x)[8], float (&y)[8], int j, int turning, bool interleaved, const float* cs, const float* sn) {
  if (!interleaved) {
    const float4* c4 = reinterpret_cast<const float4*>(cs + 8 * j);
    const float4* s4 = reinterpret_cast<const float4*>(sn + 8 * j);
    const float4 c0 = c4[0], c1 = c4[1], s0 = s4[0], s1 = s4[1];
    const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = x[i], v = y[i];
      x[i] = fmaf(u, c[i], -(v * s[i]));
      y[i] = fmaf(v, c[i], u * s[i]);
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float(&z)[8] = h ? y : x;
      const float4 c4 = *reinterpret_cast<const float4*>(cs + 4 * (j + h * turning));
      const float4 s4 = *reinterpret_cast<const float4*>(sn + 4 * (j + h * turning));
      const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = z[2 * i], v = z[2 * i + 1];
        z[2 * i] = fmaf(u, c[i], -(v * s[i]));
        z[2 * i + 1] = fmaf(v, c[i], u * s[i]);
      }
    }
  }
}

template <int AT, int FMT>
__global__ void __launch_bounds__(kThreads, 2) kv_append_rope_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ __align__(16) float table[];  // cosines [rows][rotary / 2], then sines
  __shared__ float s_max[2][kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  int b = 0, first = 0, pi = 0;
  if (!find_page<kThreads>(p.c, p.per_seq, p.pages_seq, [&](int i, int& f) { return touched(p, i, f); }, b, first, pi)) return;
  pi += first;
  const int ps = p.c.page_size, D = p.c.head_dim;
  int t0, n;
  token_range(p.c, p.per_seq, b, t0, n);
  const int len = length(p, b), start = len - n;  // place of token t0; tokens before place 0 are not stored
  const int slot0 = max(start - pi * ps, 0), rows = min(len - pi * ps, ps) - slot0;  // 1 at least
  const int lo = pi * ps + slot0;
  const int tok = t0 + lo - start;
  const bool placed = pi >= 0 && pi < p.c.max_pages;
  const int page = placed ? __ldg(p.c.page_table + (size_t)b * p.c.max_pages + pi) : -1;

  const int half = p.a.rotary >> 1, turning = half >> 3;
  float* const sines = table + p.table_rows * half;
  for (int e = threadIdx.x; e < rows * half; e += kThreads) {
    const int r = e / half, i = e - r * half;
    const int at = p.a.positions ? __ldg(p.a.positions + tok + r) : lo + r;
    float sn, cs;
    sincospif(2.0f * turn_fraction(at, __ldg(p.a.inv_freq + i)), &sn, &cs);
    table[e] = cs * p.a.rope_scale;
    sines[e] = sn * p.a.rope_scale;
  }
  __syncthreads();

  const int pl = __ffs(D) - 5;  // pairs of a row (log2)
  const int pairs = 1 << pl;
  if ((unsigned)page < (unsigned)p.c.num_pages) {
    const int teams = kWarps / p.team;
    const int tid = warp % p.team * 32 + lane, step = p.team * 32;
    int round = 0;
    for (int item0 = blockIdx.y * teams; item0 < 2 * p.c.kv_heads; item0 += gridDim.y * teams, round ^= 1) {
      // this team's head and tensor; teams past the last one only take part in the barrier
      const int item = item0 + warp / p.team;
      const bool on = item < 2 * p.c.kv_heads;
      const int h = item >> 1;
      const bool key = !(item & 1);
      const int64_t ts = key ? p.a.k_token_stride : p.a.v_token_stride;
      const uint16_t* src = static_cast<const uint16_t*>(key ? p.a.k : p.a.v) + (int64_t)tok * ts + (int64_t)h * (key ? p.a.k_head_stride : p.a.v_head_stride);
      const size_t ph = (size_t)page * p.c.kv_heads + h;
      uint8_t* dst = static_cast<uint8_t*>(key ? p.c.k : p.c.v) + ph * ps * D;
      float* scale = (key ? p.c.k_scale : p.c.v_scale) + ph;
      const float s_old = on && slot0 > 0 ? *scale : 0.0f;
      const int nv = on ? rows << pl : 0;
      auto load = [&](int v, uint4& x, uint4& y) {
        const PairAt at(v & (pairs - 1), turning);
        const uint16_t* row = src + (int64_t)(v >> pl) * ts;
        x = load_row8<AT>(row + at.a * 8, p.vec);
        y = load_row8<AT>(row + at.b * 8, p.vec);
      };
      auto values = [&](int v, uint4 a, uint4 c, float (&x)[8], float (&y)[8]) {
        unpack8<AT>(a, x);
        unpack8<AT>(c, y);
        const int j = v & (pairs - 1);
        if (key && j < turning) turn(x, y, j, turning, p.a.interleaved, table + (v >> pl) * half, sines + (v >> pl) * half);
      };
      uint4 keep[kKeep][2];
      float amax = 0.0f, x[8], y[8];
#pragma unroll
      for (int i = 0; i < kKeep; ++i)
        if (tid + i * step < nv) load(tid + i * step, keep[i][0], keep[i][1]);
#pragma unroll
      for (int i = 0; i < kKeep; ++i)
        if (tid + i * step < nv) {
          values(tid + i * step, keep[i][0], keep[i][1], x, y);
          amax = absmax8(y, absmax8(x, amax));
        }
      for (int v = tid + kKeep * step; v < nv; v += step) {
        uint4 a, c;
        load(v, a, c);
        values(v, a, c, x, y);
        amax = absmax8(y, absmax8(x, amax));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (p.team > 1) {
        if (lane == 0) s_max[round][warp] = amax;
        __syncthreads();
        for (int w = 0; w < p.team; ++w) amax = fmaxf(amax, s_max[round][warp / p.team * p.team + w]);
      }
      if (!on) continue;
      const float s_new = fmaxf(s_old, needed_scale<FMT>(amax));
      const float inv = __fdiv_rn(1.0f, s_new);
      if (slot0 > 0 && s_new != s_old) {  // uniform: the page's earlier codes move to the larger scale
        const float ratio = __fdiv_rn(s_old, s_new);
        for (int v = tid; v < slot0 * (D >> 4); v += step) {
          uint4* at = reinterpret_cast<uint4*>(dst) + v;
          *at = moved_codes<FMT>(*at, ratio);
        }
      }
      auto put = [&](int v, uint4 a, uint4 c) {
        values(v, a, c, x, y);
        const PairAt at(v & (pairs - 1), turning);
        uint8_t* row = dst + (size_t)(slot0 + (v >> pl)) * D;
        *reinterpret_cast<uint2*>(row + at.a * 8) = codes8<FMT>(x, s_new, inv);
        *reinterpret_cast<uint2*>(row + at.b * 8) = codes8<FMT>(y, s_new, inv);
      };
#pragma unroll
      for (int i = 0; i < kKeep; ++i)
        if (tid + i * step < nv) put(tid + i * step, keep[i][0], keep[i][1]);
      for (int v = tid + kKeep * step; v < nv; v += step) {
        uint4 a, c;
        load(v, a, c);
        put(v, a, c);
      }
      if (tid == 0) *scale = s_new;
    }
  }

  // queries: the page's rows, all heads, pair after pair
  const int row_pairs = p.a.heads << pl, all = rows * row_pairs, stride = gridDim.y * kThreads;
  for (int e0 = blockIdx.y * kThreads + threadIdx.x; e0 < all; e0 += kQ * stride) {
    uint4 raw[kQ][2];
    int row[kQ], hp[kQ];
#pragma unroll
    for (int k = 0; k < kQ; ++k) {
      const int e = e0 + k * stride;
      if (e >= all) continue;
      row[k] = e / row_pairs;
      hp[k] = e - row[k] * row_pairs;
      const PairAt at(hp[k] & (pairs - 1), turning);
      const uint16_t* src = static_cast<const uint16_t*>(p.a.q) + (int64_t)(tok + row[k]) * p.a.q_token_stride + (int64_t)(hp[k] >> pl) * p.a.q_head_stride;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint16_t* s = src + (c ? at.b : at.a) * 8;  // q may be q_out: no read-only loads
        if (p.vec_q) raw[k][c] = *reinterpret_cast<const uint4*>(s);
        else
          raw[k][c] = make_uint4(s[0] | (uint32_t)s[1] << 16, s[2] | (uint32_t)s[3] << 16, s[4] | (uint32_t)s[5] << 16, s[6] | (uint32_t)s[7] << 16);
      }
    }
#pragma unroll
    for (int k = 0; k < kQ; ++k) {
      if (e0 + k * stride >= all) continue;
      const int j = hp[k] & (pairs - 1);
      const PairAt at(j, turning);
      uint16_t* dst = static_cast<uint16_t*>(p.a.q_out) + (int64_t)(tok + row[k]) * p.a.q_out_token_stride + (int64_t)(hp[k] >> pl) * p.a.q_out_head_stride;
      float x[8], y[8];
      unpack8<AT>(raw[k][0], x);
      unpack8<AT>(raw[k][1], y);
      if (j < turning) {
        turn(x, y, j, turning, p.a.interleaved, table + row[k] * half, sines + row[k] * half);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float(&z)[8] = c ? y : x;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)f32_to_a16<AT>(z[2 * i]) | (uint32_t)f32_to_a16<AT>(z[2 * i + 1]) << 16;
        uint16_t* d = dst + (c ? at.b : at.a) * 8;
        if (p.vec_q) *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
        else {
#pragma unroll
          for (int i = 0; i < 4; ++i) d[2 * i] = (uint16_t)w[i], d[2 * i + 1] = (uint16_t)(w[i] >> 16);
        }
      }
    }
  }
}

template <int AT, int FMT>
cudaError_t launch_rope(const RopeParams& p, dim3 grid, cudaStream_t st) {
  const auto kern = kv_append_rope_kernel<AT, FMT>;
  const int smem = p.table_rows * p.a.rotary * 4;
  const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), smem + 1024);  // static shared memory counts too
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.gridDim = grid;
  lc.blockDim = dim3(kThreads);
  lc.dynamicSmemBytes = (size_t)smem;
  lc.stream = st;
  lc.attrs = attr;
  lc.numAttrs = api_pdl() ? 1 : 0;
  return cudaLaunchKernelEx(&lc, kern, p);
}

}  // namespace

unsigned int kv_rope_device_error(bool clear) { return fp8imma_dev::tu_device_error(clear); }

}  // namespace fp8imma_b200

using namespace fp8imma_b200;

extern "C" int fp8imma_kv_append_rope(const fp8imma_kv_cache* c, const fp8imma_kv_append_rope_args* a, void* stream) {
  FP8IMMA_RANGE("fp8imma_kv_append_rope");
  const cudaError_t e = kv_cache_check(c);
  if (e != cudaSuccess) return (int)e;
  if (!a || !a->k || !a->v || !a->inv_freq || a->a_type < 0 || a->a_type > 1) return (int)cudaErrorInvalidValue;
  if (a->rotary <= 0 || a->rotary % 16 || a->rotary > c->head_dim || !std::isfinite(a->rope_scale)) return (int)cudaErrorInvalidValue;
  if (a->heads < 0 || a->heads > 65535 || (a->heads > 0 && (!a->q || !a->q_out))) return (int)cudaErrorInvalidValue;
  RopeParams p = {};
  p.c = *c;
  p.a = *a;
  const uintptr_t kv = reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
                       (uintptr_t)((a->k_token_stride | a->k_head_stride | a->v_token_stride | a->v_head_stride) * 2);
  const uintptr_t q = a->heads == 0 ? 0 : reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->q_out) |
                       (uintptr_t)((a->q_token_stride | a->q_head_stride | a->q_out_token_stride | a->q_out_head_stride) * 2);
  if ((kv | q) & 1u) return (int)cudaErrorInvalidValue;
  p.vec = (kv & 15u) == 0;
  p.vec_q = (q & 15u) == 0;
  int64_t units;
  if (!c->cu_new) {
    p.per_seq = c->tokens / c->batch;
    p.pages_seq = (p.per_seq + c->page_size - 2) / c->page_size + 1;
    units = (int64_t)c->batch * p.pages_seq;
  } else {
    units = c->tokens / c->page_size + 2ll * c->batch;  // sum over b of ceil((n_b - 1) / page) + 1 at most
  }
  if (units > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  p.table_rows = std::min(c->page_size, c->cu_new ? c->tokens : p.per_seq);
  // a team keeps its rows in registers: kKeep pairs a lane
  const int64_t rows = std::min<int64_t>(c->page_size, ((int64_t)c->tokens + c->batch - 1) / c->batch);
  p.team = 1;
  while (p.team < kWarps && rows * (c->head_dim / 16) > (int64_t)p.team * 32 * kKeep) p.team *= 2;
  // shares of a page: as many as keep its CTAs' threads busy, as long as the
  // whole grid has few CTAs
  const int64_t most = std::max<int64_t>((2ll * c->kv_heads * p.team + kWarps - 1) / kWarps, (rows * a->heads * (c->head_dim / 16) + kThreads - 1) / kThreads);
  const int64_t shares = std::min<int64_t>({most, std::max<int64_t>(1, 8ll * num_sms_current() / units), 65535});
  const dim3 grid((unsigned)units, (unsigned)shares);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool e4 = c->format == FP8IMMA_B_E4M3;
  if (a->a_type == FP8IMMA_A_F16) return (int)(e4 ? launch_rope<0, F8_E4M3>(p, grid, st) : launch_rope<0, F8_E5M2>(p, grid, st));
  return (int)(e4 ? launch_rope<1, F8_E4M3>(p, grid, st) : launch_rope<1, F8_E5M2>(p, grid, st));
}
