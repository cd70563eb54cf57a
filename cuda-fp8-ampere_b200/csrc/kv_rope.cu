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
//
// Measured: 64 sequences of one token, 64/8 heads of 128, 4.4 us; 32 trees of up to 16
// nodes, 28/4 heads of 64, 6.1 us; prompts of 9200 tokens, 32/8 heads of 128, 60 us,
// 3.5 TB/s of the 208 MB read and written: with 124 registers 16 warps an SM go
// through search, angles, keys and queries one after another, at 1.7 instructions a
// cycle.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "kv_cache.cuh"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>
#include <cmath>
#include <cuda_runtime.h>
#include <type_traits>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;
using namespace kv;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kKeep = 2;  // pairs of pieces of a page that a thread keeps (as fp32) between the two passes
constexpr int kQ = 4;     // heads whose pair a thread has in flight

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

// An angle as position * inv_freq / 2 pi without its whole turns, in -0.5 .. 0.5. 1 / 2 pi
// and the products are held as two 64-bit numbers: one alone would leave 2^-21 of an angle at
// a position of 2^31.
struct Frequency {
  double hi, lo;  // inv_freq / 2 pi
  __device__ __forceinline__ explicit Frequency(float inv_freq) {
    constexpr double kHi = 0.15915494309189535, kLo = -9.839338337591243e-18;  // 1 / 2 pi
    hi = inv_freq * kHi;
    lo = fma((double)inv_freq, kHi, -hi) + inv_freq * kLo;
  }
  // cosine and sine of the angle: of its fraction of a turn t as fp32, then a step of the
  // first order by what that leaves (delta, up to 2^-23.3: cos (a + d) = cos a - d sin a
  // to 2^-47), so that small cosines and sines keep their relative precision too
  __device__ __forceinline__ void turn(int position, float& cs, float& sn) const {
    const double at = position, whole = at * hi, t = (whole - rint(whole)) + fma(at, lo, fma(at, hi, -whole));
    const float near = (float)t, delta = (float)((t - near) * 6.283185307179586);
    float s, c;
    sincospif(2.0f * near, &s, &c);
    cs = fmaf(-delta, s, c);
    sn = fmaf(delta, c, s);
  }
};

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

// NaN is left out by fmaxf; an infinity shows in the result, which is then made anew without any.
__device__ __forceinline__ float absmax8(const float (&x)[8], float m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
  return m;
}
__device__ __forceinline__ float absmax8_finite(const float (&x)[8], float m) {
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

// The eight cosines and sines of pair j (j < turning) of a row.
struct Turn {
  float c[8], s[8];
  __device__ __forceinline__ void load(int j, int turning, bool interleaved, const float* cs, const float* sn) {
    // interleaved: four of the first piece, four of the second
    const int at0 = interleaved ? j : 2 * j, at1 = interleaved ? j + turning : 2 * j + 1;
    const float4 c0 = reinterpret_cast<const float4*>(cs)[at0], c1 = reinterpret_cast<const float4*>(cs)[at1];
    const float4 s0 = reinterpret_cast<const float4*>(sn)[at0], s1 = reinterpret_cast<const float4*>(sn)[at1];
    c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
    s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
  }
  __device__ __forceinline__ void apply(float (&x)[8], float (&y)[8], bool interleaved) const {
    if (!interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) one(x[i], y[i], i);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        one(x[2 * i], x[2 * i + 1], i);
        one(y[2 * i], y[2 * i + 1], 4 + i);
      }
    }
  }
  __device__ __forceinline__ void one(float& u, float& v, int i) const {
    const float a = u, b = v;
    u = fmaf(a, c[i], -(b * s[i]));
    v = fmaf(b, c[i], a * s[i]);
  }
};

// PLAIN: half-split pairs and aligned rows, which are most calls; less code for the
// instruction cache.
template <int AT, int FMT, bool PLAIN>
__global__ void __launch_bounds__(kThreads, 2) kv_append_rope_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ __align__(16) float table[];  // cosines [rows][rotary / 2], then sines
  __shared__ float s_max[2][kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool interleaved = !PLAIN && p.a.interleaved, vec = PLAIN || p.vec, vec_q = PLAIN || p.vec_q;
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
  {
    // a thread keeps to one frequency
    const int per = kThreads / half, i = threadIdx.x % half;
    const Frequency f(__ldg(p.a.inv_freq + i));
    for (int r = threadIdx.x / half; r < rows && (int)threadIdx.x < per * half; r += per) {
      float sn, cs;
      f.turn(p.a.positions ? __ldg(p.a.positions + tok + r) : lo + r, cs, sn);
      table[r * half + i] = cs * p.a.rope_scale;
      sines[r * half + i] = sn * p.a.rope_scale;
    }
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
        x = load_row8<AT>(row + at.a * 8, vec);
        y = load_row8<AT>(row + at.b * 8, vec);
      };
      auto values = [&](int v, uint4 a, uint4 c, float (&x)[8], float (&y)[8]) {
        unpack8<AT>(a, x);
        unpack8<AT>(c, y);
        const int j = v & (pairs - 1);
        if (key && j < turning) {
          Turn t;
          t.load(j, turning, interleaved, table + (v >> pl) * half, sines + (v >> pl) * half);
          t.apply(x, y, interleaved);
        }
      };
      float keep[kKeep][2][8], amax = 0.0f;
      {
        uint4 raw[kKeep][2];
#pragma unroll
        for (int i = 0; i < kKeep; ++i)
          if (tid + i * step < nv) load(tid + i * step, raw[i][0], raw[i][1]);
#pragma unroll
        for (int i = 0; i < kKeep; ++i)
          if (tid + i * step < nv) {
            values(tid + i * step, raw[i][0], raw[i][1], keep[i][0], keep[i][1]);
            amax = absmax8(keep[i][1], absmax8(keep[i][0], amax));
          }
      }
#pragma unroll 1
      for (int v = tid + kKeep * step; v < nv; v += step) {
        uint4 a, c;
        float x[8], y[8];
        load(v, a, c);
        values(v, a, c, x, y);
        amax = absmax8(y, absmax8(x, amax));
      }
      if (__any_sync(0xffffffffu, amax == INFINITY)) {
        amax = 0.0f;
#pragma unroll 1
        for (int v = tid; v < nv; v += step) {
          uint4 a, c;
          float x[8], y[8];
          load(v, a, c);
          values(v, a, c, x, y);
          amax = absmax8_finite(y, absmax8_finite(x, amax));
        }
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
      auto put = [&](int v, const float(&x)[8], const float(&y)[8]) {
        const PairAt at(v & (pairs - 1), turning);
        uint8_t* row = dst + (size_t)(slot0 + (v >> pl)) * D;
        *reinterpret_cast<uint2*>(row + at.a * 8) = codes8<FMT>(x, s_new, inv);
        *reinterpret_cast<uint2*>(row + at.b * 8) = codes8<FMT>(y, s_new, inv);
      };
#pragma unroll
      for (int i = 0; i < kKeep; ++i)
        if (tid + i * step < nv) put(tid + i * step, keep[i][0], keep[i][1]);
#pragma unroll 1
      for (int v = tid + kKeep * step; v < nv; v += step) {
        uint4 a, c;
        float x[8], y[8];
        load(v, a, c);
        values(v, a, c, x, y);
        put(v, x, y);
      }
      if (tid == 0) *scale = s_new;
    }
  }

  // queries: a thread keeps to one pair of one row, its cosines and sines in
  // registers, and goes through the heads (every `groups`-th of them)
  const int places = rows << pl, threads = gridDim.y * kThreads, id = blockIdx.y * kThreads + threadIdx.x;
  const int groups = max(1, threads / places);
  for (int at = id; at < groups * places; at += threads) {
    const int group = at / places, place = at - group * places, row = place >> pl, j = place & (pairs - 1);
    const PairAt piece(j, turning);
    const uint16_t* const src = static_cast<const uint16_t*>(p.a.q) + (int64_t)(tok + row) * p.a.q_token_stride;
    uint16_t* const dst = static_cast<uint16_t*>(p.a.q_out) + (int64_t)(tok + row) * p.a.q_out_token_stride;
    Turn t;
    if (j < turning) t.load(j, turning, interleaved, table + row * half, sines + row * half);
    for (int h0 = group; h0 < p.a.heads; h0 += kQ * groups) {
      uint4 raw[kQ][2];
#pragma unroll
      for (int k = 0; k < kQ; ++k) {
        const int h = h0 + k * groups;
        if (h >= p.a.heads) break;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint16_t* s = src + (int64_t)h * p.a.q_head_stride + (c ? piece.b : piece.a) * 8;  // q may be q_out: no read-only loads
          if (vec_q) raw[k][c] = *reinterpret_cast<const uint4*>(s);
          else
            raw[k][c] = make_uint4(s[0] | (uint32_t)s[1] << 16, s[2] | (uint32_t)s[3] << 16, s[4] | (uint32_t)s[5] << 16, s[6] | (uint32_t)s[7] << 16);
        }
      }
#pragma unroll
      for (int k = 0; k < kQ; ++k) {
        const int h = h0 + k * groups;
        if (h >= p.a.heads) break;
        uint4 out[2] = {raw[k][0], raw[k][1]};  // pieces that stay are copied
        if (j < turning) {
          float x[8], y[8];
          unpack8<AT>(raw[k][0], x);
          unpack8<AT>(raw[k][1], y);
          t.apply(x, y, interleaved);
          out[0] = make_uint4(f32x2_to_a16x2<AT>(x[0], x[1]), f32x2_to_a16x2<AT>(x[2], x[3]), f32x2_to_a16x2<AT>(x[4], x[5]), f32x2_to_a16x2<AT>(x[6], x[7]));
          out[1] = make_uint4(f32x2_to_a16x2<AT>(y[0], y[1]), f32x2_to_a16x2<AT>(y[2], y[3]), f32x2_to_a16x2<AT>(y[4], y[5]), f32x2_to_a16x2<AT>(y[6], y[7]));
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint16_t* d = dst + (int64_t)h * p.a.q_out_head_stride + (c ? piece.b : piece.a) * 8;
          if (vec_q) *reinterpret_cast<uint4*>(d) = out[c];
          else {
            const uint32_t w[4] = {out[c].x, out[c].y, out[c].z, out[c].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) d[2 * i] = (uint16_t)w[i], d[2 * i + 1] = (uint16_t)(w[i] >> 16);
          }
        }
      }
    }
  }
}

template <int AT, int FMT, bool PLAIN>
cudaError_t launch_rope(RopeParams& p, int64_t units, int64_t rows, cudaStream_t st) {
  // a team keeps its rows in registers: kKeep pairs a lane
  const int64_t pairs = p.c.head_dim / 16;
  p.team = 1;
  while (p.team < kWarps && rows * pairs > (int64_t)p.team * 32 * kKeep) p.team *= 2;
  // shares of a page: as many as keep its CTAs' threads busy, as long as the
  // whole grid has few CTAs (prompts of 9200 tokens: 63 us with one share, 60 with
  // two; a kernel for the queries of its own, with twice the warps: 73)
  const int64_t cache = (2ll * p.c.kv_heads * p.team + kWarps - 1) / kWarps, queries = (rows * p.a.heads * pairs + kThreads - 1) / kThreads;
  const int64_t shares = std::max<int64_t>(1, std::min<int64_t>(std::max(cache, queries), 12ll * num_sms_current() / units));
  const auto kern = kv_append_rope_kernel<AT, FMT, PLAIN>;
  const int smem = p.table_rows * p.a.rotary * 4;
  const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), smem + 1024);  // static shared memory counts too
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.gridDim = dim3((unsigned)units, (unsigned)std::min<int64_t>(shares, 65535));
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
  if (((kv | q) & 1u) || !aligned4({a->inv_freq, a->positions})) return (int)cudaErrorInvalidValue;
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
  const int64_t rows = std::min<int64_t>(c->page_size, ((int64_t)c->tokens + c->batch - 1) / c->batch);
  const bool plain = !a->interleaved && p.vec && p.vec_q;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&](auto at, auto fmt) {
    constexpr int AT = decltype(at)::value, FMT = decltype(fmt)::value;
    return (int)(plain ? launch_rope<AT, FMT, true>(p, units, rows, st) : launch_rope<AT, FMT, false>(p, units, rows, st));
  };
  using F16 = std::integral_constant<int, 0>;
  using BF16 = std::integral_constant<int, 1>;
  using E4M3 = std::integral_constant<int, F8_E4M3>;
  using E5M2 = std::integral_constant<int, F8_E5M2>;
  if (a->a_type == FP8IMMA_A_F16) return c->format == FP8IMMA_B_E4M3 ? run(F16(), E4M3()) : run(F16(), E5M2());
  return c->format == FP8IMMA_B_E4M3 ? run(BF16(), E4M3()) : run(BF16(), E5M2());
}
