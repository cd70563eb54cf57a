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
//
// Measured: 8192 rows of 4096 (bf16, both norms, a gate a token, residual) 56 to 61
// us, 5.5 to 6.0 TB/s of the 336 MB; one row of 4096 2.0 us; 64 rows of 8192 with an
// fp32 residual 4.4 us, the chain of two sums. Without a gate, cold caches: both norms
// 62 us, one 51; with fp32 weights, which rows copied ahead do not take, 83 and 64. Rows
// that are not whole, aligned eights go an element a load: 8192 rows of 4097 288 us.
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
  int team;         // threads of a row
  int stages;       // bulk copies: rounds of rows in flight
  int stage_bytes;  // and a round's bytes: y, residual, gate of the CTA's rows
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

// Sum over the row's team: every thread gets it, in one order. A caller in a loop takes
// two places in turn: a warp may write its part of the next sum while others still read
// this one's, and it is the next sum's barrier that tells that they have.
__device__ __forceinline__ float team_sum(float x, float* s, int team, int warp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (team == 32) return x;
  const int lane = threadIdx.x & 31, warps = team / 32;
  if (lane == 0) s[warp] = x;
  __syncthreads();
  x = s[(warp & ~(warps - 1)) + (lane & (warps - 1))];
  for (int o = warps / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// 16 or 32 bytes of a tensor as they lie there: eight elements.
template <bool F32>
struct Raw {
  static constexpr int kSize = F32 ? 4 : 2;
  uint4 w[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    const uint4* s = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + at * (F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = s[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  template <int AT>
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) {
      const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (F32) {
          v[4 * i + k] = __uint_as_float(x[k]);
        } else {
          v[2 * k] = a16_to_f32<AT>((uint16_t)(x[k] & 0xFFFFu));
          v[2 * k + 1] = AT == 0 ? a16_to_f32<0>((uint16_t)(x[k] >> 16)) : __uint_as_float(x[k] & 0xFFFF0000u);
        }
      }
    }
  }
};

template <int AT>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = f32x2_to_a16x2<AT>(v[2 * i], v[2 * i + 1]);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// n contiguous bytes (a multiple of 16, both sides aligned) to shared memory
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t n, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(n),
               "r"(smem_u32(bar))
               : "memory");
}

constexpr int kMaxStages = 8;

// Rows of whole, aligned eights, V of them a thread. Teams walk over the rows;
// weights come from the caches each time, asked for before the sum that they wait
// for. BULK: one thread copies the rows of the next rounds to shared memory, which
// keeps more of them in flight than registers could. W32: weights or gate are not of
// y's type.
template <int AT, bool R32, bool W32, int V, bool BULK, int CTA>
__global__ void __launch_bounds__(CTA, CTA == 256 ? (V == 4 ? 2 : 3) : 1) residual_norm_vec_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t s_full[kMaxStages];
  __shared__ float s_sum[2][32];
  if (BULK) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < p.stages; ++i) mbar_init(&s_full[i], 1);
      fence_barrier_init();
    }
    __syncthreads();
  }
  pdl_launch_dependents();
  pdl_wait();
  const fp8imma_residual_norm_args& a = p.a;
  const int warp = threadIdx.x >> 5, tid = threadIdx.x & (p.team - 1), n = a.hidden, rows = blockDim.x / p.team;
  const int64_t step = (int64_t)gridDim.x * rows;
  int64_t row = (int64_t)blockIdx.x * rows + threadIdx.x / p.team;
  Raw<false> y[V], g[V];
  Raw<R32> r[V];
  auto inside = [&](int v) { return (v * p.team + tid) * 8 < n; };
  auto fetch = [&]() {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = (v * p.team + tid) * 8;
      if (row < a.tokens && e < n) {
        y[v].load(a.y, row * a.y_stride + e);
        if (a.residual) r[v].load(a.residual, row * a.residual_stride + e);
        else r[v].zero();
        if (!W32 && a.gate) g[v].load(a.gate, row * a.gate_stride + e);
      } else {
        y[v].zero();
        r[v].zero();
        g[v].zero();
      }
    }
  };
  // BULK: the rows of the round that begins at row `at` into a stage
  const int y_bytes = n * 2, r_bytes = a.residual ? n * Raw<R32>::kSize : 0, g_bytes = a.gate && a.gate_stride ? n * 2 : 0;
  const int row_bytes = y_bytes + r_bytes + g_bytes;
  auto copy = [&](int64_t at, int stage) {
    if (at >= a.tokens) return;
    const int many = (int)min((int64_t)rows, a.tokens - at);
    mbar_arrive_expect_tx(&s_full[stage], (uint32_t)(many * row_bytes));
    for (int i = 0; i < many; ++i) {
      uint8_t* dst = ring + stage * p.stage_bytes + i * row_bytes;
      bulk_load(dst, static_cast<const uint16_t*>(a.y) + (at + i) * a.y_stride, (uint32_t)y_bytes, &s_full[stage]);
      if (r_bytes) bulk_load(dst + y_bytes, static_cast<const char*>(a.residual) + (at + i) * a.residual_stride * Raw<R32>::kSize, (uint32_t)r_bytes, &s_full[stage]);
      if (g_bytes) bulk_load(dst + y_bytes + r_bytes, static_cast<const uint16_t*>(a.gate) + (at + i) * a.gate_stride, (uint32_t)g_bytes, &s_full[stage]);
    }
  };
  int stage = 0;
  uint32_t phase = 0;
  int turn = 0;  // of s_sum: sums alternate, whether a round has one or two
  bool ok = true;
  if (BULK && threadIdx.x == 0)
    for (int i = 0; i < p.stages; ++i) copy((int64_t)blockIdx.x * rows + i * step, i);
  const float by_n = __fdiv_rn(1.0f, (float)n);
  // all teams of a CTA go as many rounds as its first, whose rows are the lowest
  for (int64_t first = (int64_t)blockIdx.x * rows; first < a.tokens; first += step) {
    const int64_t at = row;
    if (BULK) {
      if (ok) ok = mbar_wait(&s_full[stage], phase, ERR_WAIT_FULL);
      const uint8_t* src = ring + stage * p.stage_bytes + threadIdx.x / p.team * row_bytes;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int e = (v * p.team + tid) * 8;
        y[v].zero();
        r[v].zero();
        g[v].zero();
        if (at < a.tokens && e < n) {
          y[v].load(src, e);
          if (r_bytes) r[v].load(src + y_bytes, e);
          if (g_bytes) g[v].load(src + y_bytes + r_bytes, e);
          else if (!W32 && a.gate) g[v].load(a.gate, e);
        }
      }
      __syncthreads();  // the stage has been read
      if (threadIdx.x == 0 && ok) copy(first + p.stages * step, stage);
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1;
      }
    } else {
      fetch();
    }
    float x[V][8], z[V][8], gate[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      y[v].template values<AT>(x[v]);
      r[v].template values<AT>(z[v]);
#pragma unroll
      for (int i = 0; i < 8; ++i) gate[v][i] = a.alpha;
      if (!W32 && a.gate) {
        g[v].template values<AT>(gate[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) gate[v][i] *= a.alpha;
      }
    }
    row += step;
    auto weights = [&](const void* w, int v, Raw<false>& raw) {
      if (!W32 && inside(v)) raw.load(w, (v * p.team + tid) * 8);
    };
    auto weigh = [&](const void* w, int v, const Raw<false>& raw, float (&out)[8]) {
      if (W32) {
        Eight<1> e;
        e.load(w, a.w_type, 0, (v * p.team + tid) * 8, 0, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = inside(v) ? e.v[i] + a.weight_offset : 0.0f;
      } else {
        raw.template values<AT>(out);
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] += a.weight_offset;
      }
    };
    if (W32 && a.gate && at < a.tokens) {  // never with BULK
#pragma unroll
      for (int v = 0; v < V; ++v) {
        Eight<1> e;
        e.load(a.gate, a.g_type, at * a.gate_stride, (v * p.team + tid) * 8, 0, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) gate[v][i] = inside(v) ? a.alpha * e.v[i] : 0.0f;
      }
    }
    Raw<false> w[V];
    if (a.post_weight) {
#pragma unroll
      for (int v = 0; v < V; ++v) weights(a.post_weight, v, w[v]);
      float s = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(x[v][i], x[v][i], s);
      s = team_sum(s, s_sum[turn], p.team, warp);
      turn ^= 1;
      const float f = rsqrtf(fmaf(s, by_n, a.eps));
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float u[8];
        weigh(a.post_weight, v, w[v], u);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[v][i] *= f * u[i];
      }
    }
    if (a.pre_weight) {
#pragma unroll
      for (int v = 0; v < V; ++v) weights(a.pre_weight, v, w[v]);
    }
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        z[v][i] = fmaf(gate[v][i], x[v][i], z[v][i]);
        s = inside(v) ? fmaf(z[v][i], z[v][i], s) : s;
      }
      if (a.residual_out && at < a.tokens && inside(v)) {
        const int64_t o = at * n + (v * p.team + tid) * 8;
        if (R32) {
          float4* d = reinterpret_cast<float4*>(static_cast<float*>(a.residual_out) + o);
          d[0] = make_float4(z[v][0], z[v][1], z[v][2], z[v][3]);
          d[1] = make_float4(z[v][4], z[v][5], z[v][6], z[v][7]);
        } else {
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.residual_out) + o) = pack8<AT>(z[v]);
        }
      }
    }
    if (!a.pre_weight) continue;
    s = team_sum(s, s_sum[turn], p.team, warp);
    turn ^= 1;
    const float f = rsqrtf(fmaf(s, by_n, a.eps));
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float u[8];
      weigh(a.pre_weight, v, w[v], u);
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] *= z[v][i] * f;
      if (at < a.tokens && inside(v)) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at * n + (v * p.team + tid) * 8) = pack8<AT>(u);
    }
  }
  if (BULK && !ok && threadIdx.x == 0)  // a wait ran out: what is still in flight lands before the CTA ends
    for (int i = 0; i < p.stages; ++i) mbar_wait(&s_full[i], phase ^ (i < stage ? 1 : 0), ERR_WAIT_FULL);
}

// Any size and alignment. V: eights of a thread.
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
    const float f = rsqrtf(__fdiv_rn(s, (float)n) + a.eps);
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
  const float f = rsqrtf(__fdiv_rn(s, (float)n) + a.eps);
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

template <class Kern>
cudaError_t launch(Kern kern, const NormParams& p, int ctas, int threads, int smem, cudaStream_t st) {
  const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), smem + 1024);  // static shared memory counts too
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.gridDim = dim3((unsigned)ctas);
  lc.blockDim = dim3((unsigned)threads);
  lc.dynamicSmemBytes = (size_t)smem;
  lc.stream = st;
  lc.attrs = attr;
  lc.numAttrs = api_pdl() ? 1 : 0;
  return cudaLaunchKernelEx(&lc, kern, p);
}

template <int V>
cudaError_t launch_any(const NormParams& p, cudaStream_t st) {
  const int threads = std::max(p.team, kCta), rows = threads / p.team;
  return launch(residual_norm_kernel<0, V>, p, (int)((p.a.tokens + (int64_t)rows - 1) / rows), threads, 0, st);
}

int team_of(int eights, int v) {
  int team = 32;
  while (team * v < eights) team *= 2;
  return team;
}

// Rows copied ahead: CTAs of THREADS threads, per_sm of them an SM.
template <int AT, bool R32, int V, int THREADS>
cudaError_t launch_bulk(NormParams p, int per_sm, cudaStream_t st, bool& taken) {
  const fp8imma_residual_norm_args& a = p.a;
  p.team = team_of(a.hidden / 8, V);
  const int rows = THREADS / p.team, ctas = per_sm * num_sms_current();
  p.stage_bytes = rows * a.hidden * (2 + (a.residual ? (R32 ? 4 : 2) : 0) + (a.gate && a.gate_stride ? 2 : 0));
  p.stages = std::min(kMaxStages, (220 / per_sm - 2) * 1024 / p.stage_bytes);
  taken = p.stages >= 2 && a.tokens > 2ll * ctas * rows;
  return taken ? launch(residual_norm_vec_kernel<AT, R32, false, V, true, THREADS>, p, ctas, THREADS, p.stages * p.stage_bytes, st) : cudaSuccess;
}

// Two or four eights a thread and few warps a row when there are rows for more
// than two rounds: a round is a chain of two sums over the row, and it is rows in
// work that fill the time of it (8192 rows of 4096, with residual and gates: 60 us;
// with one eight in 512 threads 76 us, without copies ahead 80). Otherwise as
// many threads a row as there are eights.
template <int AT, bool R32>
cudaError_t launch_vec(NormParams& p, bool w32, cudaStream_t st) {
  const fp8imma_residual_norm_args& a = p.a;
  const int eights = a.hidden / 8;
  if (!w32) {
    bool taken = false;
    const cudaError_t e = eights <= 512    ? launch_bulk<AT, R32, 2, 256>(p, 3, st, taken)
                          : eights <= 1024 ? launch_bulk<AT, R32, 4, 256>(p, 2, st, taken)
                                           : launch_bulk<AT, R32, 2, 1024>(p, 1, st, taken);
    if (taken) return e;
  }
  const int v = eights <= 1024 ? 1 : 2;
  p.team = team_of(eights, v);
  const int threads = std::max(p.team, kCta), rows = threads / p.team;
  const int ctas = (int)std::min<int64_t>((a.tokens + (int64_t)rows - 1) / rows, (int64_t)num_sms_current() * std::max(1, 1024 / threads));
  if (v == 1)
    return w32 ? launch(residual_norm_vec_kernel<AT, R32, true, 1, false, 1024>, p, ctas, threads, 0, st)
               : launch(residual_norm_vec_kernel<AT, R32, false, 1, false, 1024>, p, ctas, threads, 0, st);
  return w32 ? launch(residual_norm_vec_kernel<AT, R32, true, 2, false, 1024>, p, ctas, threads, 0, st)
             : launch(residual_norm_vec_kernel<AT, R32, false, 2, false, 1024>, p, ctas, threads, 0, st);
}

}  // namespace

unsigned int norm_device_error(bool clear) { return fp8imma_dev::tu_device_error(clear); }
cudaError_t norm_set_wait_limit(unsigned long long ns) { return fp8imma_dev::tu_set_wait_limit(ns); }

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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool w32 = ((a->post_weight || a->pre_weight) && a->w_type != a->a_type) || (a->gate && a->g_type != a->a_type);
  const bool r32 = a->r_type == FP8IMMA_L_F32, same = r32 || a->r_type == a->a_type;
  if (vec && same && a->hidden <= 16384) {
    if (a->a_type == FP8IMMA_A_F16) return (int)(r32 ? launch_vec<0, true>(p, w32, st) : launch_vec<0, false>(p, w32, st));
    return (int)(r32 ? launch_vec<1, true>(p, w32, st) : launch_vec<1, false>(p, w32, st));
  }
  const int eights = (a->hidden + 7) / 8, v = eights <= 256 ? 1 : eights <= 2048 ? 2 : 4;
  p.team = team_of(eights, v);
  return (int)(v == 1 ? launch_any<1>(p, st) : v == 2 ? launch_any<2>(p, st) : launch_any<4>(p, st));
}
