// Log probabilities of given tokens, entropy and top alternatives of logits
// (fp8imma_token_logprobs).
//
// Mathematics, z = x / temperature, in base 2 (u = z log2 e), one pass with a
// running reference M per lane:
//   l = sum 2^(u - M),  s = sum 2^(u - M) (u - M)
//   lse = ln2 (M + log2 l),  entropy = ln2 (log2 l - s / l),  lp(t) = z_t - lse
// and parts join as l = sum l_i 2^(M_i - M), s = sum 2^(M_i - M) (s_i + (M_i - M) l_i).
// The top logits are a warp's list of 32, one a lane in descending order; a
// logit enters it only when it exceeds the list's last, which after the first
// few hundred logits is rare, so the pass pays one comparison for it. Order is
// by the logit's bits (order-preserving), then by the lower index, so lists
// and their joins do not depend on which part is read first.
//
// Bound: the logits are read once. A row is cut into as many parts as fill the
// GPU (one row of 32000 bf16 logits: latency; thousands of rows: bandwidth);
// the last CTA to finish a row joins its parts in order.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr unsigned long long kNoKey = 0ull;  // below the key of every logit

struct LpParams {
  fp8imma_logprobs_args a;
  float to_log2;          // log2(e) / temperature
  float inv_temp;
  int parts;              // CTAs a row (row-major) or a group of rows (column-major)
  int per_part;           // logits of a part
  int groups;             // column-major: 32-row groups
  unsigned int* counters; // per row (group): finished parts; zero between calls
  float* sums;            // [parts, tokens, 4]: M, l, s, -
  unsigned long long* lists;  // [parts, tokens, 32]
};

template <int LT>
__device__ __forceinline__ float to_f32(uint32_t bits) {
  if (LT == FP8IMMA_L_F32) return __uint_as_float(bits);
  return a16_to_f32<LT>((uint16_t)bits);
}

// Descending order of logits: NaN, +inf .. -inf (-0 = +0), then the lower index.
__device__ __forceinline__ unsigned long long make_key(float v, int j) {
  const int k = __float_as_int(v);
  unsigned o = isnan(v) ? 0xffffffffu : k < 0 ? 0x80000000u - (unsigned)(k & 0x7fffffff) : 0x80000000u + (unsigned)k;
  return ((unsigned long long)o << 32) | (unsigned)(0x7fffffff - j);
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const unsigned o = (unsigned)(key >> 32);
  if (o == 0xffffffffu) return NAN;
  return o >= 0x80000000u ? __uint_as_float(o - 0x80000000u) : -__uint_as_float(0x80000000u - o);
}
__device__ __forceinline__ int key_index(unsigned long long key) { return 0x7fffffff - (int)(unsigned)key; }

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Running sums of one lane (or of a joined part).
struct Sums {
  float m = -INFINITY, l = 0.0f, s = 0.0f;
  bool bad = false;  // NaN or +inf was seen
  __device__ __forceinline__ void join(float m2, float l2, float s2) {
    const float mn = fmaxf(m, m2);
    if (mn == -INFINITY) return;
    const float a = m == -INFINITY ? 0.0f : ex2(m - mn), b = m2 == -INFINITY ? 0.0f : ex2(m2 - mn);
    const float da = m == -INFINITY ? 0.0f : m - mn, db = m2 == -INFINITY ? 0.0f : m2 - mn;
    s = a * (s + da * l) + b * (s2 + db * l2);
    l = a * l + b * l2;
    m = mn;
  }
};

// A warp's list: lane i holds the i-th largest key. Insert one key (uniform).
__device__ __forceinline__ void insert(unsigned long long& mine, unsigned long long key, int lane) {
  const unsigned below = __ballot_sync(0xffffffffu, mine < key);  // a suffix of the lanes: they move down by one
  const unsigned long long up = __shfl_up_sync(0xffffffffu, mine, 1);
  if ((below >> lane) & 1u) mine = lane > 0 && ((below >> (lane - 1)) & 1u) ? up : key;
}

// Two descending lists (one a lane) -> the 32 largest, descending.
__device__ __forceinline__ unsigned long long merge(unsigned long long a, unsigned long long b, int lane) {
  const unsigned long long r = __shfl_sync(0xffffffffu, b, 31 - lane);
  unsigned long long v = a > r ? a : r;  // the 32 largest, bitonic
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
    v = (lane & o) ? (w < v ? w : v) : (w > v ? w : v);
  }
  return v;
}
}  // namespace
}  // namespace fp8imma_b200
