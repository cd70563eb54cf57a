// Log probabilities of given tokens, entropy and top alternatives of logits
// (fp8imma_token_logprobs).
//
// Mathematics, z = x / temperature, in base 2 (c = log2 e / temperature), one
// pass with a running reference M per lane, which is a logit:
//   d = (x - M) c,  l = sum 2^d,  s = sum 2^d d
//   entropy = ln2 (log2 l - s / l),  lp(t) = (x_t - M) / temperature - ln2 log2 l
// and parts join as l = sum l_i 2^d_i, s = sum 2^d_i (s_i + d_i l_i), d_i = (M_i - M) c.
// Differences are taken before the product with c, so that equal logits give
// exactly 1 however large they are: a lane may see nothing but logits masked by
// -1e9, and c x - c M would be off by more than fp32's exponent can hold then. A
// side whose 2^d_i is zero takes no part (d_i l_i may be infinite). A pair of
// logits costs a sum more than with c M: 4096 rows of 32001 bf16 59.5 us instead of 58.8.
// The top logits are a warp's list of 32, one a lane in descending order. The
// pass compares a lane's largest of eight logits with what the list would take;
// those that reach it go to a buffer in shared memory, and 32 of them at a time
// are sorted and merged into the list. Order is by the logit's bits
// (order-preserving), then by the lower index, so lists and their joins do not
// depend on which part is read first.
//
// Bound: the logits are read once. A row is cut into as many parts as fill the
// GPU (one row of 32000 bf16 logits: latency; thousands of rows: bandwidth);
// the last CTA to finish a row joins its parts in order.
//
// Measured: 4096 rows of 32001 bf16 logits 60 us without alternatives (4.4 TB/s;
// instruction issue: an exponential and two sums a logit), 86 us with five of
// them; 16 rows of 128000 with 20, half of the logits masked, 17 us whether by
// -inf or by -1e30; one row of 32000 with 8 alternatives 9.4 us, latency: launch, part, join;
// 16 column-major rows of 128000 with 20 alternatives 32 us, the sorting of short
// parts' candidates.
#include "fp8_mma.cuh"
#include "fp8imma/fp8imma_ext.h"
#include "fp8imma_kernels.h"
#include "nvtx_range.h"
#include "sm100_async.cuh"

#include <algorithm>
#include <type_traits>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;

constexpr int kColWarps = 8;
constexpr unsigned long long kNoKey = 0ull;  // below the key of every logit

struct LpParams {
  fp8imma_logprobs_args a;
  float to_log2;          // log2(e) / temperature
  float inv_temp;
  int flush_at;           // gathered logits that are worth a sort: with a longer list a sort raises its bar less
  int parts;              // CTAs a row (row-major) or a group of rows (column-major)
  int per_part;           // logits of a part
  int group, groups;      // column-major: tokens of a group, groups
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
__device__ __forceinline__ unsigned order_bits(float v) {  // of a number
  const unsigned k = __float_as_uint(v);
  return k >> 31 ? 0x80000000u - (k & 0x7fffffffu) : k | 0x80000000u;
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

constexpr float kLowest = -3.4028234663852886e38f;  // reference before any logit was seen: the lowest number
constexpr float kRaise = 8.0f;                      // the reference follows the maximum when it lies this far above

// Running sums of a lane or of joined parts; c: log2(e) / temperature.
struct Sums {
  float m = kLowest, l = 0.0f, s = 0.0f;
  // (l, s) against a reference that lies -d higher
  static __device__ __forceinline__ void shift(float d, float& l, float& s) {
    const float f = ex2(d);
    s = f == 0.0f ? 0.0f : f * fmaf(d, l, s);
    l *= f;
  }
  __device__ __forceinline__ void join(float m2, float l2, float s2, float c) {
    const float mn = fmaxf(m, m2);
    shift((m - mn) * c, l, s);
    shift((m2 - mn) * c, l2, s2);
    l += l2;
    s += s2;
    m = mn;
  }
  // to the largest of the next logits, when it lies far above
  __device__ __forceinline__ void follow(float big, float c) {
    if ((big - m) * c > kRaise) {
      shift((m - big) * c, l, s);
      m = big;
    }
  }
  __device__ __forceinline__ void add(float x, float c) {
    const float d = (x - m) * c, e = ex2(d);
    l += e;
    s = fmaf(e, fmaxf(d, -1000.0f), s);  // a logit of -inf: 0 * -1000
  }
  __device__ __forceinline__ void warp_join(float c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      join(m2, l2, s2, c);
    }
  }
};

// The sums of two logits at a time: products and sums of pairs are one operation.
struct Pair {
  unsigned long long c, m, l, s;
  static __device__ __forceinline__ unsigned long long of(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
  }
  static __device__ __forceinline__ void to(unsigned long long x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
  static __device__ __forceinline__ unsigned long long sum(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
  }
  static __device__ __forceinline__ unsigned long long product(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
  }
  static __device__ __forceinline__ unsigned long long fma(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
  }
  __device__ __forceinline__ Pair(const Sums& z, float to_log2) : c(of(to_log2, to_log2)), m(of(-z.m, -z.m)), l(of(z.l, 0.0f)), s(of(z.s, 0.0f)) {}
  __device__ __forceinline__ void add(float x, float y) {
    float d0, d1;
    to(product(sum(of(x, y), m), c), d0, d1);
    const unsigned long long e = of(ex2(d0), ex2(d1));
    l = sum(l, e);
    s = fma(e, of(fmaxf(d0, -1000.0f), fmaxf(d1, -1000.0f)), s);  // a logit of -inf: 0 * -1000
  }
  __device__ __forceinline__ void fold(Sums& z) const {
    float a, b;
    to(l, a, b);
    z.l = a + b;
    to(s, a, b);
    z.s = a + b;
  }
};

// A warp's list: lane i holds the i-th largest key. Enters one key (the same
// in all lanes).
__device__ __forceinline__ void insert(unsigned long long& mine, unsigned long long key, int lane) {
  const unsigned long long up = __shfl_up_sync(0xffffffffu, mine, 1);
  if (mine < key) mine = lane > 0 && up < key ? up : key;
}
__device__ __forceinline__ unsigned long long step(unsigned long long v, int o, bool larger) {
  const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
  return (w > v) == larger ? w : v;
}
// Two descending lists -> the 32 largest, descending.
__device__ __forceinline__ unsigned long long merge(unsigned long long a, unsigned long long b, int lane) {
  const unsigned long long r = __shfl_sync(0xffffffffu, b, 31 - lane);
  unsigned long long v = a > r ? a : r;  // bitonic
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = step(v, o, !(lane & o));
  return v;
}
// n keys of the first lanes (kNoKey in the others) sorted and merged into a list.
__device__ __noinline__ unsigned long long sort_merge(unsigned long long list, unsigned long long key, int n, int lane) {
#pragma unroll 1
  for (int k = 2; k < 2 * n; k <<= 1)
#pragma unroll 1
    for (int o = k >> 1; o > 0; o >>= 1) key = step(key, o, !(lane & o) == !(lane & k));
  return merge(list, key, lane);
}

// A warp's list.
struct Top {
  unsigned long long mine = kNoKey, last = kNoKey;  // the lane's entry, the list's top-th
};
// Enters one key a lane (kNoKey: none).
__device__ __forceinline__ void enter(Top& t, unsigned long long key, int top, int lane) {
  unsigned who = __ballot_sync(0xffffffffu, key > t.last);
  if (!who) return;
  if (__popc(who) > 4) {
    t.mine = sort_merge(t.mine, key, 32, lane);
  } else {
    do {
      insert(t.mine, __shfl_sync(0xffffffffu, key, __ffs(who) - 1), lane);
      who &= who - 1;
    } while (who);
  }
  t.last = __shfl_sync(0xffffffffu, t.mine, top - 1);
}
// Candidates for a warp's list, gathered in shared memory: up to 31 left over
// and 8 a lane more.
constexpr int kBuffer = 32 + 256;

// The smallest value that can still enter: `floor` is a value that the row's
// top-th logit is known to reach (order bits), which an equal one may share.
__device__ __forceinline__ float enters_at(const Top& t, unsigned floor) {
  const unsigned own = t.last == kNoKey ? 0u : (unsigned)(t.last >> 32) + 1u;  // later logits come with higher indexes
  const unsigned o = max(own, floor);
  return o == 0u ? -INFINITY : key_value((unsigned long long)o << 32);
}
// Sorts the n gathered keys into the list.
__device__ __noinline__ Top flush(Top t, const unsigned long long* buf, int n, int top, int lane) {
  __syncwarp();
  for (; n > 0; n -= 32) t.mine = sort_merge(t.mine, lane < n ? buf[n - 1 - lane] : kNoKey, min(n, 32), lane);
  __syncwarp();
  t.last = __shfl_sync(0xffffffffu, t.mine, top - 1);
  return t;
}
// The value that the top-th largest of the lanes' values reaches (-inf: none).
__device__ __noinline__ float first_bar(float big, int top, int lane) {
  unsigned v = order_bits(big);
#pragma unroll 1
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll 1
    for (int o = k >> 1; o > 0; o >>= 1) {
      const unsigned w = __shfl_xor_sync(0xffffffffu, v, o);
      v = !(lane & o) == !(lane & k) ? max(v, w) : min(v, w);
    }
  return key_value((unsigned long long)__shfl_sync(0xffffffffu, v, top - 1) << 32);
}

// What a row's sums give: lp(x) = (x - at) * inv - ln_l.
struct Norm {
  float at, inv, ln_l, entropy;
  unsigned long long mine;  // the lane's entry of the list
};

// Rows that the pass cannot do: those that hold NaN or +inf or only -inf. One
// warp, two passes over the row.
template <int LT, class Load>
__device__ __noinline__ Norm careful(int vocab, int n_top, float to_log2, float inv_temp, Load load, int lane) {
  float m = -INFINITY;
  bool bad = false;
  Top top;
  for (int j0 = 0; j0 < vocab; j0 += 32) {
    const bool in = j0 + lane < vocab;
    const float x = in ? load(j0 + lane) : -INFINITY;
    bad |= !(x < INFINITY);
    m = fmaxf(m, x);
    if (n_top) enter(top, in ? make_key(x, j0 + lane) : kNoKey, n_top, lane);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  bad = __any_sync(0xffffffffu, bad) || m == -INFINITY;
  float l = 0.0f, s = 0.0f;
  for (int j = lane; j < vocab && !bad; j += 32) {
    const float d = (load(j) - m) * to_log2, e = ex2(d);
    l += e;
    s = fmaf(e, fmaxf(d, -1000.0f), s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    l += __shfl_xor_sync(0xffffffffu, l, o);
    s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  Norm n = {m, inv_temp, logf(l), logf(l) - 0.6931471805599453f * (s / l), top.mine};
  if (bad) n.at = n.entropy = NAN;
  return n;
}

// A row's results from its joined sums (those of lane 0) and list; one warp.
template <int LT>
__device__ __forceinline__ void finish(const LpParams& p, int t, Sums z, const Top& top, int lane) {
  // the same in all lanes: the branch below is taken by the warp as one
  z.m = __shfl_sync(0xffffffffu, z.m, 0);
  z.l = __shfl_sync(0xffffffffu, z.l, 0);
  z.s = __shfl_sync(0xffffffffu, z.s, 0);
  const int64_t row = (int64_t)t * p.a.token_stride;
  const void* logits = p.a.logits;
  const int64_t stride = p.a.vocab_stride;
  auto load = [logits, row, stride](int j) {
    const int64_t at = row + (int64_t)j * stride;
    return LT == FP8IMMA_L_F32 ? __ldg(static_cast<const float*>(logits) + at) : to_f32<LT>(__ldg(static_cast<const uint16_t*>(logits) + at));
  };
  const int id = __ldg(p.a.token_ids + t);
  const bool known = (unsigned)id < (unsigned)p.a.vocab;
  const float x = known ? load(id) : NAN;
  Norm n = {z.m, p.inv_temp, 0.6931471805599453f * log2f(z.l), 0.6931471805599453f * (log2f(z.l) - z.s / z.l), top.mine};
  if (!(z.l > 0.0f && z.l < INFINITY)) n = careful<LT>(p.a.vocab, p.a.top, p.to_log2, p.inv_temp, load, lane);
  if (lane == 0) {
    p.a.logprobs[t] = fmaf(x - n.at, n.inv, -n.ln_l);
    p.a.entropy[t] = n.entropy;
  }
  if (lane < p.a.top) {
    p.a.top_ids[(int64_t)t * p.a.top + lane] = key_index(n.mine);
    p.a.top_logprobs[(int64_t)t * p.a.top + lane] = fmaf(key_value(n.mine) - n.at, n.inv, -n.ln_l);
  }
}

// This CTA came last to `counter` (all of its threads call; its results are in
// global memory).
__device__ __forceinline__ bool came_last(unsigned int* counter, int parts) {
  __shared__ int s_last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned int prev;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(prev) : "l"(counter) : "memory");
    s_last = prev == (unsigned)(parts - 1);
    if (s_last) *counter = 0;  // ready for the next call
  }
  __syncthreads();
  __threadfence();
  return s_last != 0;
}

__device__ __forceinline__ void put_part(const LpParams& p, int part, int t, const Sums& z, const Top& top, int lane) {
  const int64_t at = (int64_t)part * p.a.tokens + t;
  if (lane == 0) *reinterpret_cast<float4*>(p.sums + at * 4) = make_float4(z.m, z.l, z.s, 0.0f);
  if (p.a.top) p.lists[at * 32 + lane] = top.mine;
}
// Sums of the parts first, first + stride, ... of token t, joined in this order
// 32 at a time.
__device__ __forceinline__ Sums get_sums(const LpParams& p, int first, int stride, int t, int lane) {
  Sums z;
  for (int k = first + lane * stride; k < p.parts; k += 32 * stride) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(p.sums + ((int64_t)k * p.a.tokens + t) * 4));
    z.join(v.x, v.y, v.z, p.to_log2);
  }
  z.warp_join(p.to_log2);
  return z;
}
// Their lists merged, the next one under way.
__device__ __forceinline__ Top get_lists(const LpParams& p, int first, int stride, int t, int lane) {
  Top l;
  auto load = [&](int k) { return k < p.parts ? __ldcg(p.lists + ((int64_t)k * p.a.tokens + t) * 32 + lane) : kNoKey; };
  unsigned long long next = load(first);
#pragma unroll 1
  for (int k = first; k < p.parts; k += stride) {
    const unsigned long long v = next;
    next = load(k + stride);
    l.mine = merge(l.mine, v, lane);
  }
  return l;
}
// The same for all parts by one warp where there are at least `top` of them
// (and kMostParts at most): no key below the top-th largest of their heads
// belongs to the row's list, so a lane follows the lists of its parts only as
// far as that.
constexpr int kMostParts = 96;
__device__ __noinline__ Top get_heads(const unsigned long long* lists, int64_t stride, int parts, unsigned long long* buf, int top, int lane) {
  unsigned long long h[kMostParts / 32];
#pragma unroll
  for (int e = 0; e < kMostParts / 32; ++e) h[e] = lane + 32 * e < parts ? __ldcg(lists + (lane + 32 * e) * stride) : kNoKey;
#pragma unroll
  for (int e = 0; e < kMostParts / 32; ++e) buf[lane + 32 * e] = h[e];
  const unsigned long long least = flush(Top(), buf, parts, top, lane).last;
  Top l;
  for (int d = 1;; ++d) {
    int n = 0;
#pragma unroll
    for (int e = 0; e < kMostParts / 32; ++e) {
      const bool in = h[e] != kNoKey && h[e] >= least;
      const unsigned m = __ballot_sync(0xffffffffu, in);
      if (in) buf[n + __popc(m & ((1u << lane) - 1u))] = h[e];
      n += __popc(m);
      h[e] = in && d < top ? __ldcg(lists + (lane + 32 * e) * stride + d) : kNoKey;
    }
    if (n == 0) return l;
    l = flush(l, buf, n, top, lane);
  }
}

// Largest logit of a 16-byte vector's 32-bit words, packed.
template <int LT>
__device__ __forceinline__ uint32_t max_words(uint32_t a, uint32_t b) {
  if (LT == FP8IMMA_L_F32) return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  uint32_t r;
  if (LT == FP8IMMA_L_F16) asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int LT>
__device__ __forceinline__ float max_of_word(uint32_t a) {
  if (LT == FP8IMMA_L_F32) return __uint_as_float(a);
  return fmaxf(to_f32<LT>(a & 0xFFFFu), to_f32<LT>(a >> 16));
}
template <int LT>
__device__ __forceinline__ float logit_of(const uint4& q, int i) {  // i: a constant
  const uint32_t w = LT == FP8IMMA_L_F32 ? (i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w) : (i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w);
  return LT == FP8IMMA_L_F32 ? __uint_as_float(w) : to_f32<LT>(i & 1 ? w >> 16 : w & 0xFFFFu);
}
// One logit a lane into the buffer where it may enter the list (`in`); the
// buffer's new length, the same in all lanes like the old one.
__device__ __forceinline__ int put(float x, bool in, unsigned long long* buf, int n, int j, int lane) {
  const unsigned m = __ballot_sync(0xffffffffu, in);
  if (m) {
    if (in) buf[n + __popc(m & ((1u << lane) - 1u))] = make_key(x, j);
    n += __popc(m);
  }
  return n;
}
// The same for a vector's logits; the lane's first has index j.
template <int LT>
__device__ __noinline__ int gather(uint4 q, float bar, bool in, unsigned long long* buf, int n, int j, int lane) {
#pragma unroll
  for (int i = 0; i < (LT == FP8IMMA_L_F32 ? 4 : 8); ++i) {
    const float x = logit_of<LT>(q, i);
    n = put(x, in && x >= bar, buf, n, j + i, lane);
  }
  return n;
}
template <int LT>
__device__ __forceinline__ float max_of(const uint4& q) {
  return max_of_word<LT>(max_words<LT>(max_words<LT>(q.x, q.y), max_words<LT>(q.z, q.w)));
}
// The lane's logits of four vectors that may enter the list, into the buffer,
// as few lanes have one: each finds its place by an atomic count, and what does
// not fit is counted only (the caller then goes vector by vector).
struct Quad {
  uint4 q[4];
};
template <int LT>
__device__ __noinline__ void gather(Quad v, float bar, unsigned long long* buf, unsigned int* count, int j, int stride, int valid) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k >= valid || !(max_of<LT>(v.q[k]) >= bar)) continue;
#pragma unroll
    for (int i = 0; i < (LT == FP8IMMA_L_F32 ? 4 : 8); ++i) {
      const float x = logit_of<LT>(v.q[k], i);
      if (x >= bar) {
        const unsigned at = atomicAdd(count, 1u);
        if (at < kBuffer) buf[at] = make_key(x, j + k * stride + i);
      }
    }
  }
}

// A CTA's sums and lists (one a warp) joined in the first warp, the sums in its
// lane 0: pairs of warps in a fixed order.
template <int kWarps>
__device__ __forceinline__ void join_warps(Sums& z, Top& list, float (*sums)[3], unsigned long long (*lists)[32], float c, bool top, int warp, int lane) {
  if (lane == 0) {
    sums[warp][0] = z.m;
    sums[warp][1] = z.l;
    sums[warp][2] = z.s;
  }
  if (top) lists[warp][lane] = list.mine;
  __syncthreads();
  if (top) {
#pragma unroll 1
    for (int half = kWarps / 2; half > 0; half >>= 1) {
      if (warp < half) {
        list.mine = merge(list.mine, lists[warp + half][lane], lane);
        if (half > 1) lists[warp][lane] = list.mine;
      }
      if (half > 1) __syncthreads();
    }
  }
  if (warp == 0) {
    z = Sums();
    if (lane < kWarps) {
      z.m = sums[lane][0];
      z.l = sums[lane][1];
      z.s = sums[lane][2];
    }
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, z.m, o), l2 = __shfl_xor_sync(0xffffffffu, z.l, o), s2 = __shfl_xor_sync(0xffffffffu, z.s, o);
      z.join(m2, l2, s2, c);
    }
  }
}

// Row-major logits: CTA (part, token); the warps take runs of 32 16-byte
// vectors of the part in turn, four at a time. Rows lie at any alignment:
// vectors start at 16-byte boundaries, what lies before the first and behind
// the last whole vector is read one logit a lane. The warps share the value
// that the row's top logits are known to reach, so that one warp's finds spare
// the others theirs.
template <int LT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, 32 / kWarps) logprobs_row_kernel(const __grid_constant__ LpParams p) {
  constexpr int kVec = LT == FP8IMMA_L_F32 ? 4 : 8, kSize = LT == FP8IMMA_L_F32 ? 4 : 2, kAhead = 4, kThreads = kWarps * 32;
  constexpr uint32_t kNone = LT == FP8IMMA_L_F32 ? 0xFF800000u : LT == FP8IMMA_L_BF16 ? 0xFF80FF80u : 0xFC00FC00u;  // -inf
  __shared__ float s_sums[kWarps][3];
  __shared__ unsigned long long s_list[kWarps][32];
  __shared__ unsigned long long s_buf[kWarps][kBuffer];
  __shared__ unsigned int s_floor, s_count[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) s_floor = 0u;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  const int part = blockIdx.x, V = p.a.vocab, top = p.a.top;
  const float c = p.to_log2;
  unsigned long long* const buf = s_buf[warp];
  for (int t = blockIdx.y; t < p.a.tokens; t += gridDim.y) {
    const char* row = static_cast<const char*>(p.a.logits) + (int64_t)t * p.a.token_stride * kSize;
    const int lead = min(V, (int)((16u - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / kSize);  // logits before the first whole vector
    const int vecs = (V - lead) / kVec;
    const int v0 = min(vecs, part * p.per_part), v1 = part == p.parts - 1 ? vecs : min(vecs, v0 + p.per_part);
    const uint4* base = reinterpret_cast<const uint4*>(row + lead * kSize);
    Sums z;
    Top list;
    float bar = top ? -INFINITY : INFINITY;
    bool fresh = true;  // no bar yet
    int n = 0;          // gathered
    auto end = [&](int j) {  // one logit a lane from an end of the row (j < 0: none)
      float x = -INFINITY;
      if (j >= 0) x = LT == FP8IMMA_L_F32 ? __ldg(reinterpret_cast<const float*>(row) + j) : to_f32<LT>(__ldg(reinterpret_cast<const unsigned short*>(row) + j));
      z.follow(x, c);
      z.add(x, c);
      if (top) n = put(x, j >= 0 && x >= bar, buf, n, j, lane);
    };
    // the list takes equal logits in the order of their indexes: the head first, the tail last
    if (warp == 0 && part == 0) end(lane < lead ? lane : -1);
#pragma unroll 1
    for (int vb = v0 + warp * 32; vb < v1; vb += kThreads * kAhead) {  // warp-uniform
      Quad quad;
      uint4 (&q)[kAhead] = quad.q;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int v = vb + lane + k * kThreads;
        q[k] = make_uint4(kNone, kNone, kNone, kNone);
        if (v < v1) q[k] = __ldg(base + v);
      }
      uint32_t w = kNone;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) w = max_words<LT>(w, max_words<LT>(max_words<LT>(q[k].x, q[k].y), max_words<LT>(q[k].z, q[k].w)));
      const float big = max_of_word<LT>(w);
      if (top) {
        if (fresh) bar = fmaxf(bar, first_bar(big, top, lane));  // what the top-th of the lanes' largest reaches
        else if (kWarps > 1) bar = fmaxf(bar, enters_at(Top(), *(volatile unsigned int*)&s_floor));
        fresh = false;
      }
      z.follow(big, c);
      Pair two(z, c);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (k == 0 || vb + k * kThreads < v1) {
#pragma unroll
          for (int i = 0; i < kVec; i += 2) two.add(logit_of<LT>(q[k], i), logit_of<LT>(q[k], i + 1));
        }
      two.fold(z);
      if (top && __any_sync(0xffffffffu, big >= bar)) {
        if (lane == 0) s_count[warp] = n;
        __syncwarp();
        if (big >= bar) gather<LT>(quad, bar, buf, &s_count[warp], lead + (vb + lane) * kVec, kThreads * kVec, (v1 - vb - lane + kThreads - 1) / kThreads);
        __syncwarp();
        const int found = *(volatile unsigned int*)&s_count[warp];
        bool flushed = false;
        if (found <= kBuffer) {
          n = found;
          flushed = n >= p.flush_at;
          if (flushed) list = flush(list, buf, n, top, lane);
        } else {  // equal logits everywhere, or a row that rises
#pragma unroll 1
          for (int k = 0; k < kAhead; ++k) {
            const int v = vb + lane + k * kThreads;
            const uint4 qk = k == 0 ? q[0] : k == 1 ? q[1] : k == 2 ? q[2] : q[3];
            n = gather<LT>(qk, bar, v < v1, buf, n, lead + v * kVec, lane);
            list = flush(list, buf, n, top, lane);
            n = 0;
          }
          flushed = true;
        }
        if (flushed) {
          n = 0;
          bar = fmaxf(bar, enters_at(list, 0u));
          if (kWarps > 1 && lane == 0) atomicMax(&s_floor, (unsigned)(list.last >> 32));
        }
      }
    }
    if (warp == 0 && part == p.parts - 1) {
      const int j = lead + vecs * kVec + lane;
      end(j < V ? j : -1);
    }
    if (top) list = flush(list, buf, n, top, lane);
    z.warp_join(c);
    join_warps<kWarps>(z, list, s_sums, s_list, c, top > 0, warp, lane);
    if (threadIdx.x == 0) s_floor = 0u;
    if (warp == 0) {
      if (p.parts == 1) finish<LT>(p, t, z, list, lane);
      else put_part(p, part, t, z, list, lane);
    }
    if (p.parts > 1 && came_last(p.counters + t, p.parts)) {  // the warps join every so many parts each, then theirs
      Sums all = get_sums(p, warp, kWarps, t, lane);
      Top l;
      if (top) l = get_lists(p, warp, kWarps, t, lane);
      join_warps<kWarps>(all, l, s_sums, s_list, c, top > 0, warp, lane);
      if (warp == 0) finish<LT>(p, t, all, l, lane);
    }
    __syncthreads();  // shared memory is free for the next row
  }
}

// Column-major logits (the GEMM's default output): CTA (part, group of up to
// p.group tokens). Tiles of kTile vocabulary rows go through shared memory,
// whose rows are padded so that a warp then reads a token's column without
// conflicts; the next tile is under way meanwhile. A warp keeps up to two
// tokens.
constexpr int kTile = 256;  // 128 of fp32
template <int LT>
__global__ void __launch_bounds__(kColWarps * 32, 4) logprobs_col_kernel(const __grid_constant__ LpParams p) {
  using Word = typename std::conditional<LT == FP8IMMA_L_F32, uint32_t, uint16_t>::type;
  constexpr int kWarps = kColWarps, kThreads = kColWarps * 32, kPitch = LT == FP8IMMA_L_F32 ? 9 : 18, kVec = 16 / sizeof(Word);
  constexpr int kRows = LT == FP8IMMA_L_F32 ? kTile / 2 : kTile, kEach = kRows / 32;  // rows of a tile, of a lane
  constexpr int kAhead = kRows * (LT == FP8IMMA_L_F32 ? 8 : 16) / kVec / kThreads;  // 16-byte pieces of a tile a thread
  __shared__ __align__(16) Word s_tile[kRows * kPitch];
  __shared__ unsigned long long s_buf[kWarps][kBuffer];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int part = blockIdx.x, V = p.a.vocab, top = p.a.top;
  const float c = p.to_log2;
  unsigned long long* const buf = s_buf[warp];
  for (int group = blockIdx.y; group < p.groups; group += gridDim.y) {
    const int t0 = group * p.group, n = min(p.group, p.a.tokens - t0);
    const int j0 = part * p.per_part, j1 = min(V, j0 + p.per_part);
    const Word* src = static_cast<const Word*>(p.a.logits) + t0;
    const bool vec = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t)(p.a.vocab_stride * sizeof(Word)) | (uintptr_t)(n * sizeof(Word))) & 15u) == 0;
    const int per = n / kVec;
    Sums z[2];
    Top list[2];
    uint4 next[kAhead];
    auto fetch = [&](int jt) {
      const int rows = min(kRows, j1 - jt);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int x = tid + k * kThreads, r = x / per, q = x - r * per;
        if (x < rows * per) next[k] = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)(jt + r) * p.a.vocab_stride + q * kVec));
      }
    };
    if (vec && j0 < j1) fetch(j0);
    for (int jt = j0; jt < j1; jt += kRows) {
      const int rows = min(kRows, j1 - jt);
      __syncthreads();  // the tile before has been read
      if (vec) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int x = tid + k * kThreads, r = x / per, q = x - r * per;
          if (x < rows * per) {
            uint32_t* dst = reinterpret_cast<uint32_t*>(&s_tile[r * kPitch + q * kVec]);  // even pitch for 16-bit words
            dst[0] = next[k].x;
            dst[1] = next[k].y;
            dst[2] = next[k].z;
            dst[3] = next[k].w;
          }
        }
        if (jt + kRows < j1) fetch(jt + kRows);
      } else {
#pragma unroll 8
        for (int x = tid; x < rows * n; x += kThreads) {
          const int r = x / n, q = x - r * n;
          s_tile[r * kPitch + q] = __ldg(src + (int64_t)(jt + r) * p.a.vocab_stride + q);
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int t = warp + k * kWarps;
        if (t >= n) break;
        float x[kEach];  // the lane's logits of the tile
#pragma unroll
        for (int i = 0; i < kEach; ++i) x[i] = i * 32 + lane < rows ? to_f32<LT>(s_tile[(i * 32 + lane) * kPitch + t]) : -INFINITY;
        float big = x[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) big = fmaxf(big, x[i]);
        z[k].follow(big, c);
#pragma unroll
        for (int i = 0; i < kEach; ++i) z[k].add(x[i], c);
        if (top) {
          float bar = enters_at(list[k], 0u);
          if (jt == j0) bar = fmaxf(bar, first_bar(big, top, lane));
          if (__any_sync(0xffffffffu, big >= bar)) {
            int m = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) m = put(x[i], x[i] >= bar && i * 32 + lane < rows, buf, m, jt + i * 32 + lane, lane);
            list[k] = flush(list[k], buf, m, top, lane);
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int t = warp + k * kWarps;
      if (t >= n) break;
      z[k].warp_join(c);
      if (p.parts == 1) finish<LT>(p, t0 + t, z[k], list[k], lane);
      else put_part(p, part, t0 + t, z[k], list[k], lane);
    }
    if (p.parts > 1 && came_last(p.counters + group, p.parts)) {
      for (int t = warp; t < n; t += kWarps) {
        const Sums all = get_sums(p, 0, 1, t0 + t, lane);
        Top l;
        if (top && p.parts >= top && p.parts <= kMostParts)
          l = get_heads(p.lists + (int64_t)(t0 + t) * 32, (int64_t)p.a.tokens * 32, p.parts, buf, top, lane);
        else if (top)
          l = get_lists(p, 0, 1, t0 + t, lane);
        finish<LT>(p, t0 + t, all, l, lane);
      }
    }
  }
}

template <int LT>
cudaError_t launch(LpParams& p, cudaStream_t st) {
  const bool rows = p.a.vocab_stride == 1;
  const int sms = num_sms_current();
  p.flush_at = p.a.top >= 16 ? 32 : p.a.top >= 8 ? 16 : 8;
  const int vec = LT == FP8IMMA_L_F32 ? 4 : 8;
  // Parts: enough CTAs for two (row-major: four resident) on each SM, but no
  // part below the logits that make joining it worth while.
  int warps = 8;  // of a row's CTA
  int units, full;  // units: rows or groups; full: pieces of a row that a part is made of
  if (rows) {
    units = p.a.tokens;
    full = (p.a.vocab + vec - 1) / vec;
    const int64_t want = (4ll * sms + units - 1) / units, most = (full + 255) / 256;
    p.parts = (int)std::max<int64_t>(1, std::min(want, most));
    if (units >= 2 * sms) p.parts = 1;
    // Each warp keeps a list of its own, so with many rows fewer warps a row
    // cost less (4096 rows of 32001, 5 alternatives: 1 warp 91 us, 8 warps 136
    // us), with few rows more warps fill the SMs (700 rows: 48 and 32 us).
    while (warps > 1 && (int64_t)units * warps > 48ll * sms) warps /= 2;
  } else {
    // groups of 8 tokens, one a warp; of 16 with 16-bit logits and many tokens,
    // for whole 32-byte sectors
    p.group = p.a.tokens <= 64 || LT == FP8IMMA_L_F32 ? 8 : 16;
    units = p.groups = (p.a.tokens + p.group - 1) / p.group;
    full = p.a.vocab;
    // At most 74 parts. Each finds its own bar and leaves a list, so more of them
    // sort more; above kMostParts their lists are merged one by one. 16 rows of
    // 128000 with 37, 74, 148 parts: 44, 32, 61 us with 20 alternatives, 16, 12, 11
    // without; 4 rows 48, 33, 59 and 22, 13.5, 10.
    const int64_t want = std::max<int64_t>(1, 4ll * sms / units), most = (full + kTile - 1) / kTile;
    p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 74));
  }
  p.per_part = (full + p.parts - 1) / p.parts;
  if (rows) p.per_part = (p.per_part + 31) & ~31;
  p.parts = (full + p.per_part - 1) / p.per_part;  // the last part of a row takes what is left of it
  ScopedScratch ctr, work;
  cudaError_t e = cudaSuccess;
  if (p.parts > 1) {
    const size_t at = (size_t)p.parts * p.a.tokens;
    e = ctr.get((size_t)units * 4, st, kScratchLogprobsSync);
    if (e == cudaSuccess && ctr.owned) e = cudaMemsetAsync(ctr.ptr, 0, (size_t)units * 4, st);
    if (e == cudaSuccess) e = work.get(at * (16 + 256), st, kScratchLogprobs);
    p.counters = static_cast<unsigned int*>(ctr.ptr);
    p.lists = static_cast<unsigned long long*>(work.ptr);
    p.sums = reinterpret_cast<float*>(static_cast<char*>(work.ptr) + at * 256);
  }
  if (e == cudaSuccess) {
    cudaLaunchConfig_t lc = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.gridDim = dim3(p.parts, std::min(units, 65535));
    lc.blockDim = dim3(rows ? 32 * warps : kColWarps * 32);
    lc.stream = st;
    lc.attrs = attr;
    lc.numAttrs = api_pdl() ? 1 : 0;
    e = !rows        ? cudaLaunchKernelEx(&lc, logprobs_col_kernel<LT>, p)
        : warps == 8 ? cudaLaunchKernelEx(&lc, logprobs_row_kernel<LT, 8>, p)
        : warps == 4 ? cudaLaunchKernelEx(&lc, logprobs_row_kernel<LT, 4>, p)
        : warps == 2 ? cudaLaunchKernelEx(&lc, logprobs_row_kernel<LT, 2>, p)
                     : cudaLaunchKernelEx(&lc, logprobs_row_kernel<LT, 1>, p);
  }
  const cudaError_t e1 = ctr.release(st), e2 = work.release(st);
  return e != cudaSuccess ? e : e1 != cudaSuccess ? e1 : e2;
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
  if (a->vocab > 0x7fffff00) return (int)cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(a->logits) & (a->l_type == FP8IMMA_L_F32 ? 3u : 1u)) return (int)cudaErrorInvalidValue;
  if (!aligned4({a->token_ids, a->logprobs, a->entropy}) || (a->top > 0 && !aligned4({a->top_ids, a->top_logprobs}))) return (int)cudaErrorInvalidValue;
  LpParams p = {};
  p.a = *a;
  p.inv_temp = 1.0f / a->temperature;
  p.to_log2 = 1.4426950408889634f * p.inv_temp;
  if (!(p.to_log2 < INFINITY)) return (int)cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->l_type == FP8IMMA_L_F16) return (int)launch<FP8IMMA_L_F16>(p, st);
  if (a->l_type == FP8IMMA_L_BF16) return (int)launch<FP8IMMA_L_BF16>(p, st);
  return (int)launch<FP8IMMA_L_F32>(p, st);
}
