// Attention over the paged 8-bit KV cache for many query rows a KV head
// (drafts to verify, prompts, wide groups of heads), products by tcgen05.
// Mathematics and the cut of the work are those of kv_attention.cu; a tile here
// is 128 query rows x 128 keys.
//
// Bound: with R rows a key costs 4 R D flops, and the few-row kernel converts
// every FP8 code once for each 8 or 16 rows that a warp multiplies it with; from
// about 32 rows on that conversion, not the copy, is its time. Here a code is
// converted once for up to 128 rows:
//  * the load warps copy the codes asynchronously (16 bytes a thread), 1 tile
//    ahead at 128 channels and 3 at 64, and write them as fp16 the way the tensor
//    core reads them (K rows, V transposed, both K-major with 128-byte swizzle);
//    each thread converts what it has copied, so that the copies need no barrier;
//  * one thread issues S = Q K^T (accumulators in TMEM) and O += P V, with P
//    read from TMEM;
//  * two groups of four softmax warps, one thread a row, take tiles in turn:
//    while one computes P of its tile, the tensor core makes the other's S.
// Each group keeps a running reference, sum and O of its own (TMEM: 2 x 128
// columns of S, which P overwrites, 2 x D of O); they are joined where a run
// leaves an item. V's channels lie permuted in shared memory (row c D/16 + col
// for channel 16 col + c), which spreads the transposing stores over the banks;
// O's columns come out in that order. K is held once, V twice: K is free again
// as soon as its scores are made.
//
// Measured (e4m3, fp16): 16 sequences of 8000 keys, 64 heads over 8, 128
// channels, 32 rows a KV head 125 us (2.1 TB/s), 128 rows 137 us (493 us in the
// few-row kernel); prompts of 4 x 1000 tokens, 32 heads over 8, 220 us (576);
// one of 8192 tokens 1.73 ms (7.26; 318 TFLOP/s of the causal half). What bounds
// it are the latencies of instruction issue (4.2 warps a scheduler, 0.43
// instructions a cycle, the tensor pipe 21% of the time): a tile takes some 4000
// cycles, of which its products need about 900. Loads through registers instead
// of shared memory waited for each other: 221 us where this took 121.
#include "kv_attention.cuh"
#include "sm100_umma.cuh"
#include <type_traits>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;
using namespace attn;

constexpr int kRows = 128;
constexpr int kSoftWarps = 8, kSoft = kSoftWarps * 32;

template <int D>
struct Shape {
  static constexpr int kLoadWarps = D / 16, kLoad = kLoadWarps * 32;
  static constexpr int kThreads = kSoft + kLoad + 32;
  static constexpr int kTile = kKeys * D * 2;             // fp16 bytes of K, of V, of Q
  static constexpr int kSlot = 2 * kKeys * D;             // FP8 codes of a tile
  static constexpr int kSlots = D == 64 ? 4 : 2;
  static constexpr int kPoison = kRows * D;               // 4 bits a channel, two groups
  static constexpr int kSmem = 1024 + 4 * kTile + kSlots * kSlot + kPoison;
  static constexpr int kPartFloats = kRows * D + kRows * 2;
  static constexpr int kCols = D / 16;                    // 16-channel columns
  static constexpr uint32_t kTmemS = 0, kTmemO = 2 * kKeys;  // TMEM columns of the two groups' S and O
};

// Copies of 16 and of 4 bytes, zeros where `on` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
// The word at p, or -1. The predicate sits in the asm: a branch around the load
// would end in a copy of its result, which waits for it.
__device__ __forceinline__ int ldg_if(const int* p, bool on) {
  int r = -1;
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.global.nc.u32 %0, [%1];\n\t}" : "+r"(r) : "l"(p), "r"((int)on));
  return r;
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// fp16 x fp16 -> fp32, K-major operands
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
               : "memory");
}
// a load that has to be waited for before r is read
__device__ __forceinline__ void tmem_ld16_start(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {  // r passes through, so that no use moves ahead
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two 32-bit values in one operation
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// two fp16 values times a power of two
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t x, float f) {
  const uint32_t f2 = pack_f16(f, f);
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(f2));
  return r;
}

struct TileInfo {
  float ks[8], lv[8], iv[8];  // by groups of 16 keys: K's scale, log2 of V's (-infinity: no page), 1 / V's
  int live;                   // a bit a group, and eight more: live, with a K scale that is not negative
  int odd[8];   // a load warp found non-finite values that some row may not see
};

// The tiles of a segment that some row sees.
__device__ __forceinline__ void tiles_of(const Walk& w, const Segment& g, int& from, int& to) {
  const int lo = w.s.tile0 + g.first;
  from = max(lo, g.lo / kKeys);
  to = min(lo + g.count, (g.hi + kKeys - 1) / kKeys);
}
// Some row of the segment does not see some key of the tile.
__device__ __forceinline__ bool edge_tile(const AttnParams& p, const Segment& g, int tile) {
  const int j0 = tile * kKeys, j1 = j0 + kKeys - 1;
  return j1 > g.pos_min || j1 >= g.hi || (p.a.window > 0 && j0 <= g.pos_max - p.a.window);
}

template <int FMT, int D>
__global__ void __launch_bounds__(Shape<D>::kThreads, 1) kv_attention_tc_kernel(const __grid_constant__ AttnParams p) {
  using S = Shape<D>;
  extern __shared__ uint8_t smem_raw[];
  // Tiles take their barriers in turn: K's (which s_info follows) by tile number
  // mod 4, the others mod 2. A phase of a barrier ends only after all that wait
  // for the one before it have passed: for V, S, P and O through the tile's
  // product with P, two tiles back; for K, whose place is free as soon as its
  // scores are made, through that product four tiles back.
  __shared__ uint64_t s_k_full[4], s_v_full[2], s_s_full[2], s_p_full[2], s_pv_done[2], s_q_full, s_o_free;
  __shared__ float s_scales[S::kSlots][16];
  __shared__ TileInfo s_info[4];       // by tile number mod 4: when a place is filled again, its last tile has been multiplied
  __shared__ Shared s_shared[2];
  __shared__ float s_ml[2][kRows][3];  // reference, sum, whether the group's poison marks count
  __shared__ float s_back[kRows];      // what a bf16 row of Q was divided by
  __shared__ int s_n_shared;
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* const base = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  uint8_t* const q_tile = base;
  uint8_t* const k_tile = base + S::kTile;
  auto v_tile = [&](int g) { return base + S::kTile * (2 + g); };
  uint8_t* const slots = base + 4 * S::kTile;
  uint8_t* const poison = slots + S::kSlots * S::kSlot;
  constexpr int kMmaWarp = kSoftWarps + S::kLoadWarps;

  if (tid == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(&s_k_full[i], S::kLoad);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_v_full[i], S::kLoad);
      mbar_init(&s_s_full[i], 1);
      mbar_init(&s_p_full[i], kSoft / 2);
      mbar_init(&s_pv_done[i], 1);
    }
    mbar_init(&s_q_full, kSoft);
    mbar_init(&s_o_free, kSoft);
    fence_barrier_init();
    s_n_shared = 0;
  }
  pdl_launch_dependents();
  pdl_wait();
  Walk walk;
  int units, ctas;
  if (!find_run<S::kThreads>(p, kRows, walk, units, ctas)) return;
  const Runs runs(units, ctas);
  if (warp == kMmaWarp) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  Segment seg;
  bool ok = true;  // false: a wait ran out, the rest is walked through without waiting
  auto wait = [&](uint64_t* bar, int use) {
    if (ok) ok = mbar_wait<true>(bar, (uint32_t)(use & 1), ERR_WAIT_FULL);
  };

  if (warp >= kSoftWarps && warp < kMmaWarp) {
    // ------------------------------------------------------------- loads --
    // Each thread converts the pieces that it has copied itself, so that the
    // slots need no barrier.
    const int t = tid - kSoft, ps = p.c.page_size;
    const int k_row = t / S::kCols, col = t % S::kCols;  // pieces of K: rows k_row + 32 i
    // V: four keys from 4 quad on. For 64 channels the lanes' quads are spread so that their stores fall on all banks.
    const int quad = D == 128 ? t / 8 : ((t >> 2) & 1) + 2 * (((t >> 3) & 1) + 2 * ((t >> 5) & 1) + 4 * ((t >> 4) & 1)) + 16 * (t >> 6);
    const uint32_t slot0 = smem_u32(slots) + t * 16;
    int tile = 0, to = 0, id = -1, issued = 0;
    uint32_t live_bits = 0, edge_bits = 0;  // by slot
    const int ps_log = __ffs(ps) - 1;
    bool more = true;
    // On to the next tile, and the page of its 16-key group `lane` (lanes 0 .. 7),
    // -1: none that any row sees. The load stands outside all branches: where
    // paths join, its result would be waited for.
    auto next = [&]() {
      if (++tile >= to) {
        do {
          more = walk.next(p, kRows, seg);
          if (more) tiles_of(walk, seg, tile, to);
        } while (more && tile >= to);
      }
      const int j0 = tile * kKeys + lane * 16, pi = j0 >> ps_log;
      id = ldg_if(p.c.page_table + (size_t)seg.b * p.c.max_pages + pi, more && lane < 8 && j0 < seg.hi && j0 + 15 >= seg.lo && pi < p.c.max_pages);
    };
    next();
    auto issue = [&]() {  // the copies of the next tile
      const int slot = issued % S::kSlots;
      const bool live = (unsigned)id < (unsigned)p.c.num_pages;
      const uint32_t at = slot0 + slot * S::kSlot;
      // row of the pools where the group's keys begin, -1: no page
      const int begin = live ? ((id * p.c.kv_heads + seg.h) << ps_log) + ((tile * kKeys + lane * 16) & (ps - 1)) : -1;
      auto piece = [&](const void* pool, int first, int row, uint32_t dst) {  // 16 codes of a key
        const int j = tile * kKeys + row;
        const bool on = first >= 0 && j < seg.hi && j >= seg.lo;
        copy16(dst, static_cast<const uint8_t*>(pool) + ((int64_t)(on ? first + (row & 15) : 0) * D + col * 16), on);
      };
      if (more) {
#pragma unroll
        for (int i = 0; i < 4; ++i) piece(p.c.k, __shfl_sync(0xffffffffu, begin, (k_row + 32 * i) >> 4), k_row + 32 * i, at + i * (S::kLoad * 16));
        const int first = __shfl_sync(0xffffffffu, begin, quad >> 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) piece(p.c.v, first, quad * 4 + e, at + (4 + e) * (S::kLoad * 16));
        if (t < 8) {
          const int64_t ph = live ? (int64_t)id * p.c.kv_heads + seg.h : 0;
          copy4(smem_u32(&s_scales[slot][t]), p.c.k_scale + ph, live);
          copy4(smem_u32(&s_scales[slot][8 + t]), p.c.v_scale + ph, live);
        }
        live_bits = (live_bits & ~(1u << slot)) | ((uint32_t)live << slot);
        edge_bits = (edge_bits & ~(1u << slot)) | ((uint32_t)edge_tile(p, seg, tile) << slot);
        ++issued;
      }
      next();
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < S::kSlots - 1; ++i) issue();
#pragma unroll 1
    for (int idx = 0; idx < issued; ++idx) {
      issue();
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kSlots - 1) : "memory");
      const int g = idx & 1, slot = idx % S::kSlots;
      const bool edge = (edge_bits >> slot) & 1;
      const uint8_t* const src = slots + slot * S::kSlot + t * 16;
      if (idx > 0) wait(&s_s_full[g ^ 1], (idx - 1) >> 1);  // the tile before has been multiplied with Q
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = k_row + 32 * i;
        uint8_t* dst = k_tile + (col >> 2) * (kKeys * 128) + row * 128;
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // the upper columns begin with their second half, so that the stores fall on all banks
          const int half = h ^ (col >> 2);
          const uint2 x = *reinterpret_cast<const uint2*>(src + i * (S::kLoad * 16) + half * 8);
          uint4 y;
          f8x4_to_f16x4<FMT>(x.x, y.x, y.y);
          f8x4_to_f16x4<FMT>(x.y, y.z, y.w);
          *reinterpret_cast<uint4*>(dst + ((((col & 3) * 2 + half) ^ (row & 7)) << 4)) = y;
        }
      }
      if (t < 8) {
        const bool live = (live_bits >> slot) & 1;
        const float vs = fmaxf(s_scales[slot][8 + t], kTinyScale);
        const unsigned all = __ballot_sync(0xffu, live), plain = __ballot_sync(0xffu, live && s_scales[slot][t] >= 0.0f);
        s_info[idx & 3].ks[t] = s_scales[slot][t];
        s_info[idx & 3].lv[t] = live ? lg2(vs) : -INFINITY;
        s_info[idx & 3].iv[t] = __fdividef(1.0f, vs);
        if (t == 0) s_info[idx & 3].live = (int)(all | plain << 8);
      }
      fence_proxy_async_shared();
      mbar_arrive(&s_k_full[idx & 3]);
      if (idx > 1) wait(&s_pv_done[g], (idx >> 1) - 1);  // the tile that lay here before has been multiplied with P
      bool odd = false;
      uint32_t w[4][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint4 x = *reinterpret_cast<const uint4*>(src + (4 + e) * (S::kLoad * 16));
        w[e][0] = x.x, w[e][1] = x.y, w[e][2] = x.z, w[e][3] = x.w;
      }
      if (edge) {
        // 0 * NaN must not reach the rows that do not see the key: such values are left out here and marked below
        const uint32_t mk = FMT == F8_E4M3 ? 0x7F7F7F7Fu : 0x7C7C7C7Cu;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t bad = __vcmpeq4(w[e][k] & mk, mk);
            odd |= bad != 0u;
            w[e][k] &= ~bad;
          }
      }
      uint8_t* const dst = v_tile(g) + (quad >> 4) * (D * 128) + (quad & 1) * 8;
      const int chunk = (quad & 15) >> 1;
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // channels 16 col + 4 k .. + 3
        uint32_t f[4][2];
        f8x4_to_f16x4<FMT>(__byte_perm(w[0][k], w[1][k], 0x5140), f[0][0], f[1][0]);
        f8x4_to_f16x4<FMT>(__byte_perm(w[2][k], w[3][k], 0x5140), f[0][1], f[1][1]);
        f8x4_to_f16x4<FMT>(__byte_perm(w[0][k], w[1][k], 0x7362), f[2][0], f[3][0]);
        f8x4_to_f16x4<FMT>(__byte_perm(w[2][k], w[3][k], 0x7362), f[2][1], f[3][1]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int n = (4 * k + c) * S::kCols + col;
          *reinterpret_cast<uint2*>(dst + n * 128 + ((chunk ^ (n & 7)) << 4)) = make_uint2(f[c][0], f[c][1]);
        }
      }
      odd = __any_sync(0xffffffffu, odd);
      if (lane == 0) s_info[idx & 3].odd[warp - kSoftWarps] = odd;
      fence_proxy_async_shared();
      mbar_arrive(&s_v_full[g]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------- products --
    int idx = 0, nseg = 0;
    while (walk.next(p, kRows, seg)) {
      int from, to;
      tiles_of(walk, seg, from, to);
      if (from >= to) continue;  // such segments pass neither barrier: the softmax warps could run two phases ahead
      auto product_pv = [&](int i, bool first) {  // of tile number i; the group's first of the segment overwrites O
        const int g = i & 1;
        wait(&s_v_full[g], i >> 1);
        wait(&s_p_full[g], i >> 1);
        if (first && nseg > 0) wait(&s_o_free, nseg - 1);
        tc_fence_after();
        if (lane == 0) {
          const uint64_t b = sw128_desc(smem_u32(v_tile(g)));
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)  // 16 keys: 8 columns of P, 32 bytes of V's rows; 64 keys an atom
            umma_ts(tmem + S::kTmemO + g * D, tmem + S::kTmemS + g * kKeys + 8 * k, b + (k >> 2) * (D * 128 >> 4) + (k & 3) * 2, idesc_f16(kRows, D), !(first && k == 0));
          umma_commit(&s_pv_done[g]);
        }
        __syncwarp();
      };
      for (int tile = from; tile < to; ++tile, ++idx) {
        const int g = idx & 1;
        wait(&s_k_full[idx & 3], idx >> 2);
        if (tile == from) wait(&s_q_full, nseg);
        tc_fence_after();
        if (lane == 0) {
          const uint64_t a = sw128_desc(smem_u32(q_tile)), b = sw128_desc(smem_u32(k_tile));
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_ss(tmem + S::kTmemS + g * kKeys, a + (k >> 2) * (kRows * 128 >> 4) + (k & 3) * 2, b + (k >> 2) * (kKeys * 128 >> 4) + (k & 3) * 2, idesc_f16(kRows, kKeys), k > 0);
          umma_commit(&s_s_full[g]);
        }
        __syncwarp();
        if (tile > from) product_pv(idx - 1, tile - from <= 2);
      }
      product_pv(idx - 1, to - from <= 2);
      ++nseg;  // segments with tiles
    }
  } else {
    // ----------------------------------------------------------- softmax --
    const int g = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t row_at = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + row_at + S::kTmemS + g * kKeys, o_at = tmem + row_at + S::kTmemO + g * D;
    const int walk_begin = walk.u;
    int idx = 0, n_shared = 0;
    while (walk.next(p, kRows, seg)) {
      const Seq& s = walk.s;
      int from, to;
      tiles_of(walk, seg, from, to);
      const int row = seg.rt * kRows + r;
      const bool in = row < s.rows;
      const bool active = (warp & 3) * 32 < s.rows - seg.rt * kRows;  // the warp has rows
      const int pos = in ? s.len - s.n + row / p.group : -1;
      // Q as fp16: consecutive threads take consecutive 16-byte pieces of the rows
      if (to > from) {
        constexpr int kPieces = D / 8, kEach = kRows * kPieces / kSoft;
        const bool bf = p.a.a_type == FP8IMMA_A_BF16;
        uint4 x[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int r2 = (i * kSoft + tid) / kPieces, ch = tid % kPieces * 8, row2 = seg.rt * kRows + r2;
          x[i] = make_uint4(0, 0, 0, 0);
          if (row2 < s.rows) {
            const uint16_t* src = static_cast<const uint16_t*>(p.a.q) + (int64_t)(s.t0 + row2 / p.group) * p.a.q_token_stride + (int64_t)(seg.h * p.group + row2 % p.group) * p.a.q_head_stride + ch;
            if (p.vec_q) {
              x[i] = __ldg(reinterpret_cast<const uint4*>(src));
            } else {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = (uint32_t)__ldg(src + 2 * k) | ((uint32_t)__ldg(src + 2 * k + 1) << 16);
              x[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int r2 = (i * kSoft + tid) / kPieces, ch = tid % kPieces * 8;
          if (bf) {  // a power of two brings the row to a largest magnitude of 2^8 .. 2^9
            uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            float big = 0.0f, f = 1.0f, back = 1.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) big = fmaxf(big, fmaxf(fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xFFFF0000u))));
#pragma unroll
            for (int o = 1; o < kPieces; o *= 2) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            if (big > 0.0f && big < INFINITY) {
              const int e = max(-126, min(126, (int)(__float_as_uint(big) >> 23) - 127 - 8));
              f = __uint_as_float((uint32_t)(127 - e) << 23);
              back = __uint_as_float((uint32_t)(127 + e) << 23);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = pack_f16(__uint_as_float(w[k] << 16) * f, __uint_as_float(w[k] & 0xFFFF0000u) * f);
            x[i] = make_uint4(w[0], w[1], w[2], w[3]);
            if (ch == 0) s_back[r2] = back;
          } else if (ch == 0) {
            s_back[r2] = 1.0f;
          }
          *reinterpret_cast<uint4*>(q_tile + (ch >> 6) * (kRows * 128) + r2 * 128 + ((((ch & 63) >> 3) ^ (r2 & 7)) << 4)) = x[i];
        }
        fence_proxy_async_shared();
        mbar_arrive(&s_q_full);
        named_bar_sync(1, kSoft);  // s_back
      }
      const float back = to > from ? s_back[r] : 1.0f;
      const float cq = p.a.softmax_scale * 1.4426950408889634f * back;
      float m = -INFINITY, l = 0.0f;
      int count = 0;       // the group's tiles of the segment
      bool dirty = false;  // the row has poison marks
      for (int tile = from; tile < to; ++tile, ++idx) {
        if ((idx & 1) != g) continue;
        wait(&s_s_full[g], idx >> 1);
        wait(&s_k_full[idx & 3], idx >> 2);  // s_info
        tc_fence_after();
        const TileInfo& info = s_info[idx & 3];
        __syncwarp();
        if (active) {
          const bool edge = edge_tile(p, seg, tile) || info.live != 0xffff || !(cq >= 0.0f);
          // the row sees keys v0 <= j < v0 + nv
          const int v0 = p.a.window > 0 ? max(0, pos - p.a.window + 1) : 0, nv = max(0, min(pos + 1, seg.hi) - v0);
          // A score above m by more than kRaise moves m, in whole steps: what has
          // been summed and the weights of the tile so far shrink by a power of two.
          auto raise = [&](int done, float top) {  // 32 done keys have their weights
            const bool up = top > m + kRaise;
            const float mn = !up ? m : m == -INFINITY ? top : m + ceilf(top - m), f = up ? ex2(m - mn) : 1.0f;
            // fp16's smallest number is 2^-24, so P takes the factor in halves
            const float half = f > 0.0f && up ? floorf(0.5f * (m - mn)) : 0.0f, f0 = ex2(half), f1 = f > 0.0f && up ? ex2(m - mn - half) : f;
            m = mn;
            l *= f;
            tmem_wait_st();
#pragma unroll 1
            for (int c = 0; c < done; ++c) {
              uint32_t v[16];
              tmem_ld16(s_at + 16 * c, v);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = mul_f16x2(mul_f16x2(v[i], f0), f1);
              tmem_st16(s_at + 16 * c, v);
            }
            if (count > 0) {  // O: the group's product before is done, these scores were issued after it
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                uint32_t v[16];
                tmem_ld16(o_at + c, v);
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                tmem_st16(o_at + c, v);
              }
            }
            tmem_wait_st();
          };
          // 32 keys at a time; P takes the place of scores that have been read
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t v[32], w[16];
            tmem_ld32(s_at + 32 * c, v);
            float sum[2];
            if (edge) {
              float x[32], top = -INFINITY;
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                const int i = 2 * c + k / 16;
                x[k] = fmaf(__uint_as_float(v[k]), cq * info.ks[i], info.lv[i]);
                if (!((info.live >> i) & 1) || (unsigned)(tile * kKeys + 32 * c + k - v0) >= (unsigned)nv) x[k] = -INFINITY;
                top = fmaxf(top, x[k]);
              }
              if (__any_sync(0xffffffffu, top > m + kRaise)) raise(c, top);
              const float ms = m == -INFINITY ? 0.0f : m;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                sum[h] = 0.0f;
#pragma unroll
                for (int k = 16 * h; k < 16 * h + 16; k += 2) {
                  const float a = ex2(x[k] - ms), b = ex2(x[k + 1] - ms);
                  sum[h] += a + b;
                  w[k / 2] = pack_f16(a, b);
                }
              }
            } else {
              // the largest score of 16 keys is that of their largest product
              float kc[2], top[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float most[2] = {__uint_as_float(v[16 * h]), __uint_as_float(v[16 * h + 1])};
#pragma unroll
                for (int k = 16 * h + 2; k < 16 * h + 14; k += 4) {
                  most[0] = fmaxf(most[0], fmaxf(__uint_as_float(v[k]), __uint_as_float(v[k + 1])));
                  most[1] = fmaxf(most[1], fmaxf(__uint_as_float(v[k + 2]), __uint_as_float(v[k + 3])));
                }
                most[0] = fmaxf(most[0], fmaxf(__uint_as_float(v[16 * h + 14]), __uint_as_float(v[16 * h + 15])));
                kc[h] = cq * info.ks[2 * c + h];
                top[h] = fmaf(fmaxf(most[0], most[1]), kc[h], info.lv[2 * c + h]);
              }
              const float most = fmaxf(top[0], top[1]);
              if (__any_sync(0xffffffffu, most > m + kRaise)) raise(c, most);
              const float ms = m == -INFINITY ? 0.0f : m;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float lv = info.lv[2 * c + h] - ms;
                const uint64_t kc2 = pair(kc[h], kc[h]), lv2 = pair(lv, lv);
                uint64_t two = 0;
#pragma unroll
                for (int k = 16 * h; k < 16 * h + 16; k += 2) {
                  float a, b;
                  unpair(fma2(pair(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), kc2, lv2), a, b);
                  a = ex2(a), b = ex2(b);
                  two = add2(two, pair(a, b));
                  w[k / 2] = pack_f16(a, b);
                }
                float s0, s1;
                unpair(two, s0, s1);
                sum[h] = s0 + s1;
              }
            }
            l = fmaf(sum[1], info.iv[2 * c + 1], fmaf(sum[0], info.iv[2 * c], l));
            tmem_st16(s_at + 16 * c, w);
          }
          tmem_wait_st();
        }
        wait(&s_v_full[g], idx >> 1);  // the rest of s_info
        __syncwarp();
        if (active) {
          int odd = 0;
#pragma unroll
          for (int i = 0; i < S::kLoadWarps; ++i) odd |= info.odd[i];
          if (odd) {
            // rare: mark the channels of this row that a non-finite value reaches
            uint8_t* mark = poison + (g * kRows + r) * (D / 2);
            if (!dirty)
              for (int c = 0; c < D / 2; c += 16) *reinterpret_cast<uint4*>(mark + c) = make_uint4(0, 0, 0, 0);
            dirty = true;
            const int ps = p.c.page_size;
            for (int j = max(tile * kKeys, seg.lo); j < min(min(tile * kKeys + kKeys, seg.hi), pos + 1); ++j) {
              if ((p.a.window > 0 && j <= pos - p.a.window) || !(info.live >> ((j & (kKeys - 1)) >> 4) & 1)) continue;
              const int page = __ldg(p.c.page_table + (size_t)seg.b * p.c.max_pages + j / ps);
              const uint8_t* v = static_cast<const uint8_t*>(p.c.v) + (((size_t)page * p.c.kv_heads + seg.h) * ps + (j & (ps - 1))) * D;
              for (int ch = 0; ch < D; ++ch) {
                const float x = f8_to_f32<FMT>(__ldg(v + ch));
                const int n = ch % 16 * S::kCols + ch / 16;
                if (!(fabsf(x) < INFINITY)) mark[n / 2] |= (isnan(x) ? 4 : x > 0.0f ? 1 : 2) << (n % 2 * 4);
              }
            }
          }
        }
        ++count;
        tc_fence_before();
        mbar_arrive(&s_p_full[g]);
      }
      // ------------------------------------------ the two groups' O joined --
      const int other = to > from ? to - from - count : 0;
      if (count > 0) {
        const int last = idx - 1 - ((idx - 1) & 1 ? 1 - g : g);  // the group's last tile number (idx: one past the segment's)
        wait(&s_pv_done[g], last >> 1);
      }
      s_ml[g][r][0] = m;
      s_ml[g][r][1] = l;
      s_ml[g][r][2] = dirty ? 1.0f : 0.0f;
      tc_fence_before();
      named_bar_sync(1, kSoft);
      tc_fence_after();
      const float m2 = s_ml[1 - g][r][0], l2 = s_ml[1 - g][r][1];
      const bool dirty2 = s_ml[1 - g][r][2] != 0.0f;
      const float M = fmaxf(m, m2), ms = M == -INFINITY ? 0.0f : M, f = ex2(m - ms), f2 = ex2(m2 - ms);
      const float L = g == 0 ? fmaf(l, f, l2 * f2) : fmaf(l2, f2, l * f);  // the same in both groups
      const bool shared = seg.count != s.tiles;
      const Item it = {s.t0, s.rows, seg.rt, seg.h};
      float* const part = p.parts + (int64_t)(blockIdx.x * 2 + (seg.item0 > walk_begin ? 1 : 0)) * S::kPartFloats;
      const int64_t out_row = in ? (int64_t)(s.t0 + row / p.group) * p.a.heads + seg.h * p.group + row % p.group : 0;
      const float inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
      if (active) {
#pragma unroll 1
        for (int c0 = 0; c0 < D / 2; c0 += 16) {
          const int n0 = g * (D / 2) + c0;
          __syncwarp();
          uint32_t a[16] = {}, b[16] = {};
          float o[16];
          if (count > 0) tmem_ld16_start(o_at + n0, a);
          if (other > 0) tmem_ld16_start(tmem + row_at + S::kTmemO + (1 - g) * D + n0, b);
          tmem_ld_wait(a);
          tmem_ld_wait(b);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = (count > 0 ? __uint_as_float(a[i]) * f : 0.0f) + (other > 0 ? __uint_as_float(b[i]) * f2 : 0.0f);
          if (dirty || dirty2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int bits = ((dirty ? poison[(g * kRows + r) * (D / 2) + (n0 + i) / 2] : 0) | (dirty2 ? poison[((1 - g) * kRows + r) * (D / 2) + (n0 + i) / 2] : 0)) >> (i % 2 * 4) & 15;
              if (bits) o[i] = bits == 1 ? INFINITY : bits == 2 ? -INFINITY : NAN;
            }
          }
          if (in && shared) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(part + r * D + n0 + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          } else if (in) {
            // column n is channel 16 (n % cols) + n / cols
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if ((i / S::kCols) & 1) continue;
              const int n = n0 + i;
              *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.a.out) + out_row * D + 16 * (n % S::kCols) + n / S::kCols) = out_pair(o[i] * inv, o[i + S::kCols] * inv, p.a.a_type);
            }
          }
        }
      }
      if (in && g == 0) {
        if (shared) {
          *reinterpret_cast<float2*>(part + kRows * D + 2 * r) = make_float2(M, L);
        } else if (p.a.lse) {
          p.a.lse[out_row] = L == 0.0f ? -INFINITY : 0.6931471805599453f * (M + log2f(L));
        }
      }
      if (shared && tid == 0) {
        s_shared[n_shared].item = it;
        s_shared[n_shared].index = seg.item;
        s_shared[n_shared].c0 = runs.of(seg.item0);
        s_shared[n_shared].c1 = runs.of(seg.item0 + s.tiles - 1);
        s_shared[n_shared].item0 = seg.item0;
      }
      n_shared += shared;
      tc_fence_before();
      if (to > from) mbar_arrive(&s_o_free);
      named_bar_sync(1, kSoft);  // s_ml and the poison marks are free again
    }

    if (tid == 0) s_n_shared = n_shared;
    __threadfence();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);

  // shared items: the CTA that comes last to one joins all its parts, in CTA order
  const int n_shared = s_n_shared;
  if (n_shared == 0) return;
  if (tid < n_shared) {
    unsigned int prev, *ctr = p.counters + s_shared[tid].index;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(prev) : "l"(ctr) : "memory");
    s_shared[tid].last = prev == (unsigned)(s_shared[tid].c1 - s_shared[tid].c0);
    if (s_shared[tid].last) *ctr = 0;  // ready for the next call
  }
  __syncthreads();
  __threadfence();
  for (int k = 0; k < n_shared; ++k) {
    const Shared& sh = s_shared[k];
    if (!sh.last) continue;
    const int rows = min(kRows, sh.item.rows - sh.item.rt * kRows);
    const Item it = sh.item;
    auto src = [&](int c) { return p.parts + (int64_t)(c * 2 + (sh.item0 > runs.begin(c) ? 1 : 0)) * S::kPartFloats; };
    auto out_at = [&](int r) {
      const int row = it.rt * kRows + r;
      return (int64_t)(it.t0 + row / p.group) * p.a.heads + it.h * p.group + row % p.group;
    };
    // the rows' references and sums
    for (int r = tid; r < rows; r += S::kThreads) {
      float m = -INFINITY, l = 0.0f;
      for (int c = sh.c0; c <= sh.c1; ++c) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(src(c) + kRows * D + 2 * r));
        const float mn = fmaxf(m, v.x), ms = mn == -INFINITY ? 0.0f : mn;
        l = fmaf(l, ex2(m - ms), v.y * ex2(v.x - ms));
        m = mn;
      }
      s_ml[0][r][0] = m == -INFINITY ? 0.0f : m;
      s_ml[0][r][1] = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
      if (p.a.lse) p.a.lse[out_at(r)] = l == 0.0f ? -INFINITY : 0.6931471805599453f * (m + log2f(l));
    }
    __syncthreads();
    // O: each thread has the loads of kAt places in flight
    constexpr int kAt = 4, kWorkers = S::kThreads / 32 * 32;
    for (int x0 = tid; x0 < rows * (D / 4); x0 += kWorkers * kAt) {
      float4 o[kAt];
#pragma unroll
      for (int e = 0; e < kAt; ++e) o[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int c = sh.c0; c <= sh.c1; ++c) {
        const float* const part = src(c);
        float4 v[kAt];
        float m[kAt];
#pragma unroll
        for (int e = 0; e < kAt; ++e) {
          const int x = min(x0 + e * kWorkers, rows * (D / 4) - 1);
          v[e] = __ldcg(reinterpret_cast<const float4*>(part) + x);
          m[e] = __ldcg(part + kRows * D + x / (D / 4) * 2);
        }
#pragma unroll
        for (int e = 0; e < kAt; ++e) {
          const int x = min(x0 + e * kWorkers, rows * (D / 4) - 1);
          const float f = ex2(m[e] - s_ml[0][x / (D / 4)][0]);
          o[e] = make_float4(fmaf(v[e].x, f, o[e].x), fmaf(v[e].y, f, o[e].y), fmaf(v[e].z, f, o[e].z), fmaf(v[e].w, f, o[e].w));
        }
      }
#pragma unroll
      for (int e = 0; e < kAt; ++e) {
        const int x = x0 + e * kWorkers, r = x / (D / 4), n = x % (D / 4) * 4;
        if (x >= rows * (D / 4)) break;
        const float inv = s_ml[0][r][1], w[4] = {o[e].x, o[e].y, o[e].z, o[e].w};
        uint16_t* const dst = static_cast<uint16_t*>(p.a.out) + out_at(r) * D;
#pragma unroll
        for (int i = 0; i < 4; ++i)  // column n is channel 16 (n % cols) + n / cols
          dst[16 * ((n + i) % S::kCols) + (n + i) / S::kCols] = p.a.a_type == FP8IMMA_A_F16 ? f32_to_a16<0>(w[i] * inv) : f32_to_a16<1>(w[i] * inv);
      }
    }
    __syncthreads();  // s_ml
  }
}

template <int FMT, int D>
cudaError_t launch(AttnParams& p, cudaStream_t st) {
  using S = Shape<D>;
  const auto kern = kv_attention_tc_kernel<FMT, D>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), S::kSmem);
  if (e != cudaSuccess) return e;
  const int64_t items = ((int64_t)p.c.tokens * p.group / kRows + p.c.batch) * p.c.kv_heads;
  const int64_t tiles = ((int64_t)p.c.max_pages * p.c.page_size + kKeys - 1) / kKeys;
  if (items * tiles > 0x7fffffffll) return cudaErrorInvalidValue;  // units are counted in 31 bits
  const int grid = (int)std::min<int64_t>(num_sms_current(), std::max<int64_t>(1, items * tiles));
  const size_t ctr_bytes = (size_t)items * 4, part_bytes = (size_t)grid * 2 * S::kPartFloats * 4;
  ScopedScratch ctr, part;
  e = ctr.get(ctr_bytes, st, kScratchAttn);
  if (e == cudaSuccess && ctr.owned) e = cudaMemsetAsync(ctr.ptr, 0, ctr_bytes, st);
  if (e == cudaSuccess) e = part.get(part_bytes, st, kScratchAttnParts);
  if (e == cudaSuccess) {
    p.counters = static_cast<unsigned int*>(ctr.ptr);
    p.parts = static_cast<float*>(part.ptr);
    cudaLaunchConfig_t lc = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.gridDim = dim3(grid);
    lc.blockDim = dim3(S::kThreads);
    lc.dynamicSmemBytes = S::kSmem;
    lc.stream = st;
    lc.attrs = attr;
    lc.numAttrs = api_pdl() ? 1 : 0;
    e = cudaLaunchKernelEx(&lc, kern, p);
  }
  const cudaError_t e1 = ctr.release(st), e2 = part.release(st);
  return e != cudaSuccess ? e : e1 != cudaSuccess ? e1 : e2;
}

}  // namespace

cudaError_t launch_attention_tc(AttnParams& p, cudaStream_t st) {
  if (p.c.head_dim == 64) return p.c.format == FP8IMMA_B_E4M3 ? launch<F8_E4M3, 64>(p, st) : launch<F8_E5M2, 64>(p, st);
  return p.c.format == FP8IMMA_B_E4M3 ? launch<F8_E4M3, 128>(p, st) : launch<F8_E5M2, 128>(p, st);
}
unsigned int attn_tc_device_error(bool clear) { return fp8imma_dev::tu_device_error(clear); }
cudaError_t attn_tc_set_wait_limit(unsigned long long ns) { return fp8imma_dev::tu_set_wait_limit(ns); }

}  // namespace fp8imma_b200
