// Attention over the paged 8-bit KV cache for many query rows a KV head
// (drafts to verify, prompts, wide groups of heads), products by tcgen05.
// Mathematics and the cut of the work are those of kv_attention.cu; a tile here
// is 128 query rows x 128 keys.
//
// Bound: with R rows a key costs 4 R D flops, and the few-row kernel converts
// every FP8 code once for each 8 or 16 rows that a warp multiplies it with; from
// about 32 rows on that conversion, not the copy, is its time. Here a code is
// converted once for up to 128 rows:
//  * two teams of four load warps take tiles in turn: FP8 codes go from global
//    memory to registers one tile ahead, become fp16, and are written to shared
//    memory as the tensor core reads them (K rows, V transposed, both K-major
//    with 128-byte swizzle);
//  * one thread issues S = Q K^T (accumulators in TMEM) and O += P V, with P
//    read from TMEM;
//  * two groups of four softmax warps, one thread a row, take tiles in turn as
//    well: while one computes P of its tile, the tensor core makes the other's S.
// Each group keeps a running reference, sum and O of its own (TMEM: 2 x 128
// columns of S, which P overwrites, 2 x D of O); they are joined where a run
// leaves an item. V's channels lie permuted in shared memory (row c D/16 + col
// for channel 16 col + c), which spreads the transposing stores over the banks;
// O's columns come out in that order.
#include "kv_attention.cuh"
#include "sm100_umma.cuh"
#include <type_traits>

namespace fp8imma_b200 {
namespace {

using namespace fp8imma_dev;
using namespace attn;

constexpr int kRows = 128;
constexpr int kSoftWarps = 8, kLoadWarps = 4;
constexpr int kThreads = (kSoftWarps + kLoadWarps + 1) * 32;
constexpr int kSoft = kSoftWarps * 32;

template <int D>
struct Shape {
  static constexpr int kTile = kKeys * D * 2;             // fp16 bytes of K, of V, of Q
  static constexpr int kPoison = 2 * kRows * D;
  static constexpr int kSmem = 1024 + 5 * kTile + kPoison;
  static constexpr int kPartFloats = kRows * D + kRows * 2;
  static constexpr int kCols = D / 16;                    // 16-channel columns
  static constexpr uint32_t kTmemS = 0, kTmemO = 2 * kKeys;  // TMEM columns of the two groups' S and O
};

__device__ __forceinline__ uint4 ldg_stream(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
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
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

struct TileInfo {
  float ks[8], vs[8];
  int live[8];  // by groups of 16 keys
  int odd[4];   // a load warp found non-finite values that some row may not see
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
__global__ void __launch_bounds__(kThreads, 1) kv_attention_tc_kernel(const __grid_constant__ AttnParams p) {
  using S = Shape<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_kv_full[2], s_s_full[2], s_p_full[2], s_pv_done[2], s_q_full, s_o_free;
  __shared__ TileInfo s_info[2];
  __shared__ Shared s_shared[2];
  __shared__ float s_ml[2][kRows][3];  // reference, sum, whether the group's poison marks count
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* const base = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  uint8_t* const q_tile = base;
  auto k_tile = [&](int g) { return base + S::kTile * (1 + 2 * g); };
  auto v_tile = [&](int g) { return base + S::kTile * (2 + 2 * g); };
  uint8_t* const poison = base + 5 * S::kTile;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_kv_full[i], kLoadWarps * 32);
      mbar_init(&s_s_full[i], 1);
      mbar_init(&s_p_full[i], kSoft / 2);
      mbar_init(&s_pv_done[i], 1);
    }
    mbar_init(&s_q_full, kSoft);
    mbar_init(&s_o_free, kSoft);
    fence_barrier_init();
  }
  pdl_launch_dependents();
  pdl_wait();
  Walk walk;
  int units, ctas;
  if (!find_run<kThreads>(p, kRows, walk, units, ctas)) return;
  const Runs runs(units, ctas);
  if (warp == kSoftWarps + kLoadWarps) {
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
    if (ok) ok = mbar_wait(bar, (uint32_t)(use & 1), ERR_WAIT_FULL);
  };

  if (warp >= kSoftWarps && warp < kSoftWarps + kLoadWarps) {
    // ------------------------------------------------------------- loads --
    const int t = tid - kSoft;
    const int ps = p.c.page_size;
    int tile = 0, to = 0, idx = -1;
    auto next = [&]() {  // on to the next tile
      ++idx;
      if (++tile < to) return true;
      do {
        if (!walk.next(p, kRows, seg)) return false;
        tiles_of(walk, seg, tile, to);
      } while (tile >= to);
      return true;
    };
    // page of the 16-key group `lane` of the tile (lanes 0 .. 7), -1: none that any row sees
    auto page_of = [&]() {
      const int j0 = tile * kKeys + lane * 16, pi = j0 / ps;
      int id = -1;
      if (lane < 8 && j0 < seg.hi && j0 + 15 >= seg.lo && pi < p.c.max_pages) {
        id = __ldg(p.c.page_table + (size_t)seg.b * p.c.max_pages + pi);
        if ((unsigned)id >= (unsigned)p.c.num_pages) id = -1;
      }
      return id;
    };
    uint4 kr[S::kCols], vr[S::kCols / 4][4];
    float ks = 0.0f, vs = 0.0f;
    auto load = [&](int id) {
      ks = vs = 0.0f;
      if (id >= 0) {
        const size_t ph = (size_t)id * p.c.kv_heads + seg.h;
        ks = __ldg(p.c.k_scale + ph);
        vs = __ldg(p.c.v_scale + ph);
      }
      auto piece = [&](const void* pool, int row, int col) {  // 16 codes of a key
        const int page = __shfl_sync(0xffffffffu, id, row >> 4), j = tile * kKeys + row;
        if (page < 0 || j >= seg.hi || j < seg.lo) return make_uint4(0, 0, 0, 0);
        return ldg_stream(static_cast<const uint8_t*>(pool) + (((size_t)page * p.c.kv_heads + seg.h) * ps + (j & (ps - 1))) * D + col * 16);
      };
#pragma unroll
      for (int i = 0; i < S::kCols; ++i) kr[i] = piece(p.c.k, (i * 128 + t) / S::kCols, t % S::kCols);
#pragma unroll
      for (int i = 0; i < S::kCols / 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) vr[i][e] = piece(p.c.v, (i * 128 + t) / S::kCols * 4 + e, t % S::kCols);
    };
    bool more = next();
    int id = more ? page_of() : -1;
    if (more) load(id);
    while (more) {
      const bool edge = edge_tile(p, seg, tile);
      const int live = id >= 0;
      const int g = idx & 1;
      if (idx > 1) wait(&s_pv_done[g], (idx >> 1) - 1);  // the tile that lay here before has been multiplied
      uint8_t *const kt = k_tile(g), *const vt = v_tile(g);
#pragma unroll
      for (int i = 0; i < S::kCols; ++i) {
        const int row = (i * 128 + t) / S::kCols, col = t % S::kCols;
        uint4 a, b;
        f8x4_to_f16x4<FMT>(kr[i].x, a.x, a.y);
        f8x4_to_f16x4<FMT>(kr[i].y, a.z, a.w);
        f8x4_to_f16x4<FMT>(kr[i].z, b.x, b.y);
        f8x4_to_f16x4<FMT>(kr[i].w, b.z, b.w);
        uint8_t* dst = kt + (col >> 2) * (kKeys * 128) + row * 128;
        *reinterpret_cast<uint4*>(dst + ((((col & 3) * 2) ^ (row & 7)) << 4)) = a;
        *reinterpret_cast<uint4*>(dst + ((((col & 3) * 2 + 1) ^ (row & 7)) << 4)) = b;
      }
      bool odd = false;
#pragma unroll
      for (int i = 0; i < S::kCols / 4; ++i) {
        const int quad = (i * 128 + t) / S::kCols, col = t % S::kCols;
        uint32_t w[4][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e][0] = vr[i][e].x, w[e][1] = vr[i][e].y, w[e][2] = vr[i][e].z, w[e][3] = vr[i][e].w;
          if (edge) {
            // 0 * NaN must not reach the rows that do not see the key: such values are left out here and marked below
            const uint32_t mk = FMT == F8_E4M3 ? 0x7F7F7F7Fu : 0x7C7C7C7Cu;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t bad = __vcmpeq4(w[e][k] & mk, mk);
              odd |= bad != 0u;
              w[e][k] &= ~bad;
            }
          }
        }
        uint8_t* dst = vt + (quad >> 4) * (D * 128) + (quad & 1) * 8;
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
      }
      odd = __any_sync(0xffffffffu, odd);
      if (lane == 0) s_info[g].odd[warp & 3] = odd;
      if (t < 8) {
        s_info[g].ks[t] = ks;
        s_info[g].vs[t] = vs;
        s_info[g].live[t] = live;
      }
      fence_proxy_async_shared();
      mbar_arrive(&s_kv_full[g]);
      more = next();
      if (more) {
        id = page_of();
        load(id);
      }
    }
  } else if (warp == kSoftWarps + kLoadWarps) {
    // ---------------------------------------------------------- products --
    int idx = 0, nseg = 0;
    while (walk.next(p, kRows, seg)) {
      int from, to;
      tiles_of(walk, seg, from, to);
      if (from >= to) continue;  // such segments pass neither barrier: the softmax warps could run two phases ahead
      auto product_pv = [&](int i, bool first) {  // of tile number i; the group's first of the segment overwrites O
        const int g = i & 1;
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
        wait(&s_kv_full[g], idx >> 1);
        if (tile == from) wait(&s_q_full, nseg);
        tc_fence_after();
        if (lane == 0) {
          const uint64_t a = sw128_desc(smem_u32(q_tile)), b = sw128_desc(smem_u32(k_tile(g)));
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
      // Q: this thread's half of the row, as fp16
      float back = 1.0f;
      if (to > from) {
        const uint16_t* src = static_cast<const uint16_t*>(p.a.q) +
                              (in ? (int64_t)(s.t0 + row / p.group) * p.a.q_token_stride + (int64_t)(seg.h * p.group + row % p.group) * p.a.q_head_stride : 0);
        auto eight = [&](int ch) {
          if (!in) return make_uint4(0, 0, 0, 0);
          if (p.vec_q) return __ldg(reinterpret_cast<const uint4*>(src + ch));
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldg(src + ch + 2 * i) | ((uint32_t)__ldg(src + ch + 2 * i + 1) << 16);
          return make_uint4(w[0], w[1], w[2], w[3]);
        };
        float f = 1.0f;
        const bool bf = p.a.a_type == FP8IMMA_A_BF16;
        if (bf) {  // a power of two brings the row to a largest magnitude of 2^8 .. 2^9
          float big = 0.0f;
#pragma unroll 4
          for (int c = 0; c < D; c += 8) {
            const uint4 v = eight(c);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) big = fmaxf(big, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xFFFF0000u))));
          }
          if (big > 0.0f && big < INFINITY) {
            const int e = max(-126, min(126, (int)(__float_as_uint(big) >> 23) - 127 - 8));
            f = __uint_as_float((uint32_t)(127 - e) << 23);
            back = __uint_as_float((uint32_t)(127 + e) << 23);
          }
        }
#pragma unroll 4
        for (int i = 0; i < D / 16; ++i) {
          const int ch = g * (D / 2) + i * 8;
          uint4 v = eight(ch);
          if (bf) {
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = pack_f16(__uint_as_float(w[k] << 16) * f, __uint_as_float(w[k] & 0xFFFF0000u) * f);
            v = make_uint4(w[0], w[1], w[2], w[3]);
          }
          *reinterpret_cast<uint4*>(q_tile + (ch >> 6) * (kRows * 128) + r * 128 + ((((ch & 63) >> 3) ^ (r & 7)) << 4)) = v;
        }
        fence_proxy_async_shared();
        mbar_arrive(&s_q_full);
      }
      const float cq = p.a.softmax_scale * 1.4426950408889634f * back;
      float m = -INFINITY, l = 0.0f;
      int count = 0;       // the group's tiles of the segment
      bool dirty = false;  // the row has poison marks
      for (int tile = from; tile < to; ++tile, ++idx) {
        if ((idx & 1) != g) continue;
        wait(&s_s_full[g], idx >> 1);
        tc_fence_after();
        const TileInfo& info = s_info[g];
        __syncwarp();
        if (active) {
          bool edge = edge_tile(p, seg, tile);
#pragma unroll
          for (int i = 0; i < 8; ++i) edge |= !info.live[i];
          auto score = [&](auto masked, uint32_t bits, float kc, float lv, int j) {
            float x = fmaf(__uint_as_float(bits), kc, lv);
            if (decltype(masked)::value && (j > pos || j >= seg.hi || (p.a.window > 0 && j <= pos - p.a.window))) x = -INFINITY;
            return x;
          };
          auto group_of = [&](int i, float& kc, float& lv, float& iv) {
            const float vs = info.vs[i] < kTinyScale ? kTinyScale : info.vs[i];
            kc = cq * info.ks[i];
            lv = info.live[i] ? lg2(vs) : -INFINITY;
            iv = __fdividef(1.0f, vs);
          };
          float top = -INFINITY;
          auto find_top = [&](auto masked) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t v[32];
            tmem_ld32(s_at + 32 * c, v);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float kc, lv, iv;
              group_of(2 * c + h, kc, lv, iv);
#pragma unroll
              for (int i = 0; i < 16; ++i) top = fmaxf(top, score(masked, v[16 * h + i], kc, lv, tile * kKeys + 32 * c + 16 * h + i));
            }
          }
          };
          if (edge) find_top(std::true_type()); else find_top(std::false_type());
          const bool raise = top > m + kRaise;
          if (__any_sync(0xffffffffu, raise)) {
            const float mn = raise ? top : m, f = mn == m ? 1.0f : ex2(m - mn);
            m = mn;
            l *= f;
            if (count > 0) {  // the product before is done: its keys' place has been filled again
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                uint32_t v[16];
                tmem_ld16(o_at + c, v);
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                tmem_st16(o_at + c, v);
              }
              tmem_wait_st();
            }
          }
          const float ms = m == -INFINITY ? 0.0f : m;
          auto weights = [&](auto masked) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t v[32], w[16];
            tmem_ld32(s_at + 32 * c, v);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float kc, lv, iv, sum = 0.0f;
              group_of(2 * c + h, kc, lv, iv);
              lv -= ms;
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                const int j = tile * kKeys + 32 * c + 16 * h + i;
                float a = ex2(score(masked, v[16 * h + i], kc, lv, j)), b = ex2(score(masked, v[16 * h + i + 1], kc, lv, j + 1));
                if (decltype(masked)::value && !info.live[2 * c + h]) a = b = 0.0f;
                sum += a + b;
                w[8 * h + i / 2] = pack_f16(a, b);
              }
              l = fmaf(sum, iv, l);
            }
            tmem_st16(s_at + 16 * c, w);  // P takes the place of scores that have been read
          }
          };
          if (edge) weights(std::true_type()); else weights(std::false_type());
          tmem_wait_st();
          if (info.odd[0] | info.odd[1] | info.odd[2] | info.odd[3]) {
            // rare: mark the channels of this row that a non-finite value reaches
            uint8_t* mark = poison + (g * kRows + r) * D;
            if (!dirty)
              for (int c = 0; c < D; c += 16) *reinterpret_cast<uint4*>(mark + c) = make_uint4(0, 0, 0, 0);
            dirty = true;
            const int ps = p.c.page_size;
            for (int j = max(tile * kKeys, seg.lo); j < min(min(tile * kKeys + kKeys, seg.hi), pos + 1); ++j) {
              if ((p.a.window > 0 && j <= pos - p.a.window) || !info.live[(j & (kKeys - 1)) >> 4]) continue;
              const int page = __ldg(p.c.page_table + (size_t)seg.b * p.c.max_pages + j / ps);
              const uint8_t* v = static_cast<const uint8_t*>(p.c.v) + (((size_t)page * p.c.kv_heads + seg.h) * ps + (j & (ps - 1))) * D;
              for (int ch = 0; ch < D; ++ch) {
                const float x = f8_to_f32<FMT>(__ldg(v + ch));
                if (!(fabsf(x) < INFINITY)) mark[ch % 16 * S::kCols + ch / 16] |= isnan(x) ? 4 : x > 0.0f ? 1 : 2;
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
          uint32_t a[16], b[16];
          float o[16];
          if (count > 0) tmem_ld16(o_at + n0, a);
          if (other > 0) tmem_ld16(tmem + row_at + S::kTmemO + (1 - g) * D + n0, b);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = (count > 0 ? __uint_as_float(a[i]) * f : 0.0f) + (other > 0 ? __uint_as_float(b[i]) * f2 : 0.0f);
          if (dirty || dirty2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int bits = (dirty ? poison[(g * kRows + r) * D + n0 + i] : 0) | (dirty2 ? poison[((1 - g) * kRows + r) * D + n0 + i] : 0);
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

    // shared items: the CTA that comes last to one joins all its parts, in CTA order
    if (n_shared > 0) {
      __threadfence();
      named_bar_sync(1, kSoft);
      if (tid < n_shared) {
        unsigned int prev, *ctr = p.counters + s_shared[tid].index;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(prev) : "l"(ctr) : "memory");
        s_shared[tid].last = prev == (unsigned)(s_shared[tid].c1 - s_shared[tid].c0);
        if (s_shared[tid].last) *ctr = 0;  // ready for the next call
      }
      named_bar_sync(1, kSoft);
      __threadfence();
      for (int k = 0; k < n_shared; ++k) {
        const Shared& sh = s_shared[k];
        if (!sh.last) continue;
        const int rows = min(kRows, sh.item.rows - sh.item.rt * kRows);
        for (int x = tid; x < rows * (D / 4); x += kSoft) {
          const int r2 = x / (D / 4), n = x % (D / 4) * 4;
          Joined j;  // one row: its second row's place is filled alike
          auto src = [&](int c) {
            c += sh.c0;
            return p.parts + (int64_t)(c * 2 + (sh.item0 > runs.begin(c) ? 1 : 0)) * S::kPartFloats;
          };
          j.join(sh.c1 - sh.c0 + 1,
                 [&](int c) {
                   const float2 v = __ldcg(reinterpret_cast<const float2*>(src(c) + kRows * D + 2 * r2));
                   return make_float4(v.x, v.x, v.y, v.y);
                 },
                 [&](int c) { return __ldcg(reinterpret_cast<const float4*>(src(c) + r2 * D + n)); });
          const int row = sh.item.rt * kRows + r2;
          const int64_t at = (int64_t)(sh.item.t0 + row / p.group) * p.a.heads + sh.item.h * p.group + row % p.group;
          const float inv = j.l0 == 0.0f ? 0.0f : __fdiv_rn(1.0f, j.l0);
          const float o[4] = {j.o.x, j.o.y, j.o.z, j.o.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint16_t v = p.a.a_type == FP8IMMA_A_F16 ? f32_to_a16<0>(o[i] * inv) : f32_to_a16<1>(o[i] * inv);
            static_cast<uint16_t*>(p.a.out)[at * D + 16 * ((n + i) % S::kCols) + (n + i) / S::kCols] = v;
          }
          if (n == 0 && p.a.lse) p.a.lse[at] = j.l0 == 0.0f ? -INFINITY : 0.6931471805599453f * (j.m0 + log2f(j.l0));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftWarps + kLoadWarps) tmem_dealloc(tmem, 512);
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
  p.max_items = (int)items;
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
    lc.blockDim = dim3(kThreads);
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
