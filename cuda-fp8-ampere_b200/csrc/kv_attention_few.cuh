// Attention of a step's queries over the paged 8-bit KV cache
// (fp8imma_kv_attention).
//
// Mathematics, per sequence and KV head, in base 2 (c = softmax_scale log2 e):
//   x_rj = c <q_r, K_j> ks,   w_rj = 2^(x_rj + log2 vs - M_r),
//   out_r = sum_j w_rj V_j / L_r,   L_r = sum_j w_rj / vs,   lse_r = ln2 (M_r + log2 L_r)
// with K_j, V_j the stored codes (exact in fp16) and ks, vs the scales of
// their page. Taking the value scale into the exponent keeps it out of the
// products: w is rounded to fp16 for the tensor cores relative to the largest
// weight *times scale* of the row so far, so a page with a large scale and a
// small weight is as precise as the other way round. M is a running reference
// that follows the maximum when it is exceeded by more than 2^8; sums, M and L
// are fp32.
//
// Bound: the cache is read once, 2 len D bytes a KV head; at up to ~64 query
// rows a KV head the products are far below the tensor rate, so the kernel is
// built to keep the copies running:
//  * one CTA per SM; a producer warp streams 128-key stages (one TMA box per
//    page for K and for V, 128-byte swizzle) through a ring of 2..6 stages, page
//    ids and scales fetched a batch of 32 ahead. Boxes below 4 KB are slow (2 KB:
//    3.8 TB/s, 4 KB: 6.6 TB/s), so pages smaller than that are copied 16 bytes a
//    lane by four producer warps (512 contiguous bytes a warp: 6.6 TB/s) into the
//    same places;
//  * the 128-key tiles of all (sequence, row tile, KV head) items are laid end
//    to end and cut into equal runs, one per CTA, whatever the lengths are
//    (lengths are read on the device). Items that several CTAs share are joined
//    by the last of them to finish, in CTA order, so results do not depend on
//    timing;
//  * K is the 16-row operand of mma.sync m16n8k16 (S^T = K Q^T: 16 keys x 8
//    query rows) and V^T likewise (O^T = V^T P^T), so 8 rows, one group of
//    heads, fill a tile. The order of channels within a product is free, so a
//    lane's operand is bytes that lie together in its key's row; key pairs of V
//    are interleaved with byte permutes; P^T comes from S^T by movmatrix.
//
// Measured (e4m3): 128 sequences of up to 8192 keys, 64 heads over 8 of 128
// channels, one token each, 237 to 255 us by the board (4.8 to 5.1 TB/s: equal
// runs end some 10% apart, for SMs do not get equal shares of the memory); one
// sequence of 131000 keys 57 us (4.7 TB/s with start and join); one short
// sequence 9.3 us, latency. With many rows see attention_tc_pays().
#pragma once

#include "kv_attention.cuh"

#include <algorithm>

namespace fp8imma_b200 {
namespace {  // each of the two files that instantiate the kernel has its own error word

using namespace fp8imma_dev;
using namespace attn;

constexpr int kConsumers = 8;               // consumer warps
constexpr int kProducers = 4;               // producer warps; TMA takes the first of them only
constexpr int kThreads = (kConsumers + kProducers) * 32;
constexpr int kSlots = kKeys / 16;          // pages of a stage at most

// Shapes of a variant: head_dim D, NT tiles of 8 query rows a warp, RW warps
// along the rows (8 / RW along the keys).
template <int D, int NT, int RW>
struct Shape {
  static constexpr int kRows = 8 * NT * RW;
  static constexpr int kKeyWarps = kConsumers / RW;
  // A warp takes kNG groups of 16 keys at once, where registers allow two: the
  // chains of dependent products, not the issue slots, are what a group waits
  // for. With one row warp, warps then take every other stage.
  static constexpr int kNG = (D == 64 && NT <= 2) || (D == 128 && NT == 1) ? 2 : 1;
  static constexpr int kSplit = kKeyWarps * kNG > kKeys / 16 ? kKeyWarps * kNG / (kKeys / 16) : 1;  // stages dealt to warps in turn
  static constexpr int kPosWarps = kKeyWarps / kSplit;
  static constexpr int kHalves = D == 256 ? 2 : 1;        // 128-byte column halves of a tile
  static constexpr int kTileBytes = kKeys * D;            // K (or V) of a stage
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kMT = D / 16;                      // 16-channel tiles of O^T
  static constexpr int kVecs = kMT * NT * 32;             // float4 of O of a warp
  static constexpr int kPartFloats = (kMT * NT * 4 + NT * 4) * 32;  // O, M and L of a warp, register by register
  static constexpr int kMergeBytes = kConsumers * kPartFloats * 4;
  // As many stages as fit, six at most, and a multiple of kSplit: each stage is
  // then always read by the same warps, which wait for every one of its phases
  // in turn. (A warp that skipped a stage's phase would take the parity of the
  // one before for the one it wants and read, and release, too early.)
  static constexpr int kFit = (227 * 1024 - 2048 - kMergeBytes) / kStageBytes < 6 ? (227 * 1024 - 2048 - kMergeBytes) / kStageBytes : 6;
  static constexpr int kStages = kFit / kSplit * kSplit;
  static constexpr int kSmem = kStages * kStageBytes + kMergeBytes + 1024;
};

struct StageInfo {
  float ks[kSlots], vs[kSlots];
  int live[kSlots];  // the page exists
};

// Where the x-th float4 of a part lies: two channels of two rows, as a lane's
// fragment of O^T holds them, and that lane's M and L.
template <int D, int NT, int RW>
struct Frag {
  using S = Shape<D, NT, RW>;
  int warp, lane, nt, i, at_o, at_ml;
  __device__ __forceinline__ explicit Frag(int x) {
    warp = x / S::kVecs;
    const int v = x % S::kVecs;
    lane = v & 31;
    nt = (v >> 5) % NT;
    i = (v >> 5) / NT;
    at_o = v * 4;
    at_ml = ((S::kMT * NT + nt) * 32 + lane) * 4;
  }
};

template <int D, int NT, int RW>
__device__ __forceinline__ void store(const AttnParams& p, const Item& it, const Frag<D, NT, RW>& f, const Joined& j) {
  using S = Shape<D, NT, RW>;
  constexpr int kHalfTiles = S::kMT / S::kHalves;
  const int row0 = it.rt * S::kRows + (f.warp * NT + f.nt) * 8 + 2 * (f.lane & 3);
  const int ch = f.i / kHalfTiles * 128 + (f.lane >> 2) * (2 * kHalfTiles) + 2 * (f.i % kHalfTiles);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int r = row0 + c;
    if (r >= it.rows) continue;
    const int64_t row = (int64_t)(it.t0 + r / p.group) * p.a.heads + it.h * p.group + r % p.group;
    const float L = c ? j.l1 : j.l0, inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.a.out) + row * D + ch) = out_pair((c ? j.o.y : j.o.x) * inv, (c ? j.o.w : j.o.z) * inv, p.a.a_type);
    if (p.a.lse && f.i == 0 && f.lane < 4) p.a.lse[row] = L == 0.0f ? -INFINITY : 0.6931471805599453f * ((c ? j.m1 : j.m0) + log2f(L));
  }
}

template <int FMT, int D, int NT, int RW, bool TREE>
__global__ void __launch_bounds__(kThreads, 1)
    kv_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const __grid_constant__ AttnParams p) {
  using S = Shape<D, NT, RW>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_full[S::kStages], s_empty[S::kStages];
  __shared__ StageInfo s_info[S::kStages];
  __shared__ Shared s_shared[2];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* merge = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)) + S::kStages * S::kStageBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&s_full[i], p.copy ? 1 + kProducers * 32 : 1);
      mbar_init(&s_empty[i], kConsumers / S::kSplit);
    }
    fence_barrier_init();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }

  pdl_launch_dependents();
  pdl_wait();  // all that follows may have been written by the kernel before

  Walk walk;
  int units, ctas;
  if (!find_run<kThreads>(p, S::kRows, walk, units, ctas)) return;
  const Runs runs(units, ctas);
  const int ps = p.c.page_size;
  Segment g;

  if (warp >= kConsumers) {
    // ---------------------------------------------------------- producer --
    const int pw = warp - kConsumers;
    if (pw > 0 && !p.copy) return;
    int stage = 0, issued = 0;
    uint32_t phase = 1;  // the ring starts empty
    bool ok = true;
    const int per_stage = kKeys / ps;  // pages of a stage
    const uint32_t page_bytes = (uint32_t)ps * D;
    while (ok && walk.next<TREE>(p, S::kRows, g)) {
      const int tile_lo = walk.s.tile0 + g.first, tile_hi = tile_lo + g.count;
      const int* table = p.c.page_table + (size_t)g.b * p.c.max_pages;
      // tiles with keys that some row sees
      const int from = max(tile_lo, g.lo / kKeys), to = min(tile_hi, (g.hi + kKeys - 1) / kKeys);
      // page ids and scales, a page a lane, a batch of 32 pages ahead of the
      // copies: the ids of the next batch are asked for when one begins, its
      // scales one tile later
      const int batch = 32 / per_stage;  // tiles of a batch
      auto fetch_ids = [&](int tile) {
        const int pi = tile * per_stage + lane;
        return tile < to && pi < p.c.max_pages && pi * ps < g.hi && (pi + 1) * ps > g.lo ? __ldg(table + pi) : -1;
      };
      int ids = -1, next_ids = from < to ? fetch_ids(from) : -1;
      float kss = 0.0f, vss = 0.0f, next_ks = 0.0f, next_vs = 0.0f;
      auto fetch_scales = [&]() {
        if ((unsigned)next_ids < (unsigned)p.c.num_pages) {
          const size_t ph = (size_t)next_ids * p.c.kv_heads + g.h;
          next_ks = __ldg(p.c.k_scale + ph);
          next_vs = __ldg(p.c.v_scale + ph);
        }
      };
      fetch_scales();
      for (int tile = from; tile < to && ok; ++tile) {
        const int at = (tile - from) % batch * per_stage;
        if (at == 0) {
          ids = next_ids;
          kss = next_ks;
          vss = next_vs;
          next_ids = fetch_ids(tile + batch);
        }
        const int src = at + (lane < per_stage ? lane : 0);
        const int page = __shfl_sync(0xffffffffu, ids, src);
        const bool live = lane < per_stage && (unsigned)page < (unsigned)p.c.num_pages;
        const uint32_t n_live = (uint32_t)__popc(__ballot_sync(0xffffffffu, live));
        ok = mbar_wait(&s_empty[stage], phase, ERR_WAIT_EMPTY);
        if (!ok) break;
        if (p.copy) {
          // this warp's share of the stage's pages, 512 bytes an instruction
          const uint32_t dst = smem_base + stage * S::kStageBytes;
          const unsigned live_pages = __ballot_sync(0xffffffffu, live);
          for (int sl = pw; sl < per_stage; sl += kProducers) {
            if (!((live_pages >> sl) & 1u)) continue;
            const size_t from_byte = (size_t)(__shfl_sync(0xffffffffu, ids, at + sl) * p.c.kv_heads + g.h) * page_bytes;
            const uint8_t* sk = static_cast<const uint8_t*>(p.c.k) + from_byte;
            const uint8_t* sv = static_cast<const uint8_t*>(p.c.v) + from_byte;
            for (int c = lane; c < (int)(page_bytes >> 4); c += 32) {  // 16-byte pieces of the page
              const int r = c / (8 * S::kHalves), hf = S::kHalves == 2 ? (c >> 3) & 1 : 0;  // 128-byte row and column half
              const uint32_t to = hf * (kKeys * 128) + sl * (page_bytes / S::kHalves) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
              copy16(dst + to, sk + c * 16);
              copy16(dst + S::kTileBytes + to, sv + c * 16);
            }
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&s_full[stage])) : "memory");
        } else {
          if (lane == 0 && n_live) {
            // one pending arrival stays until the scales are written below
            asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&s_full[stage])), "r"(n_live * 2 * page_bytes) : "memory");
          }
          __syncwarp();
          if (live) {
            uint8_t* dst = smem_raw + (smem_base - smem_u32(smem_raw)) + stage * S::kStageBytes;
            const int row = (page * p.c.kv_heads + g.h) * ps;  // key row of the whole pool
#pragma unroll
            for (int hf = 0; hf < S::kHalves; ++hf) {
              const int off = hf * (kKeys * 128) + lane * (int)(page_bytes / S::kHalves);
              const int y = D == 64 ? row >> 1 : row;
              tma_load_2d(dst + off, &map_k, &s_full[stage], hf * 128, y);
              tma_load_2d(dst + S::kTileBytes + off, &map_v, &s_full[stage], hf * 128, y);
            }
          }
        }
        const float ks = __shfl_sync(0xffffffffu, kss, src), vs = __shfl_sync(0xffffffffu, vss, src);
        if (at == per_stage) fetch_scales();
        if (pw == 0 && lane < kSlots) {
          s_info[stage].ks[lane] = ks;
          s_info[stage].vs[lane] = vs;
          s_info[stage].live[lane] = live;
        }
        __syncwarp();
        if (pw == 0 && lane == 0) mbar_arrive(&s_full[stage]);
        ++issued;
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (p.copy) asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok && !p.copy) {  // a wait ran out: let the copies in flight land before the CTA ends
      for (int i = 0; i < min(issued, S::kStages); ++i) {
        const int k = issued - 1 - i;
        mbar_wait(&s_full[k % S::kStages], (uint32_t)((k / S::kStages) & 1), ERR_WAIT_FULL);
      }
    }
    return;
  }

  // ------------------------------------------------------------ consumers --
  const int q4 = lane >> 2, t4 = lane & 3;  // row / column of the fragments
  const int rw = warp / S::kKeyWarps, kw = warp % S::kKeyWarps;
  // row of the group's 16 keys behind fragment row q4 (and q4 + 8): two keys
  // share a 128-byte line when D = 64, and this order keeps V's reads apart
  const int key_lo = D == 64 ? 4 * (q4 >> 1) + (q4 & 1) : q4;
  const int key_hi = D == 64 ? key_lo + 2 : q4 + 8;
  // V: keys behind this lane's operand pairs
  const int vkey[4] = {D == 64 ? 4 * t4 : 2 * t4, D == 64 ? 4 * t4 + 1 : 2 * t4 + 1, D == 64 ? 4 * t4 + 2 : 2 * t4 + 8,
                       D == 64 ? 4 * t4 + 3 : 2 * t4 + 9};
  const int kpos = kw % S::kPosWarps, turn = kw / S::kPosWarps;
  uint8_t* const ring = smem_raw + (smem_base - smem_u32(smem_raw));
  int stage = 0, count = 0;  // count: stages so far
  uint32_t phase = 0;
  bool ok = true;
  constexpr int NG = S::kNG;
  constexpr int QW = D / 8;  // 32-bit words of Q a lane and row: D / 4 channels
  uint32_t q[NT][QW];
  float cq[NT][2];
  Sight<TREE> sight[NT][2];
  const int walk_begin = walk.u;
  const bool capped = TREE && p.t.cap2 > 0.0f;
  int n_shared = 0;
  float o[S::kMT][NT][4], m[NT][2], l[NT][2];

  while (walk.next<TREE>(p, S::kRows, g)) {
    const Seq& s = walk.s;
    // queries of this lane: row q4 of each 8-row tile, channels t4 * 32 .. (D = 64: t4 * 16 ..; D = 256: in both halves)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = g.rt * S::kRows + (rw * NT + nt) * 8 + q4;
      const bool in = row < s.rows;
      const uint16_t* qp = static_cast<const uint16_t*>(p.a.q) +
                           (in ? (int64_t)(s.t0 + row / p.group) * p.a.q_token_stride + (int64_t)(g.h * p.group + row % p.group) * p.a.q_head_stride : 0);
      constexpr int W = D == 64 ? 8 : 16;  // words of a run of channels
#pragma unroll
      for (int hf = 0; hf < S::kHalves; ++hf) {
        const uint16_t* src = qp + hf * 128 + t4 * W * 2;
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) {
            if (p.vec_q) {
              v = __ldg(reinterpret_cast<const uint4*>(src + 2 * i));
            } else {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = (uint32_t)__ldg(src + 2 * (i + k)) | ((uint32_t)__ldg(src + 2 * (i + k) + 1) << 16);
              v = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          q[nt][hf * W + i] = v.x;
          q[nt][hf * W + i + 1] = v.y;
          q[nt][hf * W + i + 2] = v.z;
          q[nt][hf * W + i + 3] = v.w;
        }
      }
      float back = 1.0f;  // what the row was divided by
      if (p.a.a_type == FP8IMMA_A_BF16) {
        // bf16 -> fp16: the row is brought to a largest magnitude of 2^8 .. 2^9 by a power of two, which is exact
        // for everything within 2^22 of the largest
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < QW; ++i)
          big = fmaxf(big, fmaxf(fabsf(__uint_as_float(q[nt][i] << 16)), fabsf(__uint_as_float(q[nt][i] & 0xFFFF0000u))));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int e = (int)(__float_as_uint(big) >> 23) - 127 - 8;
        float f = 1.0f;
        if (big > 0.0f && big < INFINITY) {
          const int ec = max(-126, min(126, e));
          f = __uint_as_float((uint32_t)(127 - ec) << 23);
          back = __uint_as_float((uint32_t)(127 + ec) << 23);
        }
#pragma unroll
        for (int i = 0; i < QW; ++i) q[nt][i] = pack_f16(__uint_as_float(q[nt][i] << 16) * f, __uint_as_float(q[nt][i] & 0xFFFF0000u) * f);
      }
      // the columns 2 * t4, 2 * t4 + 1 of the S^T tiles are rows of this tile
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        cq[nt][c] = p.a.softmax_scale * 1.4426950408889634f * __shfl_sync(0xffffffffu, back, (2 * t4 + c) * 4);
        const int r = g.rt * S::kRows + (rw * NT + nt) * 8 + 2 * t4 + c;
        sight[nt][c].set(p, s, r);
        m[nt][c] = -INFINITY;
        l[nt][c] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < S::kMT; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[i][nt][c] = 0.0f;

    const int tile_lo = s.tile0 + g.first;
    const int from = max(tile_lo, g.lo / kKeys), to = min(tile_lo + g.count, (g.hi + kKeys - 1) / kKeys);
    for (int tile = from; tile < to; ++tile, ++count) {
      if (S::kSplit == 1 || count % S::kSplit == turn) {
        if (ok) ok = mbar_wait(&s_full[stage], phase, ERR_WAIT_FULL);
        const uint8_t* const kt = ring + stage * S::kStageBytes;
        const uint8_t* const vt = kt + S::kTileBytes;
#pragma unroll 1
        for (int g0 = kpos * NG; g0 < kKeys / 16; g0 += S::kPosWarps * NG) {
          // the warp's groups: which of them any row sees, whether some row does not see some key of them
          float ks[NG], lvs[NG], ivs[NG];
          bool seen[NG], any = false, edge = false;
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            const int j0 = tile * kKeys + (g0 + k) * 16, slot = (g0 + k) * 16 / ps;
            seen[k] = s_info[stage].live[slot] && j0 < g.hi && j0 + 15 >= g.lo;
            ks[k] = s_info[stage].ks[slot];
            const float vs = s_info[stage].vs[slot] < kTinyScale ? kTinyScale : s_info[stage].vs[slot];
            lvs[k] = lg2(vs);
            ivs[k] = __fdividef(1.0f, vs);
            any |= seen[k];
            edge |= !seen[k] || j0 + 15 > g.pos_min || j0 + 15 >= g.hi || (p.a.window > 0 && j0 <= g.pos_max - p.a.window);
          }
          if (!any) continue;

          // S^T = K Q^T, two chains of sums a group
          float sa[NG][NT][4], sb[NG][NT][4];
#pragma unroll
          for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c) sa[k][nt][c] = sb[k][nt][c] = 0.0f;
#pragma unroll
          for (int hf = 0; hf < S::kHalves; ++hf) {
            constexpr int W = D == 64 ? 4 : 8;  // words of K a lane and key (and half)
            uint32_t ka[NG][W], kc[NG][W];
#pragma unroll
            for (int k = 0; k < NG; ++k) {
              const int r_lo = (g0 + k) * 16 + key_lo, r_hi = (g0 + k) * 16 + key_hi;
#pragma unroll
              for (int i = 0; i < W; i += 4) {
                int xa, xc;
                if (D == 64) {
                  xa = (r_lo >> 1) * 128 + (((((r_lo & 1) << 2) + t4) ^ ((r_lo >> 1) & 7)) << 4);
                  xc = (r_hi >> 1) * 128 + (((((r_hi & 1) << 2) + t4) ^ ((r_hi >> 1) & 7)) << 4);
                } else {
                  xa = hf * (kKeys * 128) + r_lo * 128 + (((2 * t4 + i / 4) ^ (r_lo & 7)) << 4);
                  xc = hf * (kKeys * 128) + r_hi * 128 + (((2 * t4 + i / 4) ^ (r_hi & 7)) << 4);
                }
                const uint4 a = *reinterpret_cast<const uint4*>(kt + xa), c = *reinterpret_cast<const uint4*>(kt + xc);
                ka[k][i] = a.x, ka[k][i + 1] = a.y, ka[k][i + 2] = a.z, ka[k][i + 3] = a.w;
                kc[k][i] = c.x, kc[k][i + 1] = c.y, kc[k][i + 2] = c.z, kc[k][i + 3] = c.w;
              }
            }
#pragma unroll
            for (int i = 0; i < W; ++i)
#pragma unroll
              for (int k = 0; k < NG; ++k) {
                uint32_t a0, a2, a1, a3;
                f8x4_to_f16x4<FMT>(ka[k][i], a0, a2);
                f8x4_to_f16x4<FMT>(kc[k][i], a1, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma_f16(i & 1 ? sb[k][nt] : sa[k][nt], a0, a1, a2, a3, q[nt][2 * (hf * W + i)], q[nt][2 * (hf * W + i) + 1]);
              }
          }
          bool raise = false;
#pragma unroll
          for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                float x;
                if (TREE && capped) x = cap_score(p.t, (sa[k][nt][c] + sb[k][nt][c]) * (cq[nt][c & 1] * ks[k])) + lvs[k];
                else x = fmaf(sa[k][nt][c] + sb[k][nt][c], cq[nt][c & 1] * ks[k], lvs[k]);
                if (edge) {
                  const int j = tile * kKeys + (g0 + k) * 16 + (c < 2 ? key_lo : key_hi);
                  if (!seen[k] || j >= g.hi || !sight[nt][c & 1].sees(p, j)) x = -INFINITY;
                }
                sa[k][nt][c] = x;
                raise |= x > m[nt][c & 1] + kRaise;
              }
          if (__any_sync(0xffffffffu, raise)) {  // some row's maximum has moved
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float x = fmaxf(sa[0][nt][c], sa[0][nt][c + 2]);
#pragma unroll
                for (int k = 1; k < NG; ++k) x = fmaxf(x, fmaxf(sa[k][nt][c], sa[k][nt][c + 2]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                const float mn = fmaxf(m[nt][c], x);
                const float f = mn == m[nt][c] ? 1.0f : ex2(m[nt][c] - mn);
                m[nt][c] = mn;
                l[nt][c] *= f;
#pragma unroll
                for (int i = 0; i < S::kMT; ++i) {
                  o[i][nt][c] *= f;
                  o[i][nt][c + 2] *= f;
                }
              }
          }
          uint32_t pb[NG][NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float m0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1];
#pragma unroll
            for (int k = 0; k < NG; ++k) {
#pragma unroll
              for (int c = 0; c < 4; ++c) sa[k][nt][c] = ex2(sa[k][nt][c] - (c & 1 ? m1 : m0));
              l[nt][0] = fmaf(sa[k][nt][0] + sa[k][nt][2], ivs[k], l[nt][0]);
              l[nt][1] = fmaf(sa[k][nt][1] + sa[k][nt][3], ivs[k], l[nt][1]);
              pb[k][nt][0] = transpose_8x8(pack_f16(sa[k][nt][0], sa[k][nt][1]));
              pb[k][nt][1] = transpose_8x8(pack_f16(sa[k][nt][2], sa[k][nt][3]));
            }
          }

          // O^T += V^T P^T
#pragma unroll
          for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int hf = 0; hf < S::kHalves; ++hf) {
              constexpr int W = D == 64 ? 2 : 4;  // words of V a lane and key (and half): channels q4 * 4 W ..
              uint32_t v[4][W];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int r = (g0 + k) * 16 + vkey[e];
                if (D == 64) {
                  const uint2 x = *reinterpret_cast<const uint2*>(vt + (r >> 1) * 128 + (((((r & 1) << 2) + (q4 >> 1)) ^ ((r >> 1) & 7)) << 4) + (q4 & 1) * 8);
                  v[e][0] = x.x, v[e][1] = x.y;
                } else {
                  const uint4 x = *reinterpret_cast<const uint4*>(vt + hf * (kKeys * 128) + r * 128 + ((q4 ^ (r & 7)) << 4));
                  v[e][0] = x.x, v[e][1] = x.y, v[e][W - 2] = x.z, v[e][W - 1] = x.w;
                }
              }
              if (edge) {
                // a key that no row sees may hold anything, and a key that some row does not see must not reach it by 0 * NaN
                bool odd = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int j = tile * kKeys + (g0 + k) * 16 + vkey[e];
                  const bool gone = !seen[k] || j >= g.hi || j < g.lo;
#pragma unroll
                  for (int i = 0; i < W; ++i) {
                    if (gone) v[e][i] = 0u;
                    odd |= nonfinite4<FMT>(v[e][i]);
                  }
                }
                if (__any_sync(0xffffffffu, odd)) {
                  // rare: take the non-finite codes out of the product and add them to the rows that see their keys,
                  // whatever the weight (one below fp32's range is still a weight)
#pragma unroll
                  for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                      const uint32_t mk = FMT == F8_E4M3 ? 0x7F7F7F7Fu : 0x7C7C7C7Cu;
                      v[e][i] &= ~__vcmpeq4(v[e][i] & mk, mk);
                    }
#pragma unroll 1
                  for (int e = 0; e < 16; ++e) {
                    const int r = (g0 + k) * 16 + e, j = tile * kKeys + r;
                    if (j >= g.hi || j < g.lo) continue;
#pragma unroll
                    for (int i = 0; i < 2 * W; ++i)
#pragma unroll
                      for (int f = 0; f < 2; ++f) {
                        const int ch = q4 * 4 * W + 2 * i + f;  // channel within the half
                        const uint8_t byte = vt[D == 64 ? (r >> 1) * 128 + (((((r & 1) << 2) + (ch >> 4)) ^ ((r >> 1) & 7)) << 4) + (ch & 15)
                                                        : hf * (kKeys * 128) + r * 128 + (((ch >> 4) ^ (r & 7)) << 4) + (ch & 15)];
                        const float val = f8_to_f32<FMT>(byte);
                        if (!(fabsf(val) < INFINITY)) {
#pragma unroll
                          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c)
                              if (sight[nt][c].sees(p, j)) o[hf * 2 * W + i][nt][c + 2 * f] += val;
                        }
                      }
                  }
                }
              }
#pragma unroll
              for (int i = 0; i < W; ++i) {
                uint32_t a0, a1, a2, a3;
                f8x4_to_f16x4<FMT>(__byte_perm(v[0][i], v[1][i], 0x5140), a0, a1);
                f8x4_to_f16x4<FMT>(__byte_perm(v[2][i], v[3][i], 0x5140), a2, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16(o[hf * 2 * W + 2 * i][nt], a0, a1, a2, a3, pb[k][nt][0], pb[k][nt][1]);
                f8x4_to_f16x4<FMT>(__byte_perm(v[0][i], v[1][i], 0x7362), a0, a1);
                f8x4_to_f16x4<FMT>(__byte_perm(v[2][i], v[3][i], 0x7362), a2, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16(o[hf * 2 * W + 2 * i + 1][nt], a0, a1, a2, a3, pb[k][nt][0], pb[k][nt][1]);
              }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[stage]);
      }
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }

    // ------------------------------------------- join the key warps' parts --
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 4);
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 8);
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 16);
      }
    float* const mine = merge + (rw * S::kKeyWarps + kw) * S::kPartFloats;
#pragma unroll
    for (int i = 0; i < S::kMT; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        *reinterpret_cast<float4*>(mine + ((i * NT + nt) * 32 + lane) * 4) = make_float4(o[i][nt][0], o[i][nt][1], o[i][nt][2], o[i][nt][3]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      *reinterpret_cast<float4*>(mine + ((S::kMT * NT + nt) * 32 + lane) * 4) = make_float4(m[nt][0], m[nt][1], l[nt][0], l[nt][1]);
    named_bar_sync(1, kConsumers * 32);
    const Item it = {s.t0, s.rows, g.rt, g.h};
    const bool shared = g.count != s.tiles;
    float* const part = p.parts + (int64_t)(blockIdx.x * 2 + (g.item0 > walk_begin ? 1 : 0)) * RW * S::kPartFloats;
    for (int x = tid; x < RW * S::kVecs; x += kConsumers * 32) {
      const Frag<D, NT, RW> f(x);
      Joined j;
      const float* src = merge + f.warp * S::kKeyWarps * S::kPartFloats;
      j.join(S::kKeyWarps, [&](int k) { return *reinterpret_cast<const float4*>(src + k * S::kPartFloats + f.at_ml); },
             [&](int k) { return *reinterpret_cast<const float4*>(src + k * S::kPartFloats + f.at_o); });
      if (shared) {
        *reinterpret_cast<float4*>(part + f.warp * S::kPartFloats + f.at_o) = j.o;
        if (f.i == 0) *reinterpret_cast<float4*>(part + f.warp * S::kPartFloats + f.at_ml) = make_float4(j.m0, j.m1, j.l0, j.l1);
      } else {
        store<D, NT, RW>(p, it, f, j);
      }
    }
    if (shared && tid == 0) {
      s_shared[n_shared].item = it;
      s_shared[n_shared].index = g.item;
      s_shared[n_shared].c0 = runs.of(g.item0);
      s_shared[n_shared].c1 = runs.of(g.item0 + s.tiles - 1);
      s_shared[n_shared].item0 = g.item0;
    }
    n_shared += shared;
    named_bar_sync(1, kConsumers * 32);  // the merge buffer is free again
  }

  // Shared items (the run's first and last at most): the CTA that comes last
  // to an item joins all its parts, in CTA order.
  if (n_shared == 0) return;
  __threadfence();
  named_bar_sync(1, kConsumers * 32);
  if (tid < n_shared) {
    unsigned int prev, *ctr = p.counters + s_shared[tid].index;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(prev) : "l"(ctr) : "memory");
    s_shared[tid].last = prev == (unsigned)(s_shared[tid].c1 - s_shared[tid].c0);
    if (s_shared[tid].last) *ctr = 0;  // ready for the next call
  }
  named_bar_sync(1, kConsumers * 32);
  __threadfence();
  for (int k = 0; k < n_shared; ++k) {
    const Shared& sh = s_shared[k];
    if (!sh.last) continue;
    for (int x = tid; x < RW * S::kVecs; x += kConsumers * 32) {
      const Frag<D, NT, RW> f(x);
      Joined j;
      // a CTA's part of the item lies in its slot 0 when its run begins within the item
      auto src = [&](int c) {
        c += sh.c0;
        return p.parts + ((int64_t)(c * 2 + (sh.item0 > runs.begin(c) ? 1 : 0)) * RW + f.warp) * S::kPartFloats;
      };
      j.join(sh.c1 - sh.c0 + 1, [&](int c) { return __ldcg(reinterpret_cast<const float4*>(src(c) + f.at_ml)); },
             [&](int c) { return __ldcg(reinterpret_cast<const float4*>(src(c) + f.at_o)); });
      store<D, NT, RW>(p, sh.item, f, j);
    }
  }
}

template <int FMT, int D, int NT, int RW, bool TREE>
cudaError_t launch(AttnParams& p, cudaStream_t st) {
  using S = Shape<D, NT, RW>;
  static_assert(S::kStages >= 2 && S::kStages % S::kSplit == 0, "ring too short, or stages change hands");
  const auto kern = kv_attention_kernel<FMT, D, NT, RW, TREE>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), S::kSmem);
  if (e != cudaSuccess) return e;
  // 128-byte rows: two keys a row when D = 64, half a key when D = 256
  CUtensorMap mk, mv;
  const uint64_t bytes = (uint64_t)p.c.num_pages * p.c.kv_heads * p.c.page_size * D;
  const uint64_t inner = D == 256 ? 256 : 128;
  const uint32_t box_rows = (uint32_t)(D == 64 ? p.c.page_size / 2 : p.c.page_size);
  e = make_tmap_2d_u8(&mk, p.c.k, inner, bytes / inner, inner, 128, box_rows, true);
  if (e == cudaSuccess) e = make_tmap_2d_u8(&mv, p.c.v, inner, bytes / inner, inner, 128, box_rows, true);
  if (e != cudaSuccess) return e;
  const int64_t items = ((int64_t)p.c.tokens * p.group / S::kRows + p.c.batch) * p.c.kv_heads;
  const int64_t tiles = ((int64_t)p.c.max_pages * p.c.page_size + kKeys - 1) / kKeys;
  if (items * tiles > 0x7fffffffll) return cudaErrorInvalidValue;  // units are counted in 31 bits
  const int grid = (int)std::min<int64_t>(num_sms_current(), std::max<int64_t>(1, items * tiles));
  p.copy = p.c.page_size * (D == 256 ? 128 : D) < 4096;
  const size_t ctr_bytes = (size_t)items * 4, part_bytes = (size_t)grid * 2 * RW * S::kPartFloats * 4;
  ScopedScratch ctr, part;
  if (TREE) {
    const cudaError_t c = ctr.own_if_captured(st), d = part.own_if_captured(st);
    if (c != cudaSuccess || d != cudaSuccess) return c != cudaSuccess ? c : d;
  }
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
    e = cudaLaunchKernelEx(&lc, kern, mk, mv, p);
  }
  const cudaError_t e1 = ctr.release(st), e2 = part.release(st);
  return e != cudaSuccess ? e : e1 != cudaSuccess ? e1 : e2;
}

// Query rows a CTA works on at once: the rows of a sequence and KV head
// (group times its tokens, on average) rounded up, so that few rows do not pay
// for empty ones and many rows read the cache once.
template <int FMT, bool TREE>
cudaError_t launch_d(AttnParams& p, cudaStream_t st) {
  const int64_t rows = ((int64_t)p.c.tokens * p.group + p.c.batch - 1) / p.c.batch;
  // Where tiles of 8 rows leave SMs free, each takes a CTA of its own, whose eight
  // warps share the keys: a small tree over a short context is a chain of latencies.
  // Up to the border it won at each of 102 shapes (16 to 512 rows, 200 to 8000 keys,
  // 1 to 8 KV heads); this / as many rows a CTA as below / tcgen05 in us, tiles of 8
  // rows in brackets: 64 channels, 256 rows, 200 keys, 4 heads [256] 10.3/19.8/20.4;
  // 128 channels, 32 rows, 700 keys, 8 heads [192] 11.2/16.4/23.4, 32 rows, 8000
  // keys, 1 head [252] 21.9/37.2/60.7; 256 channels, 128 rows, 2000 keys, 1 head [256]
  // 15.1/54.8. The causal operator keeps to its order of sums.
  if (TREE && rows > 8 && attention_tc_forced() == 0) {
    const int64_t tiles = ((int64_t)p.c.max_pages * p.c.page_size + kKeys - 1) / kKeys * p.c.batch * p.c.kv_heads;
    if (tiles * ((rows + 7) / 8) <= 2ll * num_sms_current()) {
      if (p.c.head_dim == 256) return launch<FMT, 256, 1, 1, TREE>(p, st);
      return p.c.head_dim == 128 ? launch<FMT, 128, 1, 1, TREE>(p, st) : launch<FMT, 64, 1, 1, TREE>(p, st);
    }
  }
  if (attention_tc_pays(p, rows)) return TREE ? launch_attention_tree_tc(p, st) : launch_attention_tc(p, st);
  if (p.c.head_dim == 256) {
    if (rows <= 8) return launch<FMT, 256, 1, 1, TREE>(p, st);
    if (rows <= 16) return launch<FMT, 256, 1, 2, TREE>(p, st);
    if (rows <= 32) return launch<FMT, 256, 1, 4, TREE>(p, st);
    return launch<FMT, 256, 1, 8, TREE>(p, st);
  }
  if (p.c.head_dim == 128) {
    if (rows <= 8) return launch<FMT, 128, 1, 1, TREE>(p, st);
    if (rows <= 16) return launch<FMT, 128, 2, 1, TREE>(p, st);
    if (rows <= 32) return launch<FMT, 128, 1, 4, TREE>(p, st);
    return launch<FMT, 128, 2, 4, TREE>(p, st);
  }
  if (rows <= 8) return launch<FMT, 64, 1, 1, TREE>(p, st);
  if (rows <= 16) return launch<FMT, 64, 2, 1, TREE>(p, st);
  if (rows <= 32) return launch<FMT, 64, 2, 2, TREE>(p, st);
  return launch<FMT, 64, 2, 4, TREE>(p, st);
}

}  // namespace
}  // namespace fp8imma_b200
