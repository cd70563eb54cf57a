// The C entry of the cache attention (fp8imma_kv_attention) and the rule between
// its two kernels (kv_attention_few.cuh, kv_attention_tc.cu).
#include "kv_attention_few.cuh"
#include "nvtx_range.h"

#include <atomic>

namespace fp8imma_b200 {
namespace {

std::atomic<int> g_tc_rows{0};  // rows from which tcgen05 is used, 0: by attention_tc_pays()

}  // namespace

// Whether rows and tiles are enough for the tcgen05 kernel (kv_attention_tc.cu).
// Its tile of up to 128 rows costs much the same whatever the rows (1.7 us a tile
// and SM at 128 channels, 1.3 at 64) and a call about 10 us more than here (TMEM, a
// deeper pipeline); here a tile costs by the rows that launch_d() rounds them up to:
// 128 channels 2.3 us with 32 rows, 4.4 with 64, as much again for each further 64;
// about half of that at 64 channels. With up to 16 rows (32 of 64 channels) it never
// pays, with up to twice as many from 16 (8) tiles an SM on, with more from 1.5 on.
// Measured, this kernel against that one, in us, tiles an SM in brackets:
//   128 channels, 16 rows: [28] 53/76, [221] 308/468
//     24 rows: [7] 36/42, [14] 52/53, [17] 62/60, [28] 84/78, [221] 541/472
//     40 rows: [0.9] 32/31, [1.7] 29/27, [7] 61/42, [28] 154/79, [221] 1033/477
//     128 rows: [0.9] 35/41, [1.7] 49/33, [14] 146/70;  512 rows: [14] 169/78
//   64 channels, 28 rows: [14] 37/46, [111] 186/207
//     35 rows: [3.5] 29/31, [7] 40/39, [9] 45/40, [111] 332/207
//     112 rows: [1.3] 26/30, [1.7] 31/28, [9] 70/44
// Tiles are counted by what the page tables can hold, since lengths lie on the
// device: under a table for 131072 keys, 24 rows of 8 sequences of 300 take 30 us
// there where they would take 24 here, of 32 sequences of 1000 64 for 56.
bool attention_tc_pays(const AttnParams& p, int64_t rows) {
  const int D = p.c.head_dim;
  if (D == 256) return false;
  const int forced = g_tc_rows.load();
  if (forced > 0) return rows >= forced;
  const int none = D == 64 ? 32 : 16;
  if (rows <= none) return false;
  int64_t keys = (int64_t)p.c.max_pages * p.c.page_size;
  if (p.a.window > 0) keys = std::min<int64_t>(keys, (int64_t)p.a.window + rows / p.group + kKeys);
  const int64_t tiles = (keys + kKeys - 1) / kKeys * ((rows + 127) / 128) * p.c.batch * p.c.kv_heads;
  return 2 * tiles >= (rows <= 2 * none ? (D == 64 ? 16 : 32) : 3) * (int64_t)num_sms_current();
}

void attn_set_tc_rows(int rows) { g_tc_rows.store(rows); }
int attention_tc_forced() { return g_tc_rows.load(); }
unsigned int attn_device_error(bool clear) { return fp8imma_dev::tu_device_error(clear); }
cudaError_t attn_set_wait_limit(unsigned long long ns) { return fp8imma_dev::tu_set_wait_limit(ns); }

}  // namespace fp8imma_b200

using namespace fp8imma_b200;

extern "C" int fp8imma_kv_attention(const fp8imma_kv_cache* c, const fp8imma_kv_attention_args* a, void* stream) {
  FP8IMMA_RANGE("fp8imma_kv_attention");
  const cudaError_t e = kv_cache_check(c);
  if (e != cudaSuccess) return (int)e;
  if (!a || !a->q || !a->out || a->a_type < 0 || a->a_type > 1) return (int)cudaErrorInvalidValue;
  if (a->heads <= 0 || a->heads % c->kv_heads || a->heads > 65535 || a->window < 0) return (int)cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a->q) & 1u) || !aligned4({a->lse})) return (int)cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(a->out) & 15u) return (int)cudaErrorInvalidValue;
  if ((int64_t)c->tokens * (a->heads / c->kv_heads) > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  AttnParams p = {};
  p.c = *c;
  p.a = *a;
  p.per_seq = c->cu_new ? 0 : c->tokens / c->batch;
  p.group = a->heads / c->kv_heads;
  p.vec_q = ((reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)((a->q_token_stride | a->q_head_stride) * 2)) & 15u) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return (int)(c->format == FP8IMMA_B_E4M3 ? launch_d<F8_E4M3, false>(p, st) : launch_d<F8_E5M2, false>(p, st));
}
