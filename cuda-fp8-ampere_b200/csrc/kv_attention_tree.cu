// Attention over the paged 8-bit cache for the nodes of drafted trees, with capped
// scores (fp8imma_kv_attention_tree). The kernels are those of the causal attention
// (kv_attention_few.cuh, kv_attention_tc.cu) in variants of their own (TREE):
//   x_rj = cap tanh(s_rj / cap),  s_rj = softmax_scale <q_r, K_j>,
// and in the tiles that hold keys of the step a row's mask bits decide what it
// sees. All tiles before those are multiplied as in the causal attention.
//
// Measured (one B200): 32 sequences of up to 8192 keys, 64/8 heads of 128, up to 16
// nodes, capped 275 to 314 us by the board; two documents of up to 100000 keys, 64 nodes
// of 32/8 heads, capped 379 to 410. Two of 100000 each: 378 us without a cap, 476 with all
// scores within it, 640 where every tile holds some beyond it. One sequence of 700
// keys, 8 nodes of 32/8 heads 11 us.
#include "kv_attention_few.cuh"
#include "nvtx_range.h"

#include <cmath>

namespace fp8imma_b200 {

unsigned int attn_tree_device_error(bool clear) { return fp8imma_dev::tu_device_error(clear); }
cudaError_t attn_tree_set_wait_limit(unsigned long long ns) { return fp8imma_dev::tu_set_wait_limit(ns); }

}  // namespace fp8imma_b200

using namespace fp8imma_b200;

extern "C" int fp8imma_kv_attention_tree(const fp8imma_kv_cache* c, const fp8imma_kv_attention_tree_args* a, void* stream) {
  FP8IMMA_RANGE("fp8imma_kv_attention_tree");
  const cudaError_t e = kv_cache_check(c);
  if (e != cudaSuccess) return (int)e;
  if (!a || !a->q || !a->out || a->a_type < 0 || a->a_type > 1) return (int)cudaErrorInvalidValue;
  if (a->heads <= 0 || a->heads % c->kv_heads || a->heads > 65535 || a->window < 0) return (int)cudaErrorInvalidValue;
  if (!(a->softcap >= 0.0f) || !std::isfinite(a->softcap) || !std::isfinite(a->softmax_scale)) return (int)cudaErrorInvalidValue;
  if ((a->tree_mask && a->mask_words <= 0) || (a->positions && !a->tree_mask)) return (int)cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a->q) & 1u) || !aligned4({a->tree_mask, a->positions, a->lse})) return (int)cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(a->out) & 15u) return (int)cudaErrorInvalidValue;
  if ((int64_t)c->tokens * (a->heads / c->kv_heads) > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  AttnParams p = {};
  p.c = *c;
  p.a.a_type = a->a_type;
  p.a.heads = a->heads;
  p.a.window = a->window;
  p.a.softmax_scale = a->softmax_scale;
  p.a.q = a->q;
  p.a.q_token_stride = a->q_token_stride;
  p.a.q_head_stride = a->q_head_stride;
  p.a.out = a->out;
  p.a.lse = a->lse;
  p.t.mask = a->tree_mask;
  p.t.positions = a->positions;
  p.t.words = a->mask_words;
  attn::set_cap(p.t, a->softcap);
  p.per_seq = c->cu_new ? 0 : c->tokens / c->batch;
  p.group = a->heads / c->kv_heads;
  p.vec_q = ((reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)((a->q_token_stride | a->q_head_stride) * 2)) & 15u) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return (int)(c->format == FP8IMMA_B_E4M3 ? launch_d<F8_E4M3, true>(p, st) : launch_d<F8_E5M2, true>(p, st));
}
