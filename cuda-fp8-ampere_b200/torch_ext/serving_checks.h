// Checks of arguments shared by the bindings of the decode-step operators
// (serving_ops.cpp, layer_ops.cpp).
#pragma once

#include <torch/extension.h>

#include <string>

#include "fp8imma/fp8imma_ext.h"

namespace fp8imma_torch {

inline void check_launch(int err, const char* what) { TORCH_CHECK(err == 0, what, " failed, cudaError_t=", err); }

inline int act_type(const torch::Tensor& x, const char* name) {
  if (x.scalar_type() == at::kHalf) return FP8IMMA_A_F16;
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, name, " must be fp16 or bf16");
  return FP8IMMA_A_BF16;
}

inline int byte_format(const std::string& f, const char* name) {
  if (f == "e4m3") return FP8IMMA_B_E4M3;
  TORCH_CHECK(f == "e5m2", name, " must be 'e4m3' or 'e5m2'");
  return FP8IMMA_B_E5M2;
}

inline bool is_bytes(const torch::Tensor& x) {
  const auto t = x.scalar_type();
  return t == at::kByte || t == at::kFloat8_e4m3fn || t == at::kFloat8_e5m2;
}

// bytes of any dtype that does not name the other format
inline void check_format(const torch::Tensor& x, int format, const char* name) {
  const auto t = x.scalar_type();
  TORCH_CHECK(t == at::kByte || t == (format == FP8IMMA_B_E4M3 ? at::kFloat8_e4m3fn : at::kFloat8_e5m2), name, " is ", t,
              ", but the format asked for is ", format == FP8IMMA_B_E4M3 ? "'e4m3'" : "'e5m2'");
}

inline void check_on(const torch::Tensor& x, const torch::Tensor& like, const char* name) {
  TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(x.device() == like.device(), name, " must be on ", like.device());
}

inline void check_packed(const torch::Tensor& x, const torch::Tensor& like, at::ScalarType dt, const char* name) {
  check_on(x, like, name);
  TORCH_CHECK(x.scalar_type() == dt, name, " must be ", dt);
  TORCH_CHECK(x.is_contiguous(), name, " must be contiguous");
}

inline int to_int(int64_t v, const char* name) {
  TORCH_CHECK(v >= 0 && v <= 0x7fffffffll, name, " is out of range");
  return (int)v;
}

inline fp8imma_kv_cache cache_args(const torch::Tensor& rows, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                            const torch::Tensor& k_scale, const torch::Tensor& v_scale, const torch::Tensor& page_table,
                            const torch::Tensor& seq_lens, const c10::optional<torch::Tensor>& cu_seqlens,
                            const std::string& fmt) {
  fp8imma_kv_cache c = {};
  c.format = byte_format(fmt, "fmt");
  for (const auto* x : {&k_cache, &v_cache}) {
    check_on(*x, rows, "k_cache / v_cache");
    TORCH_CHECK(is_bytes(*x) && x->dim() == 4 && x->is_contiguous(),
                "k_cache / v_cache must be contiguous uint8 [num_pages, kv_heads, page_size, head_dim]");
    check_format(*x, c.format, "k_cache / v_cache");
  }
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache must have the same shape");
  for (const auto* x : {&k_scale, &v_scale}) {
    check_packed(*x, rows, at::kFloat, "k_scale / v_scale");
    TORCH_CHECK(x->dim() == 2 && x->size(0) == k_cache.size(0) && x->size(1) == k_cache.size(1),
                "k_scale / v_scale must have shape [num_pages, kv_heads]");
  }
  check_packed(page_table, rows, at::kInt, "page_table");
  check_packed(seq_lens, rows, at::kInt, "seq_lens");
  TORCH_CHECK(page_table.dim() == 2, "page_table must have shape [batch, max_pages]");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == page_table.size(0), "seq_lens must have shape [batch]");
  c.k = k_cache.data_ptr();
  c.v = v_cache.data_ptr();
  c.k_scale = k_scale.data_ptr<float>();
  c.v_scale = v_scale.data_ptr<float>();
  c.page_table = page_table.data_ptr<int>();
  c.seq_lens = seq_lens.data_ptr<int>();
  c.num_pages = to_int(k_cache.size(0), "num_pages");
  c.kv_heads = to_int(k_cache.size(1), "kv_heads");
  c.page_size = to_int(k_cache.size(2), "page_size");
  c.head_dim = to_int(k_cache.size(3), "head_dim");
  TORCH_CHECK(c.page_size == 16 || c.page_size == 32 || c.page_size == 64 || c.page_size == 128,
              "page_size must be 16, 32, 64 or 128");
  TORCH_CHECK(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, "head_dim must be 64, 128 or 256");
  c.batch = to_int(page_table.size(0), "batch");
  c.max_pages = to_int(page_table.size(1), "max_pages");
  c.tokens = to_int(rows.size(0), "tokens");
  if (cu_seqlens.has_value()) {
    check_packed(*cu_seqlens, rows, at::kInt, "cu_seqlens");
    TORCH_CHECK(cu_seqlens->dim() == 1 && cu_seqlens->size(0) == page_table.size(0) + 1,
                "cu_seqlens must have shape [batch + 1]");
    c.cu_new = cu_seqlens->data_ptr<int>();
  } else {
    TORCH_CHECK(c.batch > 0 && c.tokens % c.batch == 0, "without cu_seqlens every sequence has tokens / batch tokens");
  }
  return c;
}

}  // namespace fp8imma_torch
