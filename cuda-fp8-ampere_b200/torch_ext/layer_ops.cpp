// PyTorch binding of the operators between a step's products (module
// fp8imma_ext): the residual connection with its norms (residual_norm),
// low-rank adapters (lora_add), the cache's append with the position rotation
// (kv_append_rope) and its attention for drafted trees (kv_attention_tree).
// Arguments and results are documented at the C entry points in
// include/fp8imma/fp8imma_ext.h; each call runs on the current stream of its
// tensors' device.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <string>
#include <tuple>

#include "serving_checks.h"

namespace {

using namespace fp8imma_torch;
using OptTensor = c10::optional<torch::Tensor>;

// A result, straight from the allocator: on the smallest calls the dispatcher's
// way to it costs as much as the kernel (1 us each).
torch::Tensor fresh(const torch::Tensor& like, c10::IntArrayRef sizes, at::ScalarType dt) {
  return at::detail::empty_cuda(sizes, dt, like.device(), c10::nullopt);
}

int real_type(const torch::Tensor& x, const char* name) {
  if (x.scalar_type() == at::kHalf) return FP8IMMA_L_F16;
  if (x.scalar_type() == at::kBFloat16) return FP8IMMA_L_BF16;
  TORCH_CHECK(x.scalar_type() == at::kFloat, name, " must be fp16, bf16 or fp32");
  return FP8IMMA_L_F32;
}

// an output may be the input itself (same address and strides), but not lie across it
void check_apart(const torch::Tensor& out, const torch::Tensor& in, const char* what, bool itself = true) {
  if (!out.numel() || !in.numel()) return;
  if (itself && out.data_ptr() == in.data_ptr() && out.strides() == in.strides() && out.scalar_type() == in.scalar_type()) return;
  auto end = [](const torch::Tensor& x) {
    int64_t n = 1;
    for (int64_t d = 0; d < x.dim(); ++d) n += (x.size(d) - 1) * x.stride(d);
    return static_cast<const char*>(x.data_ptr()) + n * x.element_size();
  };
  TORCH_CHECK(end(out) <= static_cast<const char*>(in.data_ptr()) || end(in) <= static_cast<const char*>(out.data_ptr()), what);
}

// Whether rows (t, h) of x and y, [tokens, heads, dim] of one type with contiguous last
// dimensions, share an element; with `other` false a row does not meet itself. Slices of
// one buffer may lie in turn with one another.
bool rows_meet(const torch::Tensor& x, const torch::Tensor& y, bool other = true) {
  const int64_t T = x.size(0), D = x.size(2), Hx = x.size(1), Hy = y.size(1);
  if (!x.numel() || !y.numel()) return false;
  const int64_t off = (static_cast<const char*>(x.data_ptr()) - static_cast<const char*>(y.data_ptr())) / (int64_t)x.element_size();
  // a dimension of one element has no stride of its own
  const int64_t hx = Hx == 1 ? 0 : x.stride(1), hy = Hy == 1 ? 0 : y.stride(1), sx = T == 1 ? 0 : x.stride(0), sy = T == 1 ? 0 : y.stride(0);
  const int64_t lx = (Hx - 1) * hx + D, ly = (Hy - 1) * hy + D;  // a token's span
  if (off + (T - 1) * sx + lx <= 0 || off >= (T - 1) * sy + ly) return false;
  if (sx != sy) return true;  // not told apart
  if (other && sx >= std::max(lx, ly)) {  // spans within the token stride: apart in the first tokens is apart in all
    const int64_t r = ((off % sx) + sx) % sx;
    if (r >= ly && r + lx <= sx) return false;
  }
  // heads within tokens, or tokens within heads
  if (!other && ((T == 1 || sx >= lx) && (Hx == 1 || hx >= D))) return false;
  if (!other && ((Hx == 1 || hx >= (T - 1) * sx + D) && (T == 1 || sx >= D))) return false;
  for (int64_t i = 0; i < Hx; ++i)
    for (int64_t j = 0; j < Hy; ++j) {
      // rows i and j of tokens dt apart, where they come nearest
      const int64_t at = off + i * hx - j * hy, dt0 = sx ? std::clamp(-at / sx, 1 - T, T - 1) : 0;
      for (int64_t dt = std::max(dt0 - 1, 1 - T); dt <= std::min(dt0 + 1, T - 1); ++dt)
        if (std::abs(at + dt * sx) < D && (other || i != j || dt != 0)) return true;
    }
  return false;
}

// a [tokens, hidden] tensor with contiguous rows; its row stride
int64_t rows_of(const torch::Tensor& x, const torch::Tensor& like, const char* name) {
  check_on(x, like, name);
  TORCH_CHECK(x.dim() == 2 && x.sizes() == like.sizes(), name, " must be shaped like y");
  TORCH_CHECK(x.size(1) == 1 || x.stride(1) == 1, "the last dimension of ", name, " must be contiguous");
  return x.size(0) == 1 ? x.size(1) : x.stride(0);
}

std::tuple<torch::Tensor, OptTensor> residual_norm(const torch::Tensor& y, const OptTensor& residual, const OptTensor& post_weight,
                                                   const OptTensor& pre_weight, const OptTensor& gate, double alpha, double eps,
                                                   double weight_offset, const OptTensor& residual_out, const OptTensor& out) {
  TORCH_CHECK(y.is_cuda(), "y must be a CUDA tensor");
  fp8imma_residual_norm_args a = {};
  a.a_type = act_type(y, "y");
  a.y_stride = rows_of(y, y, "y");
  const int64_t T = y.size(0), H = y.size(1);
  TORCH_CHECK(H >= 1 && H <= FP8IMMA_NORM_MAX_HIDDEN, "hidden must be 1 .. ", FP8IMMA_NORM_MAX_HIDDEN);
  a.r_type = residual.has_value() ? real_type(*residual, "residual") : residual_out.has_value() ? real_type(*residual_out, "residual_out") : a.a_type;
  TORCH_CHECK(a.r_type == a.a_type || a.r_type == FP8IMMA_L_F32, "residual must have y's dtype or fp32");
  if (residual.has_value()) a.residual_stride = rows_of(*residual, y, "residual");
  if (gate.has_value()) {
    check_on(*gate, y, "gate");
    a.g_type = real_type(*gate, "gate");
    if (gate->dim() == 2) a.gate_stride = rows_of(*gate, y, "gate");
    else TORCH_CHECK(gate->dim() == 1 && gate->size(0) == H && gate->is_contiguous(), "gate must have shape [hidden] or [tokens, hidden]");
  }
  a.w_type = a.a_type;
  for (const auto* w : {&post_weight, &pre_weight}) {
    if (!w->has_value()) continue;
    check_on(**w, y, "post_weight / pre_weight");
    TORCH_CHECK((*w)->dim() == 1 && (*w)->size(0) == H && (*w)->is_contiguous(), "post_weight / pre_weight must have shape [hidden]");
    a.w_type = real_type(**w, "post_weight / pre_weight");
  }
  TORCH_CHECK(!post_weight.has_value() || !pre_weight.has_value() || post_weight->scalar_type() == pre_weight->scalar_type(),
              "post_weight and pre_weight must have the same dtype");
  TORCH_CHECK(!out.has_value() || pre_weight.has_value(), "out is written with pre_weight only");
  a.alpha = (float)alpha;
  a.eps = (float)eps;
  a.weight_offset = (float)weight_offset;
  TORCH_CHECK(std::isfinite(a.alpha) && std::isfinite(a.weight_offset), "alpha and weight_offset must be finite");
  TORCH_CHECK(a.eps >= 0 && std::isfinite(a.eps), "eps must not be negative");
  const c10::cuda::CUDAGuard guard(y.device());
  torch::Tensor r;
  if (residual_out.has_value()) {
    r = *residual_out;
    check_on(r, y, "residual_out");
    TORCH_CHECK(real_type(r, "residual_out") == a.r_type, "residual_out must have residual's dtype");
    TORCH_CHECK(r.sizes() == y.sizes() && r.is_contiguous(), "residual_out must be contiguous and shaped like y");
  } else {
    r = fresh(y, y.sizes(), a.r_type == FP8IMMA_L_F32 ? at::kFloat : y.scalar_type());
  }
  OptTensor h;
  if (pre_weight.has_value()) {
    if (out.has_value()) {
      h = *out;
      check_packed(*h, y, y.scalar_type(), "out");
      TORCH_CHECK(h->sizes() == y.sizes(), "out must be shaped like y");
    } else {
      h = fresh(y, y.sizes(), y.scalar_type());
    }
  }
  const char* across = "residual_out and out must be the inputs themselves or lie apart from them";
  for (const torch::Tensor* o : {&r, h.has_value() ? &*h : &r}) {
    check_apart(*o, y, across);
    if (residual.has_value()) check_apart(*o, *residual, across);
    for (const auto* x : {&gate, &post_weight, &pre_weight})
      if (x->has_value()) check_apart(*o, **x, across, false);
  }
  if (h.has_value()) check_apart(*h, r, "residual_out and out must lie apart", false);
  if (T == 0) return {r, h};
  a.tokens = to_int(T, "tokens");
  a.hidden = (int)H;
  a.y = y.data_ptr();
  a.residual = residual.has_value() ? residual->data_ptr() : nullptr;
  a.gate = gate.has_value() ? gate->data_ptr() : nullptr;
  a.post_weight = post_weight.has_value() ? post_weight->data_ptr() : nullptr;
  a.pre_weight = pre_weight.has_value() ? pre_weight->data_ptr() : nullptr;
  a.residual_out = r.data_ptr();
  a.out = h.has_value() ? h->data_ptr() : nullptr;
  check_launch(fp8imma_residual_norm(&a, (void*)at::cuda::getCurrentCUDAStream()), "fp8imma_residual_norm");
  return {r, h};
}

torch::Tensor lora_add(const torch::Tensor& base, const torch::Tensor& x, const torch::Tensor& lora_a, const torch::Tensor& lora_b,
                       const torch::Tensor& adapter_ids, const OptTensor& scales, const OptTensor& out) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  fp8imma_lora_args a = {};
  a.a_type = act_type(x, "x");
  TORCH_CHECK(x.dim() == 2 && (x.size(1) == 1 || x.stride(1) == 1), "x must be [tokens, in_features] with contiguous rows");
  const int64_t T = x.size(0), K = x.size(1);
  check_packed(lora_a, x, x.scalar_type(), "lora_a");
  check_packed(lora_b, x, x.scalar_type(), "lora_b");
  TORCH_CHECK(lora_a.dim() == 3 && lora_a.size(2) == K, "lora_a must have shape [adapters, rank, in_features]");
  const int64_t L = lora_a.size(0), R = lora_a.size(1);
  TORCH_CHECK(lora_b.dim() == 3 && lora_b.size(0) == L && lora_b.size(2) == R, "lora_b must have shape [adapters, out_features, rank]");
  const int64_t N = lora_b.size(1);
  TORCH_CHECK(L >= 1 && N >= 1 && K >= 1, "lora_a / lora_b must not be empty");
  TORCH_CHECK(R >= 8 && R <= FP8IMMA_LORA_MAX_RANK && R % 8 == 0, "rank must be a multiple of 8, at most ", FP8IMMA_LORA_MAX_RANK);
  TORCH_CHECK(K % 8 == 0, "in_features must be a multiple of 8");
  check_packed(adapter_ids, x, at::kInt, "adapter_ids");
  TORCH_CHECK(adapter_ids.dim() == 1 && adapter_ids.size(0) == T, "adapter_ids must have shape [tokens]");
  if (scales.has_value()) {
    check_packed(*scales, x, at::kFloat, "scales");
    TORCH_CHECK(scales->dim() == 1 && scales->size(0) == L, "scales must have shape [adapters]");
  }
  check_on(base, x, "base");
  a.d_type = act_type(base, "base");
  TORCH_CHECK(base.dim() == 2 && base.size(0) == T && base.size(1) == N, "base must have shape [tokens, out_features]");
  // contiguous along one dimension, the other's lines apart
  auto layout = [&](const torch::Tensor& t, bool& row, bool& col) {
    row = (N == 1 || t.stride(1) == 1) && (T == 1 || t.stride(0) >= N);
    col = (T == 1 || t.stride(0) == 1) && (N == 1 || t.stride(1) >= T);
  };
  bool row, col;
  layout(base, row, col);
  TORCH_CHECK(row || col, "base must be contiguous along one dimension");
  const c10::cuda::CUDAGuard guard(x.device());
  torch::Tensor o;
  if (out.has_value()) {
    o = *out;
    check_on(o, x, "out");
    TORCH_CHECK(o.scalar_type() == base.scalar_type() && o.sizes() == base.sizes(), "out must have base's shape and dtype");
    bool orow, ocol;
    layout(o, orow, ocol);
    TORCH_CHECK((row && orow) || (col && ocol), "out must be contiguous along the same dimension as base");
    row = row && orow;
    const char* across = "out must be base itself or lie apart from the inputs";
    check_apart(o, base, across);
    for (const auto* t : {&x, &lora_a, &lora_b}) check_apart(o, *t, across, false);
  } else if (row) {
    o = fresh(base, {T, N}, base.scalar_type());
  } else {
    o = at::detail::empty_strided_cuda({T, N}, {1, T}, base.scalar_type(), base.device());
  }
  if (T == 0) return o;
  a.tokens = to_int(T, "tokens");
  a.in_features = to_int(K, "in_features");
  a.out_features = to_int(N, "out_features");
  a.rank = (int)R;
  a.adapters = to_int(L, "adapters");
  a.x = x.data_ptr();
  a.x_stride = T == 1 ? K : x.stride(0);
  TORCH_CHECK(a.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0, "rows of x must be 16-byte aligned");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(lora_a.data_ptr()) | reinterpret_cast<uintptr_t>(lora_b.data_ptr())) % 16 == 0,
              "lora_a / lora_b must be 16-byte aligned");
  a.lora_a = lora_a.data_ptr();
  a.lora_b = lora_b.data_ptr();
  a.adapter_ids = adapter_ids.data_ptr<int>();
  a.scales = scales.has_value() ? scales->data_ptr<float>() : nullptr;
  a.base = base.data_ptr();
  a.out = o.data_ptr();
  // a dimension of one element has no stride of its own
  auto strides = [&](const torch::Tensor& t, int64_t& ts, int64_t& fs) {
    ts = row ? (T == 1 ? N : t.stride(0)) : 1;
    fs = row ? 1 : (N == 1 ? T : t.stride(1));
  };
  strides(base, a.base_token_stride, a.base_feature_stride);
  strides(o, a.out_token_stride, a.out_feature_stride);
  check_launch(fp8imma_lora_add(&a, (void*)at::cuda::getCurrentCUDAStream()), "fp8imma_lora_add");
  return o;
}

OptTensor kv_append_rope(const OptTensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& k_cache,
                         const torch::Tensor& v_cache, const torch::Tensor& k_scale, const torch::Tensor& v_scale,
                         const torch::Tensor& page_table, const torch::Tensor& seq_lens, const torch::Tensor& inv_freq,
                         const OptTensor& cu_seqlens, const OptTensor& positions, double rope_scale, bool interleaved,
                         const std::string& fmt, const OptTensor& q_out) {
  TORCH_CHECK(k.is_cuda(), "k must be a CUDA tensor");
  check_on(v, k, "v");
  fp8imma_kv_append_rope_args a = {};
  a.a_type = act_type(k, "k");
  TORCH_CHECK(v.scalar_type() == k.scalar_type(), "k and v must have the same dtype");
  const fp8imma_kv_cache c = cache_args(k, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cu_seqlens, fmt);
  TORCH_CHECK(k.dim() == 3 && k.size(1) == c.kv_heads && k.size(2) == c.head_dim && v.sizes() == k.sizes(),
              "k and v must have shape [tokens, kv_heads, head_dim]");
  TORCH_CHECK(k.stride(2) == 1 && v.stride(2) == 1, "the last dimension of k and v must be contiguous");
  check_packed(inv_freq, k, at::kFloat, "inv_freq");
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.size(0) >= 8 && inv_freq.size(0) % 8 == 0 && 2 * inv_freq.size(0) <= c.head_dim,
              "inv_freq must have shape [rotary / 2], rotary a multiple of 16 up to head_dim");
  a.rotary = (int)(2 * inv_freq.size(0));
  a.interleaved = interleaved;
  a.rope_scale = (float)rope_scale;
  TORCH_CHECK(std::isfinite(a.rope_scale), "rope_scale must be finite");
  if (positions.has_value()) {
    check_packed(*positions, k, at::kInt, "positions");
    TORCH_CHECK(positions->dim() == 1 && positions->size(0) == k.size(0), "positions must have shape [tokens]");
    a.positions = positions->data_ptr<int>();
  }
  const c10::cuda::CUDAGuard guard(k.device());
  OptTensor o;
  TORCH_CHECK(q.has_value() || !q_out.has_value(), "q_out is written with q only");
  if (q.has_value()) {
    check_on(*q, k, "q");
    TORCH_CHECK(q->scalar_type() == k.scalar_type(), "q must have k's dtype");
    TORCH_CHECK(q->dim() == 3 && q->size(0) == k.size(0) && q->size(2) == c.head_dim && q->stride(2) == 1,
                "q must have shape [tokens, heads, head_dim], its last dimension contiguous");
    TORCH_CHECK(q->size(1) >= 1 && q->size(1) <= 65535, "heads must be 1 .. 65535");
    if (q_out.has_value()) {
      o = *q_out;
      check_on(*o, k, "q_out");
      TORCH_CHECK(o->scalar_type() == q->scalar_type() && o->sizes() == q->sizes() && o->stride(2) == 1,
                  "q_out must have q's shape and dtype, its last dimension contiguous");
      if (o->data_ptr() != q->data_ptr() || o->strides() != q->strides()) {
        TORCH_CHECK(o->is_contiguous(), "q_out must be q itself or contiguous");
        const char* across = "q_out must be q itself or lie apart from q, k and v";
        check_apart(*o, *q, across);
        check_apart(*o, k, across, false);
        check_apart(*o, v, across, false);
      } else {
        TORCH_CHECK(!rows_meet(*o, *o, false), "rows of q must lie apart where q_out is q");
        TORCH_CHECK(!rows_meet(*o, k) && !rows_meet(*o, v), "q must lie apart from k and v where q_out is q");
      }
    } else {
      o = fresh(*q, q->sizes(), q->scalar_type());
    }
  }
  if (c.tokens == 0) return o;
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_token_stride = k.stride(0);
  a.k_head_stride = k.stride(1);
  a.v_token_stride = v.stride(0);
  a.v_head_stride = v.stride(1);
  a.inv_freq = inv_freq.data_ptr<float>();
  if (q.has_value()) {
    a.heads = (int)q->size(1);
    a.q = q->data_ptr();
    a.q_token_stride = q->stride(0);
    a.q_head_stride = q->stride(1);
    a.q_out = o->data_ptr();
    a.q_out_token_stride = o->stride(0);
    a.q_out_head_stride = o->stride(1);
  }
  check_launch(fp8imma_kv_append_rope(&c, &a, (void*)at::cuda::getCurrentCUDAStream()), "fp8imma_kv_append_rope");
  return o;
}

std::tuple<torch::Tensor, torch::Tensor> kv_attention_tree(
    const torch::Tensor& q, const torch::Tensor& k_cache, const torch::Tensor& v_cache, const torch::Tensor& k_scale,
    const torch::Tensor& v_scale, const torch::Tensor& page_table, const torch::Tensor& seq_lens, const OptTensor& tree_mask,
    const OptTensor& cu_seqlens, const OptTensor& positions, c10::optional<double> softmax_scale, double softcap, int64_t window,
    const std::string& fmt, const OptTensor& out) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  fp8imma_kv_attention_tree_args a = {};
  a.a_type = act_type(q, "q");
  TORCH_CHECK(q.dim() == 3, "q must have shape [tokens, heads, head_dim]");
  const fp8imma_kv_cache c = cache_args(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cu_seqlens, fmt);
  TORCH_CHECK(q.size(2) == c.head_dim, "q must have the cache's head_dim");
  TORCH_CHECK(q.stride(2) == 1, "the last dimension of q must be contiguous");
  TORCH_CHECK(c.kv_heads > 0 && q.size(1) > 0 && q.size(1) % c.kv_heads == 0, "heads must be a multiple of kv_heads");
  TORCH_CHECK(window >= 0, "window must not be negative");
  a.heads = to_int(q.size(1), "heads");
  a.window = to_int(std::min<int64_t>(window, 0x7fffffff), "window");
  a.softmax_scale = softmax_scale.has_value() ? (float)*softmax_scale : (float)(1.0 / std::sqrt((double)c.head_dim));
  TORCH_CHECK(std::isfinite(a.softmax_scale), "softmax_scale must be finite");
  a.softcap = (float)softcap;
  TORCH_CHECK(a.softcap >= 0 && std::isfinite(a.softcap), "softcap must not be negative");
  if (tree_mask.has_value()) {
    check_packed(*tree_mask, q, at::kInt, "tree_mask");
    TORCH_CHECK(tree_mask->dim() == 2 && tree_mask->size(0) == q.size(0) && tree_mask->size(1) >= 1, "tree_mask must have shape [tokens, words]");
    a.tree_mask = reinterpret_cast<const uint32_t*>(tree_mask->data_ptr<int>());
    a.mask_words = to_int(tree_mask->size(1), "words");
  }
  if (positions.has_value()) {
    TORCH_CHECK(tree_mask.has_value(), "positions are taken with tree_mask only");
    check_packed(*positions, q, at::kInt, "positions");
    TORCH_CHECK(positions->dim() == 1 && positions->size(0) == q.size(0), "positions must have shape [tokens]");
    a.positions = positions->data_ptr<int>();
  }
  const c10::cuda::CUDAGuard guard(q.device());
  torch::Tensor o;
  if (out.has_value()) {
    o = *out;
    check_packed(o, q, q.scalar_type(), "out");
    TORCH_CHECK(o.sizes() == q.sizes(), "out must be shaped like q");
    check_apart(o, q, "out must lie apart from q", false);
  } else {
    o = fresh(q, q.sizes(), q.scalar_type());
  }
  torch::Tensor lse = fresh(q, {q.size(0), q.size(1)}, at::kFloat);
  if (c.tokens == 0) return {o, lse};
  a.q = q.data_ptr();
  a.q_token_stride = q.stride(0);
  a.q_head_stride = q.stride(1);
  a.out = o.data_ptr();
  a.lse = lse.data_ptr<float>();
  check_launch(fp8imma_kv_attention_tree(&c, &a, (void*)at::cuda::getCurrentCUDAStream()), "fp8imma_kv_attention_tree");
  return {o, lse};
}

}  // namespace

void register_layer_ops(pybind11::module_& m) {
  m.def("residual_norm", &residual_norm,
        "Residual connection with the norms on both sides of it (fp8imma_residual_norm)\n"
        "residual' = residual + alpha * gate * (rms_norm(y) by post_weight, or y); out = rms_norm(residual') by pre_weight\n"
        "y: [tokens, hidden] fp16/bf16; residual: y's dtype or fp32; weights [hidden], gate [hidden] or [tokens, hidden] fp16/bf16/fp32\n"
        "weights count as weight + weight_offset\n"
        "Returns (residual' in residual's dtype, out in y's dtype or None without pre_weight)",
        py::arg("y"), py::arg("residual") = py::none(), py::arg("post_weight") = py::none(), py::arg("pre_weight") = py::none(),
        py::arg("gate") = py::none(), py::arg("alpha") = 1.0, py::arg("eps") = 1e-6, py::arg("weight_offset") = 0.0,
        py::arg("residual_out") = py::none(), py::arg("out") = py::none());
  m.def("lora_add", &lora_add,
        "Low-rank adapters of many requests beside a projection (fp8imma_lora_add)\n"
        "out[t] = base[t] + scales[e] * lora_b[e] @ (lora_a[e] @ x[t]), e = adapter_ids[t] (outside [0, adapters): none)\n"
        "base: [tokens, out_features] fp16/bf16, contiguous along either dimension; x: [tokens, in_features] fp16/bf16\n"
        "lora_a: [adapters, rank, in_features], lora_b: [adapters, out_features, rank] in x's dtype; adapter_ids: [tokens] int32\n"
        "Returns out in base's dtype and layout; out= may be base",
        py::arg("base"), py::arg("x"), py::arg("lora_a"), py::arg("lora_b"), py::arg("adapter_ids"),
        py::arg("scales") = py::none(), py::arg("out") = py::none());
  m.def("kv_append_rope", &kv_append_rope,
        "kv_append with the position rotation of queries and keys on the way (fp8imma_kv_append_rope)\n"
        "q: [tokens, heads, head_dim] or None; inv_freq: [rotary / 2] fp32; positions: [tokens] int32 (default: the token's place)\n"
        "interleaved: channels (2i, 2i + 1) turn together instead of (i, i + rotary / 2); the other arguments as in kv_append\n"
        "Returns the rotated q (q_out= may be q)",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"),
        py::arg("page_table"), py::arg("seq_lens"), py::arg("inv_freq"), py::arg("cu_seqlens") = py::none(),
        py::arg("positions") = py::none(), py::arg("rope_scale") = 1.0, py::arg("interleaved") = false, py::arg("fmt") = "e4m3",
        py::arg("q_out") = py::none());
  m.def("kv_attention_tree", &kv_attention_tree,
        "kv_attention for the nodes of drafted trees, with capped scores (fp8imma_kv_attention_tree)\n"
        "tree_mask: [tokens, words] int32, bit j of a token's row: it sees its sequence's j-th token of the step (None: causal)\n"
        "positions: [tokens] int32, for the window; softcap: scores become softcap * tanh(score / softcap) (0: as they are)\n"
        "The other arguments as in kv_attention\n"
        "Returns (out [tokens, heads, head_dim], lse [tokens, heads] fp32)",
        py::arg("q"), py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"), py::arg("page_table"),
        py::arg("seq_lens"), py::arg("tree_mask") = py::none(), py::arg("cu_seqlens") = py::none(), py::arg("positions") = py::none(),
        py::arg("softmax_scale") = py::none(), py::arg("softcap") = 0.0, py::arg("window") = 0, py::arg("fmt") = "e4m3",
        py::arg("out") = py::none());
}
