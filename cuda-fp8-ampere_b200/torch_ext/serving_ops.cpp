// PyTorch binding of the decode-step operators (module fp8imma_ext): the paged
// 8-bit KV cache (kv_append, kv_attention), the few-token mixture-of-experts
// layer (moe_forward) and the scoring of logits (token_logprobs). Arguments
// and results are documented at the C entry points in
// include/fp8imma/fp8imma_ext.h; each call runs on the current stream of its
// tensors' device.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <string>
#include <tuple>

#include "serving_checks.h"

namespace {

using namespace fp8imma_torch;

void kv_append(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
               const torch::Tensor& k_scale, const torch::Tensor& v_scale, const torch::Tensor& page_table,
               const torch::Tensor& seq_lens, const c10::optional<torch::Tensor>& cu_seqlens, const std::string& fmt) {
  TORCH_CHECK(k.is_cuda(), "k must be a CUDA tensor");
  check_on(v, k, "v");
  fp8imma_kv_append_args a = {};
  a.a_type = act_type(k, "k");
  TORCH_CHECK(v.scalar_type() == k.scalar_type(), "k and v must have the same dtype");
  const fp8imma_kv_cache c = cache_args(k, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cu_seqlens, fmt);
  TORCH_CHECK(k.dim() == 3 && k.size(1) == c.kv_heads && k.size(2) == c.head_dim && v.sizes() == k.sizes(),
              "k and v must have shape [tokens, kv_heads, head_dim]");
  TORCH_CHECK(k.stride(2) == 1 && v.stride(2) == 1, "the last dimension of k and v must be contiguous");
  if (c.tokens == 0) return;
  const c10::cuda::CUDAGuard guard(k.device());
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_token_stride = k.stride(0);
  a.k_head_stride = k.stride(1);
  a.v_token_stride = v.stride(0);
  a.v_head_stride = v.stride(1);
  check_launch(fp8imma_kv_append(&c, &a, (void*)at::cuda::getCurrentCUDAStream()), "fp8imma_kv_append");
}

std::tuple<torch::Tensor, torch::Tensor> kv_attention(
    const torch::Tensor& q, const torch::Tensor& k_cache, const torch::Tensor& v_cache, const torch::Tensor& k_scale,
    const torch::Tensor& v_scale, const torch::Tensor& page_table, const torch::Tensor& seq_lens,
    const c10::optional<torch::Tensor>& cu_seqlens, c10::optional<double> softmax_scale, int64_t window,
    const std::string& fmt, const c10::optional<torch::Tensor>& out) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  fp8imma_kv_attention_args a = {};
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
  const c10::cuda::CUDAGuard guard(q.device());
  torch::Tensor o;
  if (out.has_value()) {
    o = *out;
    check_packed(o, q, q.scalar_type(), "out");
    TORCH_CHECK(o.sizes() == q.sizes(), "out must be shaped like q");
  } else {
    o = torch::empty(q.sizes(), q.options());
  }
  torch::Tensor lse = torch::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  if (c.tokens == 0) return {o, lse};
  a.q = q.data_ptr();
  a.q_token_stride = q.stride(0);
  a.q_head_stride = q.stride(1);
  a.out = o.data_ptr();
  a.lse = lse.data_ptr<float>();
  check_launch(fp8imma_kv_attention(&c, &a, (void*)at::cuda::getCurrentCUDAStream()), "fp8imma_kv_attention");
  return {o, lse};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> moe_forward(
    const torch::Tensor& x, const torch::Tensor& router, const torch::Tensor& w_gate_up, const torch::Tensor& s_gate_up,
    const torch::Tensor& w_down, const torch::Tensor& s_down, int64_t top_k, bool renormalize, const std::string& act,
    const std::string& b_format, const c10::optional<torch::Tensor>& out) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  fp8imma_moe_args a = {};
  a.a_type = act_type(x, "x");
  TORCH_CHECK(x.dim() == 2 && (x.size(1) == 1 || x.stride(1) == 1), "x must be [tokens, hidden] with contiguous rows");
  check_packed(router, x, x.scalar_type(), "router");
  TORCH_CHECK(router.dim() == 2 && router.size(1) == x.size(1), "router must have shape [experts, hidden]");
  const int64_t T = x.size(0), H = x.size(1), E = router.size(0);
  a.format = byte_format(b_format, "b_format");
  for (const auto* w : {&w_gate_up, &w_down}) {
    check_on(*w, x, "w_gate_up / w_down");
    TORCH_CHECK(is_bytes(*w) && w->dim() == 3 && w->is_contiguous(), "w_gate_up / w_down must be contiguous 3-D uint8");
    check_format(*w, a.format, "w_gate_up / w_down");
  }
  const int64_t I = w_down.size(2);
  TORCH_CHECK(w_gate_up.size(0) == E && w_gate_up.size(1) == 2 * I && w_gate_up.size(2) == H,
              "w_gate_up must have shape [experts, 2 * inter, hidden]");
  TORCH_CHECK(w_down.size(0) == E && w_down.size(1) == H, "w_down must have shape [experts, hidden, inter]");
  check_packed(s_gate_up, x, at::kFloat, "s_gate_up");
  check_packed(s_down, x, at::kFloat, "s_down");
  TORCH_CHECK(s_gate_up.numel() == E * 2 * I && s_down.numel() == E * H,
              "s_gate_up / s_down must hold one scale per weight row");
  TORCH_CHECK(T <= FP8IMMA_MOE_MAX_TOKENS, "moe_forward takes at most ", FP8IMMA_MOE_MAX_TOKENS, " tokens");
  TORCH_CHECK(E <= FP8IMMA_MOE_MAX_EXPERTS, "moe_forward takes at most ", FP8IMMA_MOE_MAX_EXPERTS, " experts");
  TORCH_CHECK(top_k >= 1 && top_k <= FP8IMMA_MOE_MAX_TOP_K && top_k <= E, "top_k must be 1 .. min(experts, ",
              FP8IMMA_MOE_MAX_TOP_K, ")");
  TORCH_CHECK(H % 16 == 0 && I % 16 == 0, "hidden and inter must be multiples of 16");
  if (act == "silu") a.act = 3;
  else if (act == "gelu") a.act = 2;
  else TORCH_CHECK(false, "act must be 'silu' or 'gelu'");
  const c10::cuda::CUDAGuard guard(x.device());
  torch::Tensor o;
  if (out.has_value()) {
    o = *out;
    check_packed(o, x, x.scalar_type(), "out");
    TORCH_CHECK(o.sizes() == x.sizes(), "out must be shaped like x");
  } else {
    o = torch::empty({T, H}, x.options());
  }
  torch::Tensor ids = torch::empty({T, top_k}, x.options().dtype(at::kInt));
  torch::Tensor wts = torch::empty({T, top_k}, x.options().dtype(at::kFloat));
  if (T == 0) return {o, ids, wts};
  a.renormalize = renormalize;
  a.tokens = (int)T;
  a.experts = (int)E;
  a.top_k = (int)top_k;
  a.hidden = to_int(H, "hidden");
  a.inter = to_int(I, "inter");
  a.x = x.data_ptr();
  a.x_token_stride = x.stride(0);
  a.router = router.data_ptr();
  a.w_gate_up = w_gate_up.data_ptr();
  a.s_gate_up = s_gate_up.data_ptr<float>();
  a.w_down = w_down.data_ptr();
  a.s_down = s_down.data_ptr<float>();
  a.out = o.data_ptr();
  a.ids = ids.data_ptr<int>();
  a.weights = wts.data_ptr<float>();
  check_launch(fp8imma_moe_forward(&a, (void*)at::cuda::getCurrentCUDAStream()), "fp8imma_moe_forward");
  return {o, ids, wts};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> token_logprobs(const torch::Tensor& logits,
                                                                                      const torch::Tensor& tokens,
                                                                                      int64_t top, double temperature) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  TORCH_CHECK(logits.dim() == 2, "logits must have shape [tokens, vocab]");
  const int64_t T = logits.size(0), V = logits.size(1);
  check_packed(tokens, logits, at::kInt, "tokens");
  TORCH_CHECK(tokens.dim() == 1 && tokens.size(0) == T, "tokens must have shape [tokens]");
  fp8imma_logprobs_args a = {};
  if (logits.scalar_type() == at::kHalf) a.l_type = FP8IMMA_L_F16;
  else if (logits.scalar_type() == at::kBFloat16) a.l_type = FP8IMMA_L_BF16;
  else if (logits.scalar_type() == at::kFloat) a.l_type = FP8IMMA_L_F32;
  else TORCH_CHECK(false, "logits must be fp16, bf16 or fp32");
  a.token_stride = logits.stride(0);
  a.vocab_stride = logits.stride(1);
  // a dimension of one element has no stride of its own
  if (V == 1) a.vocab_stride = 1;
  if (T == 1 && a.vocab_stride != 1) a.token_stride = 1;
  TORCH_CHECK(a.vocab_stride == 1 || a.token_stride == 1, "logits must be contiguous along one dimension");
  TORCH_CHECK(top >= 0 && top <= FP8IMMA_LOGPROBS_MAX_TOP && top <= V, "top must be 0 .. min(vocab, ",
              FP8IMMA_LOGPROBS_MAX_TOP, ")");
  TORCH_CHECK(V >= 1, "vocab must not be empty");
  a.temperature = (float)temperature;
  TORCH_CHECK(a.temperature > 0 && std::isfinite(a.temperature), "temperature must be positive and finite");
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  torch::Tensor lp = torch::empty({T}, f32), ent = torch::empty({T}, f32);
  torch::Tensor ids = torch::empty({T, top}, logits.options().dtype(at::kInt)), tlp = torch::empty({T, top}, f32);
  if (T == 0) return {lp, ent, ids, tlp};
  a.tokens = to_int(T, "tokens");
  a.vocab = to_int(V, "vocab");
  a.top = (int)top;
  a.logits = logits.data_ptr();
  a.token_ids = tokens.data_ptr<int>();
  a.logprobs = lp.data_ptr<float>();
  a.entropy = ent.data_ptr<float>();
  a.top_ids = top ? ids.data_ptr<int>() : nullptr;
  a.top_logprobs = top ? tlp.data_ptr<float>() : nullptr;
  check_launch(fp8imma_token_logprobs(&a, (void*)at::cuda::getCurrentCUDAStream()), "fp8imma_token_logprobs");
  return {lp, ent, ids, tlp};
}

}  // namespace

void register_serving_ops(pybind11::module_& m) {
  m.def("kv_append", &kv_append,
        "Store the step's K/V rows in the paged 8-bit cache (fp8imma_kv_append)\n"
        "k, v: [tokens, kv_heads, head_dim] fp16/bf16; k_cache, v_cache: [num_pages, kv_heads, page_size, head_dim] uint8\n"
        "k_scale, v_scale: [num_pages, kv_heads] fp32; page_table: [batch, max_pages] int32\n"
        "seq_lens: [batch] int32, counting the step's tokens; cu_seqlens: [batch + 1] int32 offsets of the step's tokens",
        py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"),
        py::arg("page_table"), py::arg("seq_lens"), py::arg("cu_seqlens") = py::none(), py::arg("fmt") = "e4m3");
  m.def("kv_attention", &kv_attention,
        "Causal attention of the step's queries over the paged 8-bit cache (fp8imma_kv_attention)\n"
        "q: [tokens, heads, head_dim] fp16/bf16; the other tensors as in kv_append\n"
        "Returns (out [tokens, heads, head_dim], lse [tokens, heads] fp32)",
        py::arg("q"), py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"),
        py::arg("page_table"), py::arg("seq_lens"), py::arg("cu_seqlens") = py::none(),
        py::arg("softmax_scale") = py::none(), py::arg("window") = 0, py::arg("fmt") = "e4m3",
        py::arg("out") = py::none());
  m.def("moe_forward", &moe_forward,
        "Mixture-of-experts layer with FP8 weights for 1..64 tokens (fp8imma_moe_forward)\n"
        "x: [tokens, hidden] fp16/bf16; router: [experts, hidden]; w_gate_up: [experts, 2 * inter, hidden] uint8 (gate rows, then up rows)\n"
        "w_down: [experts, hidden, inter] uint8; s_gate_up, s_down: one fp32 scale per weight row (quantize_weights)\n"
        "act: 'silu' or 'gelu' (tanh form)\n"
        "Returns (out [tokens, hidden], ids [tokens, top_k] int32, weights [tokens, top_k] fp32)",
        py::arg("x"), py::arg("router"), py::arg("w_gate_up"), py::arg("s_gate_up"), py::arg("w_down"),
        py::arg("s_down"), py::arg("top_k"), py::arg("renormalize") = true, py::arg("act") = "silu",
        py::arg("b_format") = "e4m3", py::arg("out") = py::none());
  m.def("token_logprobs", &token_logprobs,
        "Log probabilities of given tokens, entropy and top alternatives (fp8imma_token_logprobs)\n"
        "logits: [tokens, vocab] fp16/bf16/fp32, contiguous along either dimension; tokens: [tokens] int32\n"
        "Returns (logprobs [tokens], entropy [tokens], top_ids [tokens, top] int32, top_logprobs [tokens, top])",
        py::arg("logits"), py::arg("tokens"), py::arg("top") = 0, py::arg("temperature") = 1.0);
}
