// fp8imma extension C ABI — B200 (sm_100a).
//
// Entry points for features the reference API (imma_fp8.h) has no slot for:
// per-row dynamic activation quantisation, an fp32 per-column scale fused
// into the epilogue, bf16 output, row-major output, E5M2 weight storage, the
// native FP8 tensor-core path, an int32 accumulator export, and the fp8wgt
// torch extension's fp16-activation kernel as a C entry point.
// Same conventions as the reference C ABI: plain pointers, void* stream
// (cudaStream_t), int return = cudaError_t (0 = success); the library
// launches asynchronously on the caller's stream.
#pragma once

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum fp8imma_a_type { FP8IMMA_A_F16 = 0, FP8IMMA_A_BF16 = 1, FP8IMMA_A_S8 = 2 };

// B byte format. On the int8-exact path E4M3 decodes through the reference
// table semantics (exponent 15: +-Inf for mantissa 0, NaN otherwise); on the
// native path E4M3 is the hardware E4M3FN format. E5M2 is IEEE-like on both.
enum fp8imma_b_format { FP8IMMA_B_E4M3 = 0, FP8IMMA_B_E5M2 = 1 };

enum fp8imma_path {
  FP8IMMA_PATH_INT8_EXACT = 0,  // reference arithmetic, bit-exact int32 accumulators
  FP8IMMA_PATH_FP8_NATIVE = 1   // activations -> E4M3 per row, FP8 tensor cores, fp32 accumulate
};

enum fp8imma_act_quant {
  FP8IMMA_AQ_TENSOR = 0,  // one a_inv_scale / global_scale for the tensor (reference behaviour)
  FP8IMMA_AQ_ROW = 1      // per-row absmax: a_inv_m = 127/absmax_m, g_m = 1/a_inv_m
};

enum fp8imma_out_type { FP8IMMA_OUT_F16 = 0, FP8IMMA_OUT_BF16 = 1 };
enum fp8imma_out_layout { FP8IMMA_OUT_COL = 0 /* D[n*M+m] */, FP8IMMA_OUT_ROW = 1 /* D[m*N+n] */ };

typedef struct fp8imma_gemm_args {
  int path;        // fp8imma_path
  int a_type;      // fp8imma_a_type (S8 only on the int8-exact path)
  int b_format;    // fp8imma_b_format
  int act_quant;   // fp8imma_act_quant (int8-exact path; the native path is always per row)
  int out_type;    // fp8imma_out_type
  int out_layout;  // fp8imma_out_layout
  int M, N, K;
  const void* A;               // [M,K] row-major
  const void* B;               // [N,K] row-major FP8 bytes
  const void* col_scales_u16;  // int8-exact path: [N] fp16 int8-step scales (required)
  const float* col_scales_f32; // optional [N] fp32 multiplier (sigma_c); native path: weight scale
  float global_scale;          // int8-exact path with FP8IMMA_AQ_TENSOR
  float a_inv_scale;           // int8-exact path with FP8IMMA_AQ_TENSOR
  void* D;                     // output, out_type / out_layout
  int32_t* acc_out;            // optional [N,M] int32 accumulators (int8-exact path)
} fp8imma_gemm_args;

// Extended GEMM. No reference counterpart (extends imma_fp8.h:230). On the
// int8-exact path with act_quant = TENSOR, out F16/COL, no col_scales_f32 it
// equals fp8imma_launch_imma_fp8_actquant_v4_{f16,bf16} bit for bit.
// Temporaries (per-row scales, int8 / E4M3 copies of the operands on the
// large-M paths, quantised activation rows) live in per-(device, stream)
// scratch buffers allocated on the first call that needs them and reused by
// later calls on that stream; a call captured in a CUDA graph before its
// buffer exists uses stream-ordered cudaMallocAsync / cudaFreeAsync instead.
int fp8imma_gemm(const fp8imma_gemm_args* args, void* stream);

// fp8imma_gemm with a fused epilogue after the scales, in fp32 before the
// final rounding: + bias[n] (device fp32 [N], or null), then `act`:
// 0 none, 1 ReLU, 2 GELU (tanh form), 3 SiLU. Both paths, every kernel.
int fp8imma_gemm_epilogue(const fp8imma_gemm_args* args, const float* bias, int act, void* stream);

// fp8imma_gemm with host-side activations and result: copies A_host (M x K
// elements of the activation type; page-locked memory for an asynchronous
// copy) into args->A, runs fp8imma_gemm, and copies args->D (M x N outputs)
// back into D_host, all queued on `stream` (the call returns before the
// copies finish; synchronise the stream before reading D_host). args->A and
// args->D are the caller's device staging buffers. On the decode shapes
// (int8-exact path, per-tensor quantisation, fp16 / bf16 activations, M small
// enough for the balanced decode kernel) with page-locked A_host and D_host,
// once the stream has run one such call, the kernels read A_host and write
// D_host in place instead (no copies): args->D still receives the result,
// args->A is then not written.
int fp8imma_gemm_host_io(const fp8imma_gemm_args* args, const void* A_host, void* D_host, void* stream);

// Weight quantiser (no reference counterpart beyond an approximate per-tensor
// benchmark encoder): W [N,K] (fp16 / bf16 / fp32, finite) -> FP8 bytes
// B_out [N,K] with a per-row (= per output column) scale:
//   sigma_n = max(absmax_k |W[n,k]|, 1e-30) / fmax, B = fp8_rne_satfinite(W / sigma_n),
// col_scale_out[n] = sigma_n (fp32, the native path's column scale; may be
// null), step_out[n] = fp16(max_k |decode(B[n,k])| / 127) (the int8 step the
// reference API takes as col_scales; may be null).
enum fp8imma_w_type { FP8IMMA_W_F16 = 0, FP8IMMA_W_BF16 = 1, FP8IMMA_W_F32 = 2 };
enum fp8imma_q_format {
  FP8IMMA_Q_E4M3FN = 0,   // fmax 448 (hardware E4M3FN range)
  FP8IMMA_Q_E5M2 = 1,     // fmax 57344
  FP8IMMA_Q_E4M3_REF = 2  // fmax 240: codes the reference decode table reads as finite
};
int fp8imma_quantize_weights(const void* W, int w_type, int N, int K, int fmt, void* B_out, float* col_scale_out,
                             uint16_t* step_out, void* stream);

// Largest M accepted by fp8imma_gemm_rowquant_noalloc.
#define FP8IMMA_NOALLOC_MAX_M 4096

// Allocation-free per-row-quantised GEMM. No counterpart in the reference (it
// has no per-row quantisation). Same arguments and results as fp8imma_gemm
// with path = FP8IMMA_PATH_INT8_EXACT and act_quant = FP8IMMA_AQ_ROW, for
// callers that may not allocate device memory: runtimes that reserve HBM for
// their own pool up front, serving loops that forbid allocation on the
// request path, and plugin hosts that pass the plugin only caller-owned
// buffers. The caller still passes A, B, scales and D; the per-row values the
// two internal kernels exchange live in a fixed device array of
// FP8IMMA_NOALLOC_MAX_M rows (24 KB) that every GPU loading the library keeps
// until exit. M > FP8IMMA_NOALLOC_MAX_M returns cudaErrorInvalidValue.
// It calls no cudaMalloc / cudaFree / cudaMallocAsync. The first call on each
// device looks up the array's device address (cudaGetSymbolAddress, with that
// device current); make that first call before any stream capture. Every call
// on a device shares the one array (each call overwrites the rows it uses
// before reading them), so calls that overlap on the GPU, e.g. on two streams
// at once, race and must not be issued. fp8imma_set_pdl and fp8imma_set_splitk
// apply as for fp8imma_gemm. Every M runs the small-M kernels (split-K /
// decode; the tensor-core path needs scratch), so M in the hundreds or
// thousands is correct but far slower than through fp8imma_gemm.
int fp8imma_gemm_rowquant_noalloc(const fp8imma_gemm_args* args, void* stream);

// fp8wgt linear: C[M,N] (fp32, row-major) = A[M,K] (fp16) x decode(B[N,K])^T,
// decode(b) = fp16_rn(float(lut_e4m3[b]) * scale_b). Replaces
// torch_ext/fp8wgt/fp8wgt_ext_cuda.cu:223 fp8_linear_forward (kernel :135),
// as a C entry point; runs on `stream` (the reference used the default stream).
int fp8imma_fp8wgt_linear_forward(const void* A_f16, const void* B_u8, float scale_b, void* C_f32,
                                  int M, int N, int K, void* stream);

// Column-parallel GEMM with the output gather fused in (no reference
// counterpart: the reference has no multi-GPU code). Rank `rank` of `world`
// (<= 8) passes its weight shard (args->B, [N_shard, K]) and shard scales;
// the GEMM writes this rank's [N_shard, M] slice of the col-major output into
// rows rank*N_shard.. of its own full buffer peer_out[rank] ([world*N_shard,
// M]) and into the same rows of every peer's buffer over NVLink (peer
// stores, from the GEMM's epilogue or a gather kernel, see
// fp8imma_set_fused_gather), then waits until every rank's slice has arrived
// here. peer_out / peer_signal hold device pointers to all ranks' buffers,
// valid in this process (e.g. a symmetric allocation); each signal pad needs
// 64 zero-initialised uint32 slots; `epoch` must grow by one per call
// (1, 2, ...), or be 0: the epoch is then counted on the device in the pad
// of this rank, so a captured CUDA graph can be replayed.
// Int8-exact path, per-tensor quantisation, col-major output, small M (the
// split-K kernel). The call returns when the launches are queued; the output
// is complete on every rank once this stream reaches the end of the call.
// The caller must not rewrite an output buffer that a peer may still be
// reading from the previous call (alternate two buffers).
int fp8imma_gemm_allgather(const fp8imma_gemm_args* args, void* const* peer_out, void* const* peer_signal, int world,
                           int rank, unsigned int epoch, void* stream);
// 1: the gather of fp8imma_gemm_allgather runs in the GEMM's own epilogue
// (peer stores + one system-scope release per CTA, first CTA waits for the
// peers); 0 (default, measured faster: 17.3 vs 19.4 us per decode step on 2
// GPUs): a separate gather kernel after the GEMM. Each form keeps its own
// counters and epoch in the signal pad, so the setting may change between
// calls.
int fp8imma_set_fused_gather(int enable);

// ------------------------------------------------- decode-step operators ----
// What a decode step needs around the FP8-weight GEMMs. No reference
// counterpart. Activations are fp16 or bf16 (a_type: FP8IMMA_A_F16 or
// FP8IMMA_A_BF16); FP8 bytes are E4M3FN or E5M2 (FP8IMMA_B_E4M3 / _E5M2).
// Forward only, like the GEMMs. Strides are in elements. Same errors as above:
// cudaErrorInvalidConfiguration for an empty problem, cudaErrorInvalidValue
// for a missing pointer, one that is not aligned to its elements, or an
// argument outside its range.

// A paged KV cache in 8 bits with one fp32 scale per (page, KV head) for the
// keys and one for the values: value = code * scale. Page p holds `page_size`
// consecutive tokens of one sequence; a sequence's page_table row lists its
// pages in token order, seq_lens[b] is its number of tokens counting those of
// the present step, and its step's tokens (packed, sequence after sequence;
// cu_new[b] .. cu_new[b+1] of the packed axis) are the last ones of it. One
// page belongs to one sequence while tokens are appended to it; attention may
// read a page through several tables (shared prefixes). A page id outside
// [0, num_pages) is a hole: nothing is stored there and attention skips it.
// Tokens past max_pages * page_size have no place: they are neither stored nor
// read. Scales are not negative. A cu_new that descends anywhere sets the error
// word (fp8imma_device_error(): 7) and nothing is written; rows of the packed
// axis that no sequence owns are not read, and not written.
typedef struct fp8imma_kv_cache {
  void* k;                    // [num_pages, kv_heads, page_size, head_dim] FP8 bytes, 16-byte aligned
  void* v;
  float* k_scale;             // [num_pages, kv_heads]
  float* v_scale;
  const int32_t* page_table;  // [batch, max_pages]
  const int32_t* seq_lens;    // [batch]
  const int32_t* cu_new;      // [batch + 1], or null: tokens / batch tokens for every sequence
  int format;                 // fp8imma_b_format
  int num_pages, kv_heads, page_size, head_dim;  // page_size 16, 32, 64 or 128; head_dim 64, 128 or 256
  int batch, max_pages;
  int tokens;                 // packed tokens of this step, all sequences
} fp8imma_kv_cache;

// Store the step's key and value rows. The scale of a page and head is the
// smallest power of two (2^-126 at least) that brings its rows within the
// format's range; when a row outgrows the scale of a page that holds earlier
// tokens, the page's codes move to the larger scale (an exact shift of the
// exponent but for codes that fall below the format's smallest step). A page
// whose first token is stored starts anew. NaN is kept, +-Inf saturates.
typedef struct fp8imma_kv_append_args {
  int a_type;
  const void* k;  // [tokens, kv_heads, head_dim], last dimension contiguous
  const void* v;
  int64_t k_token_stride, k_head_stride;
  int64_t v_token_stride, v_head_stride;
} fp8imma_kv_append_args;
int fp8imma_kv_append(const fp8imma_kv_cache* cache, const fp8imma_kv_append_args* args, void* stream);

// Causal attention of the step's queries over the cache (grouped heads: query
// head h reads KV head h / (heads / kv_heads)):
//   out[t,h] = sum_j softmax_j(softmax_scale * <q[t,h], K_j>) V_j
// over keys j <= pos(t), and j > pos(t) - window when window > 0, pos(t) being
// the token's place in its sequence. A row that no key is left for gives 0
// and lse = -inf. Statistics and sums are fp32.
typedef struct fp8imma_kv_attention_args {
  int a_type;                 // of q and out
  int heads;                  // query heads, a multiple of kv_heads
  int window;                 // 0: no window
  float softmax_scale;
  const void* q;              // [tokens, heads, head_dim], last dimension contiguous
  int64_t q_token_stride, q_head_stride;
  void* out;                  // [tokens, heads, head_dim] contiguous
  float* lse;                 // optional [tokens, heads]: log of the row's sum of exponentials
} fp8imma_kv_attention_args;
int fp8imma_kv_attention(const fp8imma_kv_cache* cache, const fp8imma_kv_attention_args* args, void* stream);

// A mixture-of-experts layer for a few tokens (1 .. FP8IMMA_MOE_MAX_TOKENS):
//   r = x Wr^T; S = the top_k largest of a row's r (ties: lowest index);
//   p = softmax of r over S (renormalize), or over all experts;
//   out = sum_{e in S} p_e (act(x Wg_e^T) * (x Wu_e^T)) Wd_e^T
// with FP8 expert weights as fp8imma_quantize_weights makes them (one fp32
// scale per weight row). Sums are fp32; the product act(g) * u is rounded to
// fp16 before the second product, after a power of two taken from its own
// values: to 2^-11, or to 2^-24 of the row's largest where that is more.
#define FP8IMMA_MOE_MAX_TOKENS 64
#define FP8IMMA_MOE_MAX_TOP_K 16
#define FP8IMMA_MOE_MAX_EXPERTS 1024
typedef struct fp8imma_moe_args {
  int a_type;                 // of x, router and out
  int format;                 // fp8imma_b_format
  int act;                    // 2 GELU (tanh form), 3 SiLU
  int renormalize;
  int tokens, experts, top_k;
  int hidden, inter;          // multiples of 16
  const void* x;              // [tokens, hidden], last dimension contiguous
  int64_t x_token_stride;
  const void* router;         // [experts, hidden]
  const void* w_gate_up;      // [experts, 2 * inter, hidden]: gate rows, then up rows; 16-byte aligned
  const float* s_gate_up;     // [experts, 2 * inter]
  const void* w_down;         // [experts, hidden, inter]; 16-byte aligned
  const float* s_down;        // [experts, hidden]
  void* out;                  // [tokens, hidden] contiguous
  int32_t* ids;               // optional [tokens, top_k]
  float* weights;             // optional [tokens, top_k]
} fp8imma_moe_args;
int fp8imma_moe_forward(const fp8imma_moe_args* args, void* stream);

// Scores of logits x [tokens, vocab], z = x / temperature:
//   logprob[t] = z[t, token[t]] - lse_t, lse_t = log sum_j exp z[t,j]
//   entropy[t] = - sum_j p_j log p_j, p = softmax z
//   top_ids / top_logprobs: the `top` largest logits of the row in descending
//   order (equal logits: lowest index first; NaN counts as the largest)
// -inf logits take no part (p = 0). A token id outside [0, vocab) gives NaN,
// and so does a row that holds NaN or +inf or only -inf.
#define FP8IMMA_LOGPROBS_MAX_TOP 32
enum fp8imma_l_type { FP8IMMA_L_F16 = 0, FP8IMMA_L_BF16 = 1, FP8IMMA_L_F32 = 2 };
typedef struct fp8imma_logprobs_args {
  int l_type;                 // fp8imma_l_type
  int tokens, vocab;
  int top;                    // 0 .. FP8IMMA_LOGPROBS_MAX_TOP, at most vocab
  float temperature;          // > 0
  const void* logits;
  int64_t token_stride;       // row-major: vocab_stride 1 (or column-major, as
  int64_t vocab_stride;       // the GEMM's default output: token_stride 1)
  const int32_t* token_ids;   // [tokens]
  float* logprobs;            // [tokens]
  float* entropy;             // [tokens]
  int32_t* top_ids;           // [tokens, top] (null when top is 0)
  float* top_logprobs;        // [tokens, top]
} fp8imma_logprobs_args;
int fp8imma_token_logprobs(const fp8imma_logprobs_args* args, void* stream);

// ------------------------------------- operators between the products ----
// The rest of a layer of a decode or verify step. Same conventions as above.

// The residual connection with the norms on both sides of it, o = weight_offset:
//   b = rms(y) (post_weight + o), or y without post_weight
//   r' = residual + alpha * gate * b      (no residual: 0, no gate: 1)
//   h = rms(r') (pre_weight + o),         rms(x) = x / sqrt(mean(x^2) + eps)
// in fp32, r' (residual_out) and h (out) rounded once each; h is made from the
// unrounded r'. A sum of squares past fp32's range counts as infinite (h = 0). residual_out may be residual, out may be y, where strides agree.
#define FP8IMMA_NORM_MAX_HIDDEN 32768
typedef struct fp8imma_residual_norm_args {
  int a_type;                 // of y and out
  int r_type;                 // fp8imma_l_type of residual and residual_out
  int w_type;                 // fp8imma_l_type of the weights
  int g_type;                 // fp8imma_l_type of the gate
  int tokens, hidden;         // hidden 1 .. FP8IMMA_NORM_MAX_HIDDEN
  float alpha, eps, weight_offset;
  const void* y;              // [tokens, hidden], last dimension contiguous
  int64_t y_stride;
  const void* residual;       // optional [tokens, hidden], last dimension contiguous
  int64_t residual_stride;
  const void* gate;           // optional [tokens, hidden], or [hidden] with gate_stride 0
  int64_t gate_stride;
  const void* post_weight;    // optional [hidden]
  const void* pre_weight;     // optional [hidden]
  void* residual_out;         // [tokens, hidden] contiguous (optional with pre_weight)
  void* out;                  // [tokens, hidden] contiguous, with pre_weight only
} fp8imma_residual_norm_args;
int fp8imma_residual_norm(const fp8imma_residual_norm_args* args, void* stream);

// Low-rank adapters of many requests beside a projection:
//   out[t,n] = base[t,n] + scales[e] sum_r lora_b[e,n,r] sum_k lora_a[e,r,k] x[t,k],
// e = adapter_ids[t]; an id outside [0, adapters) leaves the token without an
// adapter (out = base). base is the projection's result in either layout (the
// GEMM's default is column-major). Neighbouring tokens of one adapter share its
// weights' way to the SM, so requests are best laid one after another. Sums are
// fp32; the inner sums enter the second product as two 16-bit numbers each, and
// what an infinity in x or in an adapter reaches comes out infinite or NaN.
#define FP8IMMA_LORA_MAX_RANK 128
typedef struct fp8imma_lora_args {
  int a_type;                 // of x, lora_a and lora_b
  int d_type;                 // fp8imma_out_type of base and out
  int tokens, in_features, out_features, rank, adapters;  // in_features and rank multiples of 8, rank <= FP8IMMA_LORA_MAX_RANK
  const void* x;              // [tokens, in_features], last dimension contiguous, rows 16-byte aligned
  int64_t x_stride;
  const void* lora_a;         // [adapters, rank, in_features], 16-byte aligned
  const void* lora_b;         // [adapters, out_features, rank], 16-byte aligned
  const int32_t* adapter_ids; // [tokens]
  const float* scales;        // optional [adapters]
  const void* base;           // one of the two strides is 1
  int64_t base_token_stride, base_feature_stride;
  void* out;                  // laid out along the same dimension; may be base
  int64_t out_token_stride, out_feature_stride;
} fp8imma_lora_args;
int fp8imma_lora_add(const fp8imma_lora_args* args, void* stream);

// fp8imma_kv_append with the position rotation of queries and keys on the way.
// Channels (i, i + rotary / 2) of the first `rotary` of a head (interleaved:
// (2i, 2i + 1)) turn by the angle position * inv_freq[i], taken modulo a turn in
// 64 bits, and are multiplied by rope_scale; the other channels stay. Keys enter
// the cache from fp32, queries are rounded to their type. Queries of every
// token that a sequence owns are written, whether its key has a place or not.
typedef struct fp8imma_kv_append_rope_args {
  int a_type;
  int heads;                  // query heads (0: no queries)
  int rotary;                 // a multiple of 16, at most head_dim
  int interleaved;
  float rope_scale;
  const float* inv_freq;      // [rotary / 2]
  const int32_t* positions;   // optional [tokens]; without: the token's place in its sequence
  const void* q;              // [tokens, heads, head_dim], last dimension contiguous, as k and v
  const void* k;              // [tokens, kv_heads, head_dim]
  const void* v;
  int64_t q_token_stride, q_head_stride;
  int64_t k_token_stride, k_head_stride;
  int64_t v_token_stride, v_head_stride;
  void* q_out;                // [tokens, heads, head_dim], last dimension contiguous; may be q, where q's rows lie
                              // apart from one another and from those of k and v
  int64_t q_out_token_stride, q_out_head_stride;
} fp8imma_kv_append_rope_args;
int fp8imma_kv_append_rope(const fp8imma_kv_cache* cache, const fp8imma_kv_append_rope_args* args, void* stream);

// fp8imma_kv_attention for the nodes of drafted trees, with capped scores.
// Keys before the step are seen by all of the step's tokens; of the step's own,
// token i (counted within its sequence) sees token j where bit j % 32 of
// tree_mask[t][j / 32] is set, t being i's packed place (tokens past the mask's
// words are not seen). That is a tree when each node's bits are its ancestors
// and itself, and any other mask within the step as well. Without tree_mask the
// step is causal. A window holds back keys before the step only:
// j > position(t) - window, the positions (a node's depth counts from the
// step's first place) taken between the step's first and last place; without
// them a token's place counts. softcap > 0: scores are
// softcap * tanh(s / softcap), s = softmax_scale <q, K_j>, off by 2^-21 relative
// under any finite cap (one below 2^-30 counts as that, one above 2^99 too).
typedef struct fp8imma_kv_attention_tree_args {
  int a_type;                 // of q and out
  int heads;                  // query heads, a multiple of kv_heads
  int window;                 // 0: no window
  int mask_words;             // words of a mask row
  float softmax_scale, softcap;
  const void* q;              // [tokens, heads, head_dim], last dimension contiguous
  int64_t q_token_stride, q_head_stride;
  const uint32_t* tree_mask;  // optional [tokens, mask_words]
  const int32_t* positions;   // optional [tokens], with tree_mask only
  void* out;                  // [tokens, heads, head_dim] contiguous
  float* lse;                 // optional [tokens, heads]
} fp8imma_kv_attention_tree_args;
int fp8imma_kv_attention_tree(const fp8imma_kv_cache* cache, const fp8imma_kv_attention_tree_args* args, void* stream);

// Tuning / introspection (no reference counterpart).
// Force the K split of the small-M kernel (0 = automatic; 1, 2, 4 or 8).
int fp8imma_set_splitk(int splits);
// Small-M kernel form when no split is forced. Stream-K: persistent CTAs
// with an even share of the weight bytes each, partial sums in a per-device
// scratch ring allocated on first use. Clusters: K slices of a column tile
// reducing in distributed shared memory. 1 (default) = stream-K where the
// cluster form would need more than one wave of CTAs, else clusters;
// 2 = always stream-K; 0 = always clusters.
int fp8imma_set_stream_k(int mode);
// Largest M routed to the small-M split-K kernel (default 64).
int fp8imma_set_small_m_max(int m);
// Large-M tensor-core kernel: 1 (default) = CTA-pair kernel (tcgen05
// cta_group::2, 256x256 tiles), 0 = single-CTA kernel (128x256 tiles).
int fp8imma_set_tc_pair(int enable);
// K splits of the CTA-pair tcgen05 kernel: -1 (default) = automatic (split
// when the 256 x 256 tiles would leave most CTA pairs idle, e.g. M <= 512 at
// N = 4096), 1 = never, n > 1 = forced. Partial accumulators go to
// stream-ordered scratch and a second kernel finishes the epilogue.
int fp8imma_set_tc_splitk(int splits);
// Activation rows per CTA-pair tile (the MMA's N): 0 (default) = chosen per
// shape to balance the rounds of tiles over the CTA pairs; 256, 192 or 128
// forced.
int fp8imma_set_tc_tile_x(int rows);
// 1 (default): when the CTA-pair kernel's last round of tiles would leave more
// than half of the CTA pairs idle, those tiles run as two half-width items
// each (4096 x 4096: 34 of 256 tiles); 0: all tiles at full width.
int fp8imma_set_tc_half_tail(int enable);
// 1 (default): small-M shapes that fit one wave of at most 64 weight columns
// per SM (e.g. N = K = 4096) run the balanced decode kernel (one CTA per SM,
// CTA pairs splitting K); 2: the decode kernel without the early weight
// transcode (it otherwise converts its weights to int8 in shared memory while
// the activations are still to come); 0: they run the split-K cluster kernel.
// Results are identical in every mode. No reference counterpart (tuning
// switch).
int fp8imma_set_decode_kernel(int enable);
// Query rows of a sequence and KV head (tokens of the step x heads / kv_heads,
// on average) from which fp8imma_kv_attention multiplies on tcgen05 (head_dim 64
// and 128; for tests and measurements). 0, the default: by rows and by the tiles
// that the page tables hold. The two kernels' results differ by roundings only.
int fp8imma_set_attention_tc_rows(int rows);
// Programmatic dependent launch (default on). A small-M GEMM then starts
// streaming its weights and reading its column scales while the previous
// kernel in the stream is still running; activations are read, and outputs
// written, only after that kernel has finished (a kernel launched after the
// GEMM without the attribute is ordered as usual). Turn it off when weights or
// scales are written by the kernel launched just before the GEMM.
int fp8imma_set_pdl(int enable);
// Kernel family the last fp8imma call on this thread launched:
// 0 none, 1 small-M split-K, 2 generic fallback, 3 tcgen05 GEMM, 4 native FP8
// tcgen05 GEMM, 5 native FP8 small-M split-K, 6 balanced decode kernel.
int fp8imma_last_path(void);
const char* fp8imma_version(void);
// Error word of the current device: non-zero when a kernel gave up a bounded
// wait on its internal pipeline (the kernel then returned early and its output
// is not valid). Synchronises the device. clear != 0 resets it.
unsigned int fp8imma_device_error(int clear);
// Wall-time limit of every bounded wait in the kernels (mbarrier pipelines,
// the NVLink gather's peer flags) on the current device, in nanoseconds;
// default 2e9; values below 1e6 act as 1e6. A wait that runs out records a code in the error word above and
// lets its kernel finish. No reference counterpart (failure handling).
int fp8imma_set_wait_limit_ns(unsigned long long ns);

#ifdef __cplusplus
}  // extern "C"
#endif
