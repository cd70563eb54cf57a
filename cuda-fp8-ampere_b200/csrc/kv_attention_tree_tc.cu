// The tcgen05 cache attention for fp8imma_kv_attention_tree: the TREE variant of the
// kernel in kv_attention_tc.cu.
#define FP8IMMA_ATTENTION_TREE
#include "kv_attention_tc.cu"

namespace fp8imma_b200 {

cudaError_t launch_attention_tree_tc(attn::AttnParams& p, cudaStream_t st) { return launch_tc_d<true>(p, st); }
unsigned int attn_tree_tc_device_error(bool clear) { return fp8imma_dev::tu_device_error(clear); }
cudaError_t attn_tree_tc_set_wait_limit(unsigned long long ns) { return fp8imma_dev::tu_set_wait_limit(ns); }

}  // namespace fp8imma_b200
