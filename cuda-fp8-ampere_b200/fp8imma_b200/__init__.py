"""fp8imma on B200 (sm_100a): Python side of the drop-in.

The product is ``libfp8imma.so`` (CUDA kernels + the reference C ABI, see
``include/fp8imma/imma_fp8.h`` and ``fp8imma_ext.h``) and the torch extension
modules ``fp8imma_ext`` / ``fp8wgt_ext`` that call it. This package loads them
(failing loudly when they are missing), exposes a ctypes handle on the C ABI,
and holds the column-parallel multi-GPU wrapper (``sharded``).

There is no CPU fallback: every entry point runs the sm_100a kernels.
"""
from __future__ import annotations

import ctypes
import os
import sys

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))  # cuda-fp8-ampere_b200/
LIB_PATH = os.path.join(PKG_DIR, "libfp8imma.so")

if PKG_DIR not in sys.path:
    sys.path.insert(0, PKG_DIR)

_lib = None

# reference C ABI entry points (include/fp8imma/imma_fp8.h) and extensions
REF_SYMBOLS = [
    "fp8imma_init_fp8_e4m3_lut",
    "fp8imma_launch_imma_fp8_jit_v2",
    "fp8imma_launch_imma_fp8_jit_v2_i8lut",
    "fp8imma_launch_imma_fp8_actquant_v3_f16",
    "fp8imma_launch_imma_fp8_actquant_v3_bf16",
    "fp8imma_launch_imma_fp8_actquant_v4_texscale_f16",
    "fp8imma_launch_imma_fp8_actquant_v4_texscale_bf16",
    "fp8imma_launch_imma_fp8_actquant_v4_f16",
    "fp8imma_launch_imma_fp8_actquant_v4_bf16",
]
EXT_SYMBOLS = [
    "fp8imma_gemm",
    "fp8imma_gemm_host_io",
    "fp8imma_gemm_epilogue",
    "fp8imma_gemm_rowquant_noalloc",
    "fp8imma_gemm_allgather",
    "fp8imma_set_fused_gather",
    "fp8imma_fp8wgt_linear_forward",
    "fp8imma_quantize_weights",
    "fp8imma_kv_append",
    "fp8imma_kv_attention",
    "fp8imma_moe_forward",
    "fp8imma_token_logprobs",
    "fp8imma_residual_norm",
    "fp8imma_lora_add",
    "fp8imma_kv_append_rope",
    "fp8imma_kv_attention_tree",
    "fp8imma_set_splitk",
    "fp8imma_set_stream_k",
    "fp8imma_set_small_m_max",
    "fp8imma_last_path",
    "fp8imma_set_pdl",
    "fp8imma_set_decode_kernel",
    "fp8imma_set_attention_tc_rows",
    "fp8imma_set_wait_limit_ns",
    "fp8imma_set_tc_pair",
    "fp8imma_set_tc_splitk",
    "fp8imma_set_tc_tile_x",
    "fp8imma_set_tc_half_tail",
    "fp8imma_device_error",
    "fp8imma_version",
]


class FP8ImmaGemmArgs(ctypes.Structure):
    """Mirror of ``fp8imma_gemm_args`` (include/fp8imma/fp8imma_ext.h)."""

    _fields_ = [
        ("path", ctypes.c_int), ("a_type", ctypes.c_int), ("b_format", ctypes.c_int),
        ("act_quant", ctypes.c_int), ("out_type", ctypes.c_int), ("out_layout", ctypes.c_int),
        ("M", ctypes.c_int), ("N", ctypes.c_int), ("K", ctypes.c_int),
        ("A", ctypes.c_void_p), ("B", ctypes.c_void_p), ("col_scales_u16", ctypes.c_void_p),
        ("col_scales_f32", ctypes.c_void_p), ("global_scale", ctypes.c_float),
        ("a_inv_scale", ctypes.c_float), ("D", ctypes.c_void_p), ("acc_out", ctypes.c_void_p),
    ]


def _struct(name: str, doc: str, **groups):
    """A ctypes mirror of a C argument structure from (type letter, names) pairs in order."""
    kinds = {"i": ctypes.c_int, "p": ctypes.c_void_p, "l": ctypes.c_int64, "f": ctypes.c_float}
    fields = [(n, kinds[key[0]]) for key, names in groups.items() for n in names.split()]
    return type(name, (ctypes.Structure,), {"__doc__": doc, "_fields_": fields})


# Mirrors of the argument structures of the decode-step operators
# (include/fp8imma/fp8imma_ext.h); the keyword's first letter is the type.
FP8ImmaKvCache = _struct(
    "FP8ImmaKvCache", "fp8imma_kv_cache", p0="k v k_scale v_scale page_table seq_lens cu_new",
    i1="format num_pages kv_heads page_size head_dim batch max_pages tokens")
FP8ImmaKvAppendArgs = _struct(
    "FP8ImmaKvAppendArgs", "fp8imma_kv_append_args", i0="a_type", p1="k v",
    l2="k_token_stride k_head_stride v_token_stride v_head_stride")
FP8ImmaKvAttentionArgs = _struct(
    "FP8ImmaKvAttentionArgs", "fp8imma_kv_attention_args", i0="a_type heads window", f1="softmax_scale", p2="q",
    l3="q_token_stride q_head_stride", p4="out lse")
FP8ImmaMoeArgs = _struct(
    "FP8ImmaMoeArgs", "fp8imma_moe_args", i0="a_type format act renormalize tokens experts top_k hidden inter", p1="x",
    l2="x_token_stride", p3="router w_gate_up s_gate_up w_down s_down out ids weights")
FP8ImmaLogprobsArgs = _struct(
    "FP8ImmaLogprobsArgs", "fp8imma_logprobs_args", i0="l_type tokens vocab top", f1="temperature", p2="logits",
    l3="token_stride vocab_stride", p4="token_ids logprobs entropy top_ids top_logprobs")
FP8ImmaResidualNormArgs = _struct(
    "FP8ImmaResidualNormArgs", "fp8imma_residual_norm_args", i0="a_type r_type w_type g_type tokens hidden",
    f1="alpha eps weight_offset", p2="y", l3="y_stride", p4="residual", l5="residual_stride", p6="gate", l7="gate_stride",
    p8="post_weight pre_weight residual_out out")
FP8ImmaLoraArgs = _struct(
    "FP8ImmaLoraArgs", "fp8imma_lora_args", i0="a_type d_type tokens in_features out_features rank adapters", p1="x",
    l2="x_stride", p3="lora_a lora_b adapter_ids scales base", l4="base_token_stride base_feature_stride", p5="out",
    l6="out_token_stride out_feature_stride")
FP8ImmaKvAppendRopeArgs = _struct(
    "FP8ImmaKvAppendRopeArgs", "fp8imma_kv_append_rope_args", i0="a_type heads rotary interleaved", f1="rope_scale",
    p2="inv_freq positions q k v",
    l3="q_token_stride q_head_stride k_token_stride k_head_stride v_token_stride v_head_stride", p4="q_out",
    l5="q_out_token_stride q_out_head_stride")
FP8ImmaKvAttentionTreeArgs = _struct(
    "FP8ImmaKvAttentionTreeArgs", "fp8imma_kv_attention_tree_args", i0="a_type heads window mask_words",
    f1="softmax_scale softcap", p2="q", l3="q_token_stride q_head_stride", p4="tree_mask positions out lse")


def lib() -> ctypes.CDLL:
    """ctypes handle on libfp8imma.so with argument types declared."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError("libfp8imma.so is not built (%s); run cuda-fp8-ampere_b200/build.py" % LIB_PATH)
    L = ctypes.CDLL(LIB_PATH)
    P, I, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    L.fp8imma_init_fp8_e4m3_lut.restype = None
    L.fp8imma_init_fp8_e4m3_lut.argtypes = []
    for name in ("fp8imma_launch_imma_fp8_jit_v2", "fp8imma_launch_imma_fp8_jit_v2_i8lut"):
        f = getattr(L, name)
        f.restype = I
        f.argtypes = [I, P, P, P, P, I, I, I, F, P]
    for name in REF_SYMBOLS[3:]:
        f = getattr(L, name)
        f.restype = I
        f.argtypes = [I, P, P, P, P, I, I, I, F, F, P]
    L.fp8imma_gemm.restype = I
    L.fp8imma_gemm.argtypes = [ctypes.POINTER(FP8ImmaGemmArgs), P]
    L.fp8imma_gemm_host_io.restype = I
    L.fp8imma_gemm_epilogue.restype = I
    L.fp8imma_gemm_epilogue.argtypes = [ctypes.POINTER(FP8ImmaGemmArgs), P, I, P]
    L.fp8imma_gemm_host_io.argtypes = [ctypes.POINTER(FP8ImmaGemmArgs), P, P, P]
    L.fp8imma_gemm_allgather.restype = I
    L.fp8imma_set_fused_gather.restype = I
    L.fp8imma_set_fused_gather.argtypes = [I]
    L.fp8imma_gemm_allgather.argtypes = [ctypes.POINTER(FP8ImmaGemmArgs), P, P, I, I, ctypes.c_uint, P]
    L.fp8imma_gemm_rowquant_noalloc.restype = I
    L.fp8imma_gemm_rowquant_noalloc.argtypes = [ctypes.POINTER(FP8ImmaGemmArgs), P]
    L.fp8imma_quantize_weights.restype = I
    L.fp8imma_quantize_weights.argtypes = [P, I, I, I, I, P, P, P, P]
    L.fp8imma_kv_append.restype = I
    L.fp8imma_kv_append.argtypes = [ctypes.POINTER(FP8ImmaKvCache), ctypes.POINTER(FP8ImmaKvAppendArgs), P]
    L.fp8imma_kv_attention.restype = I
    L.fp8imma_kv_attention.argtypes = [ctypes.POINTER(FP8ImmaKvCache), ctypes.POINTER(FP8ImmaKvAttentionArgs), P]
    L.fp8imma_moe_forward.restype = I
    L.fp8imma_moe_forward.argtypes = [ctypes.POINTER(FP8ImmaMoeArgs), P]
    L.fp8imma_token_logprobs.restype = I
    L.fp8imma_token_logprobs.argtypes = [ctypes.POINTER(FP8ImmaLogprobsArgs), P]
    L.fp8imma_residual_norm.restype = I
    L.fp8imma_residual_norm.argtypes = [ctypes.POINTER(FP8ImmaResidualNormArgs), P]
    L.fp8imma_lora_add.restype = I
    L.fp8imma_lora_add.argtypes = [ctypes.POINTER(FP8ImmaLoraArgs), P]
    L.fp8imma_kv_append_rope.restype = I
    L.fp8imma_kv_append_rope.argtypes = [ctypes.POINTER(FP8ImmaKvCache), ctypes.POINTER(FP8ImmaKvAppendRopeArgs), P]
    L.fp8imma_kv_attention_tree.restype = I
    L.fp8imma_kv_attention_tree.argtypes = [ctypes.POINTER(FP8ImmaKvCache), ctypes.POINTER(FP8ImmaKvAttentionTreeArgs), P]
    L.fp8imma_fp8wgt_linear_forward.restype = I
    L.fp8imma_fp8wgt_linear_forward.argtypes = [P, P, F, P, I, I, I, P]
    L.fp8imma_set_splitk.restype = I
    L.fp8imma_set_splitk.argtypes = [I]
    L.fp8imma_set_stream_k.restype = I
    L.fp8imma_set_stream_k.argtypes = [I]
    L.fp8imma_set_small_m_max.restype = I
    L.fp8imma_set_small_m_max.argtypes = [I]
    L.fp8imma_set_tc_pair.restype = I
    L.fp8imma_set_tc_pair.argtypes = [I]
    L.fp8imma_set_tc_splitk.restype = I
    L.fp8imma_set_tc_splitk.argtypes = [I]
    L.fp8imma_set_tc_tile_x.restype = I
    L.fp8imma_set_tc_tile_x.argtypes = [I]
    L.fp8imma_set_tc_half_tail.restype = I
    L.fp8imma_set_tc_half_tail.argtypes = [I]
    L.fp8imma_set_pdl.restype = I
    L.fp8imma_set_pdl.argtypes = [I]
    L.fp8imma_set_attention_tc_rows.restype = I
    L.fp8imma_set_attention_tc_rows.argtypes = [I]
    L.fp8imma_set_decode_kernel.restype = I
    L.fp8imma_set_decode_kernel.argtypes = [I]
    L.fp8imma_set_wait_limit_ns.restype = I
    L.fp8imma_set_wait_limit_ns.argtypes = [ctypes.c_ulonglong]
    L.fp8imma_device_error.restype = ctypes.c_uint
    L.fp8imma_device_error.argtypes = [I]
    L.fp8imma_last_path.restype = I
    L.fp8imma_last_path.argtypes = []
    L.fp8imma_version.restype = ctypes.c_char_p
    L.fp8imma_version.argtypes = []
    _lib = L
    return L


def ext():
    """The compiled torch extension ``fp8imma_ext`` (reference module name)."""
    import torch  # noqa: F401  (loads libtorch before the extension)
    import fp8imma_ext

    return fp8imma_ext


def wgt_ext():
    import torch  # noqa: F401
    import fp8wgt_ext

    return fp8wgt_ext
