"""CPU checks of the C entry points of the operators of a step: an address that is not aligned to its
elements is refused before any launch."""
import ctypes

import pytest

import fp8imma_b200 as F
from test_layer_args import LORA, NORM, ROPE, TREE
from test_serving_args import APPEND, ATTEND, CACHE, INVALID_VALUE, MOE, P, SCORE


@pytest.mark.parametrize("name", ["k_scale", "v_scale", "page_table", "seq_lens", "cu_new"])
@pytest.mark.parametrize("by", [1, 2])
def test_cache(name, by):
    c = F.FP8ImmaKvCache(**(CACHE | {name: P + by}))
    assert F.lib().fp8imma_kv_append(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAppendArgs(**APPEND)), None) == INVALID_VALUE
    assert F.lib().fp8imma_kv_attention(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAttentionArgs(**ATTEND)), None) == INVALID_VALUE
    assert F.lib().fp8imma_kv_append_rope(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAppendRopeArgs(**ROPE)), None) == INVALID_VALUE
    assert F.lib().fp8imma_kv_attention_tree(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAttentionTreeArgs(**TREE)), None) == INVALID_VALUE


@pytest.mark.parametrize("name", ["inv_freq", "positions"])
def test_rope(name):
    a = F.FP8ImmaKvAppendRopeArgs(**(ROPE | {name: P + 2}))
    assert F.lib().fp8imma_kv_append_rope(ctypes.byref(F.FP8ImmaKvCache(**CACHE)), ctypes.byref(a), None) == INVALID_VALUE


@pytest.mark.parametrize("name", ["tree_mask", "positions", "lse"])
def test_tree(name):
    a = F.FP8ImmaKvAttentionTreeArgs(**(TREE | {name: P + 2}))
    assert F.lib().fp8imma_kv_attention_tree(ctypes.byref(F.FP8ImmaKvCache(**CACHE)), ctypes.byref(a), None) == INVALID_VALUE


@pytest.mark.parametrize("change", [dict(adapter_ids=P + 2), dict(scales=P + 1), dict(base=P + 1), dict(out=P + 1)])
def test_lora(change):
    assert F.lib().fp8imma_lora_add(ctypes.byref(F.FP8ImmaLoraArgs(**(LORA | change))), None) == INVALID_VALUE


@pytest.mark.parametrize("change", [dict(y=P + 1), dict(residual=P + 1), dict(out=P + 1), dict(residual_out=P + 1), dict(pre_weight=P + 1), dict(gate=P + 1),
                                    dict(r_type=2, residual_out=P + 2)])
def test_norm(change):
    assert F.lib().fp8imma_residual_norm(ctypes.byref(F.FP8ImmaResidualNormArgs(**(NORM | change))), None) == INVALID_VALUE


def test_attention():
    a = F.FP8ImmaKvAttentionArgs(**(ATTEND | dict(lse=P + 2)))
    assert F.lib().fp8imma_kv_attention(ctypes.byref(F.FP8ImmaKvCache(**CACHE)), ctypes.byref(a), None) == INVALID_VALUE


@pytest.mark.parametrize("name", ["s_gate_up", "s_down", "ids", "weights", "out"])
def test_moe(name):
    assert F.lib().fp8imma_moe_forward(ctypes.byref(F.FP8ImmaMoeArgs(**(MOE | {name: P + 2}))), None) == INVALID_VALUE


@pytest.mark.parametrize("name", ["token_ids", "logprobs", "entropy", "top_ids", "top_logprobs"])
def test_logprobs(name):
    assert F.lib().fp8imma_token_logprobs(ctypes.byref(F.FP8ImmaLogprobsArgs(**(SCORE | {name: P + 1}))), None) == INVALID_VALUE
