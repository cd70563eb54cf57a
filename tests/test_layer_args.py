"""CPU checks of the C entry points of the operators between the products: bad arguments return the CUDA error code
before any launch, the ctypes mirrors match the C structures, and the torch entry points refuse CPU tensors."""
import ctypes
import os
import subprocess

import pytest

import fp8imma_b200 as F
from test_serving_args import CACHE, CACHE_BAD, INVALID_CONFIG, INVALID_VALUE, P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAN, INF = float("nan"), float("inf")

NORM = dict(a_type=0, r_type=0, w_type=0, g_type=0, tokens=2, hidden=64, alpha=1.0, eps=1e-6, weight_offset=0.0, y=P, y_stride=64, residual=P,
            residual_stride=64, gate=None, gate_stride=0, post_weight=P, pre_weight=P, residual_out=P, out=P)
LORA = dict(a_type=0, d_type=0, tokens=2, in_features=64, out_features=32, rank=16, adapters=2, x=P, x_stride=64, lora_a=P, lora_b=P, adapter_ids=P,
            scales=None, base=P, base_token_stride=32, base_feature_stride=1, out=P, out_token_stride=32, out_feature_stride=1)
ROPE = dict(a_type=0, heads=4, rotary=64, interleaved=0, rope_scale=1.0, inv_freq=P, positions=None, q=P, k=P, v=P, q_token_stride=256, q_head_stride=64,
            k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, q_out=P, q_out_token_stride=256, q_out_head_stride=64)
TREE = dict(a_type=0, heads=4, window=0, mask_words=1, softmax_scale=0.125, softcap=0.0, q=P, q_token_stride=256, q_head_stride=64, tree_mask=P,
            positions=None, out=P, lse=None)


@pytest.mark.parametrize("change, code", [
    (dict(tokens=0), INVALID_CONFIG), (dict(hidden=0), INVALID_CONFIG), (dict(hidden=32769), INVALID_VALUE), (dict(a_type=2), INVALID_VALUE),
    (dict(r_type=3), INVALID_VALUE), (dict(w_type=-1), INVALID_VALUE), (dict(g_type=3), INVALID_VALUE), (dict(y=None), INVALID_VALUE),
    (dict(y=P + 1), INVALID_VALUE), (dict(out=None), INVALID_VALUE), (dict(pre_weight=None), INVALID_VALUE), (dict(y_stride=-64), INVALID_VALUE),
    (dict(residual_out=None, pre_weight=None, out=None), INVALID_VALUE), (dict(eps=-1.0), INVALID_VALUE), (dict(eps=NAN), INVALID_VALUE),
    (dict(eps=INF), INVALID_VALUE), (dict(r_type=2, residual=P + 2), INVALID_VALUE), (dict(g_type=2, gate=P + 2), INVALID_VALUE),
    (dict(w_type=2, post_weight=P + 2), INVALID_VALUE)])
def test_norm_arguments(change, code):
    assert F.lib().fp8imma_residual_norm(ctypes.byref(F.FP8ImmaResidualNormArgs(**(NORM | change))), None) == code


@pytest.mark.parametrize("change, code", [
    (dict(tokens=0), INVALID_CONFIG), (dict(in_features=0), INVALID_CONFIG), (dict(out_features=0), INVALID_CONFIG), (dict(rank=0), INVALID_CONFIG),
    (dict(adapters=0), INVALID_CONFIG), (dict(rank=12), INVALID_VALUE), (dict(rank=136), INVALID_VALUE), (dict(in_features=60), INVALID_VALUE),
    (dict(a_type=2), INVALID_VALUE), (dict(d_type=2), INVALID_VALUE), (dict(x=None), INVALID_VALUE), (dict(x=P + 8), INVALID_VALUE),
    (dict(x_stride=68), INVALID_VALUE), (dict(lora_a=P + 2), INVALID_VALUE), (dict(lora_b=None), INVALID_VALUE), (dict(adapter_ids=None), INVALID_VALUE),
    (dict(base=None), INVALID_VALUE), (dict(out=None), INVALID_VALUE), (dict(base=P + 1), INVALID_VALUE), (dict(base_feature_stride=2), INVALID_VALUE),
    (dict(out_token_stride=1, out_feature_stride=2), INVALID_VALUE), (dict(base_token_stride=-32), INVALID_VALUE)])
def test_lora_arguments(change, code):
    assert F.lib().fp8imma_lora_add(ctypes.byref(F.FP8ImmaLoraArgs(**(LORA | change))), None) == code


@pytest.mark.parametrize("change, code", CACHE_BAD)
def test_cache_arguments(change, code):
    c = F.FP8ImmaKvCache(**(CACHE | change))
    assert F.lib().fp8imma_kv_append_rope(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAppendRopeArgs(**ROPE)), None) == code
    assert F.lib().fp8imma_kv_attention_tree(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAttentionTreeArgs(**TREE)), None) == code


@pytest.mark.parametrize("change", [
    dict(a_type=2), dict(heads=-1), dict(heads=65536), dict(rotary=0), dict(rotary=24), dict(rotary=80), dict(rope_scale=NAN), dict(rope_scale=INF),
    dict(inv_freq=None), dict(q=None), dict(q_out=None), dict(k=None), dict(v=None), dict(k=P + 1), dict(q=P + 1)])
def test_rope_arguments(change):
    c = F.FP8ImmaKvCache(**CACHE)
    assert F.lib().fp8imma_kv_append_rope(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAppendRopeArgs(**(ROPE | change))), None) == INVALID_VALUE


@pytest.mark.parametrize("change", [
    dict(a_type=2), dict(heads=3), dict(heads=0), dict(window=-1), dict(q=None), dict(out=None), dict(q=P + 1), dict(out=P + 2), dict(mask_words=0),
    dict(tree_mask=None, positions=P), dict(softcap=-1.0), dict(softcap=NAN), dict(softcap=INF), dict(softmax_scale=NAN)])
def test_tree_arguments(change):
    c = F.FP8ImmaKvCache(**CACHE)
    assert F.lib().fp8imma_kv_attention_tree(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAttentionTreeArgs(**(TREE | change))), None) == INVALID_VALUE


def test_null_structures():
    L = F.lib()
    c = F.FP8ImmaKvCache(**CACHE)
    assert L.fp8imma_residual_norm(None, None) == INVALID_VALUE
    assert L.fp8imma_lora_add(None, None) == INVALID_VALUE
    for f in (L.fp8imma_kv_append_rope, L.fp8imma_kv_attention_tree):
        assert f(None, None, None) == INVALID_VALUE
        assert f(ctypes.byref(c), None, None) == INVALID_VALUE


def test_structures_match_the_header(tmp_path):
    """Sizes and offsets of the ctypes mirrors against the C compiler's."""
    names = [("FP8ImmaResidualNormArgs", "fp8imma_residual_norm_args"), ("FP8ImmaLoraArgs", "fp8imma_lora_args"),
             ("FP8ImmaKvAppendRopeArgs", "fp8imma_kv_append_rope_args"), ("FP8ImmaKvAttentionTreeArgs", "fp8imma_kv_attention_tree_args")]
    lines = []
    for py, c in names:
        for f, _ in getattr(F, py)._fields_:
            lines.append('printf("%%zu ", offsetof(%s, %s));' % (c, f))
        lines.append('printf("%%zu\\n", sizeof(%s));' % c)
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fp8imma/fp8imma_ext.h"\nint main(void) { %s return 0; }\n' % "\n".join(lines))
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    for (py, _), line in zip(names, got):
        s = getattr(F, py)
        assert [int(x) for x in line.split()] == [getattr(s, f).offset for f, _ in s._fields_] + [ctypes.sizeof(s)]


def test_torch_entries_refuse_cpu_tensors():
    import torch

    e = F.ext()
    z = torch.zeros
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        e.residual_norm(z(1, 16))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        e.lora_add(z(1, 16), z(1, 16), z(1, 8, 16), z(1, 16, 8), z(1))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        e.kv_append_rope(None, z(1, 1, 64), z(1, 1, 64), z(1, 1, 16, 64), z(1, 1, 16, 64), z(1, 1), z(1, 1), z(1, 1), z(1), z(32))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        e.kv_attention_tree(z(1, 1, 64), z(1, 1, 16, 64), z(1, 1, 16, 64), z(1, 1), z(1, 1), z(1, 1), z(1))
