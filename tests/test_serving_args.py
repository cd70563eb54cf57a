"""CPU checks of the decode-step operators' C entry points: bad arguments return the CUDA error code before any
launch, the ctypes mirrors match the C structures, and the torch entry points refuse CPU tensors."""
import ctypes
import os
import subprocess

import pytest

import fp8imma_b200 as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID_VALUE, INVALID_CONFIG = 1, 9
P = 4096  # a 16-byte aligned address that is never dereferenced: validation fails first

CACHE = dict(k=P, v=P, k_scale=P, v_scale=P, page_table=P, seq_lens=P, cu_new=None, format=0, num_pages=4, kv_heads=2, page_size=16,
             head_dim=64, batch=2, max_pages=2, tokens=2)
CACHE_BAD = [(dict(tokens=0), INVALID_CONFIG), (dict(batch=0), INVALID_CONFIG), (dict(num_pages=0), INVALID_CONFIG), (dict(max_pages=0), INVALID_CONFIG),
             (dict(kv_heads=0), INVALID_CONFIG), (dict(k=None), INVALID_VALUE), (dict(v=P + 8), INVALID_VALUE), (dict(k_scale=None), INVALID_VALUE),
             (dict(page_table=None), INVALID_VALUE), (dict(seq_lens=None), INVALID_VALUE), (dict(format=2), INVALID_VALUE),
             (dict(page_size=48), INVALID_VALUE), (dict(head_dim=96), INVALID_VALUE), (dict(tokens=3), INVALID_VALUE),
             (dict(num_pages=1 << 27), INVALID_VALUE), (dict(max_pages=1 << 28), INVALID_VALUE)]
APPEND = dict(a_type=0, k=P, v=P, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64)
ATTEND = dict(a_type=0, heads=4, window=0, softmax_scale=0.125, q=P, q_token_stride=256, q_head_stride=64, out=P, lse=None)
MOE = dict(a_type=0, format=0, act=3, renormalize=1, tokens=2, experts=4, top_k=2, hidden=64, inter=32, x=P, x_token_stride=64, router=P,
           w_gate_up=P, s_gate_up=P, w_down=P, s_down=P, out=P, ids=None, weights=None)
SCORE = dict(l_type=0, tokens=2, vocab=16, top=2, temperature=1.0, logits=P, token_stride=16, vocab_stride=1, token_ids=P, logprobs=P, entropy=P,
             top_ids=P, top_logprobs=P)


@pytest.mark.parametrize("change, code", CACHE_BAD)
def test_cache_arguments(change, code):
    L = F.lib()
    c = F.FP8ImmaKvCache(**(CACHE | change))
    assert L.fp8imma_kv_append(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAppendArgs(**APPEND)), None) == code
    assert L.fp8imma_kv_attention(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAttentionArgs(**ATTEND)), None) == code


def test_null_structures():
    L = F.lib()
    c = F.FP8ImmaKvCache(**CACHE)
    assert L.fp8imma_kv_append(None, None, None) == INVALID_VALUE
    assert L.fp8imma_kv_append(ctypes.byref(c), None, None) == INVALID_VALUE
    assert L.fp8imma_kv_attention(ctypes.byref(c), None, None) == INVALID_VALUE
    assert L.fp8imma_moe_forward(None, None) == INVALID_VALUE
    assert L.fp8imma_token_logprobs(None, None) == INVALID_VALUE


@pytest.mark.parametrize("change", [dict(a_type=2), dict(k=None), dict(v=None), dict(k=P + 1)])
def test_append_arguments(change):
    c = F.FP8ImmaKvCache(**CACHE)
    assert F.lib().fp8imma_kv_append(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAppendArgs(**(APPEND | change))), None) == INVALID_VALUE


@pytest.mark.parametrize("change", [dict(a_type=2), dict(heads=3), dict(heads=0), dict(window=-1), dict(q=None), dict(out=None), dict(q=P + 1), dict(out=P + 2)])
def test_attention_arguments(change):
    c = F.FP8ImmaKvCache(**CACHE)
    assert F.lib().fp8imma_kv_attention(ctypes.byref(c), ctypes.byref(F.FP8ImmaKvAttentionArgs(**(ATTEND | change))), None) == INVALID_VALUE


@pytest.mark.parametrize("change, code", [(dict(tokens=0), INVALID_CONFIG), (dict(experts=0), INVALID_CONFIG), (dict(hidden=0), INVALID_CONFIG),
                                          (dict(inter=0), INVALID_CONFIG), (dict(tokens=65), INVALID_VALUE), (dict(experts=1025), INVALID_VALUE),
                                          (dict(top_k=0), INVALID_VALUE), (dict(top_k=5), INVALID_VALUE), (dict(experts=64, top_k=17), INVALID_VALUE),
                                          (dict(hidden=40), INVALID_VALUE), (dict(inter=24), INVALID_VALUE), (dict(act=1), INVALID_VALUE),
                                          (dict(a_type=2), INVALID_VALUE), (dict(format=2), INVALID_VALUE), (dict(x=None), INVALID_VALUE),
                                          (dict(router=None), INVALID_VALUE), (dict(w_gate_up=P + 4), INVALID_VALUE), (dict(w_down=None), INVALID_VALUE),
                                          (dict(s_down=None), INVALID_VALUE), (dict(out=None), INVALID_VALUE)])
def test_moe_arguments(change, code):
    assert F.lib().fp8imma_moe_forward(ctypes.byref(F.FP8ImmaMoeArgs(**(MOE | change))), None) == code


@pytest.mark.parametrize("change, code", [(dict(tokens=0), INVALID_CONFIG), (dict(vocab=0), INVALID_CONFIG), (dict(top=33, vocab=64), INVALID_VALUE),
                                          (dict(top=17), INVALID_VALUE), (dict(top=-1), INVALID_VALUE), (dict(temperature=0.0), INVALID_VALUE),
                                          (dict(temperature=float("nan")), INVALID_VALUE), (dict(temperature=float("inf")), INVALID_VALUE),
                                          (dict(l_type=3), INVALID_VALUE), (dict(vocab_stride=2), INVALID_VALUE), (dict(logits=None), INVALID_VALUE),
                                          (dict(token_ids=None), INVALID_VALUE), (dict(top_ids=None), INVALID_VALUE), (dict(entropy=None), INVALID_VALUE)])
def test_score_arguments(change, code):
    assert F.lib().fp8imma_token_logprobs(ctypes.byref(F.FP8ImmaLogprobsArgs(**(SCORE | change))), None) == code


def test_structures_match_the_header(tmp_path):
    """Sizes and last offsets of the ctypes mirrors against the C compiler's."""
    names = [("FP8ImmaKvCache", "fp8imma_kv_cache"), ("FP8ImmaKvAppendArgs", "fp8imma_kv_append_args"),
             ("FP8ImmaKvAttentionArgs", "fp8imma_kv_attention_args"), ("FP8ImmaMoeArgs", "fp8imma_moe_args"),
             ("FP8ImmaLogprobsArgs", "fp8imma_logprobs_args")]
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
        e.kv_append(z(1, 1, 64), z(1, 1, 64), z(1, 1, 16, 64), z(1, 1, 16, 64), z(1, 1), z(1, 1), z(1, 1), z(1))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        e.kv_attention(z(1, 1, 64), z(1, 1, 16, 64), z(1, 1, 16, 64), z(1, 1), z(1, 1), z(1, 1), z(1))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        e.moe_forward(z(1, 16), z(1, 16), z(1, 32, 16), z(1, 32), z(1, 16, 16), z(1, 16), 1)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        e.token_logprobs(z(1, 16), z(1))
