"""Refusals of the cross-attention and cache-eviction entry points: bad arguments come back as codes before any device is
touched, and as RuntimeError from the Python layers."""
import ctypes as C
import importlib
import math
import sys

import pytest
import torch

from cuda_b200 import _lib as L
from cuda_b200 import compat, ops


@pytest.fixture(scope="module")
def lib():
    return L.load()


@pytest.fixture(scope="module")
def ext():
    sys.path.insert(0, compat.PATH)
    try:
        return importlib.import_module("fused_online_softmax_cuda")
    finally:
        sys.path.remove(compat.PATH)


def cross(**kw):
    p = L.CrossAttentionParams(q=0x1000, k=0x2000, v=0x3000, out=0x4000, q_strides=(2048, 512, 64), k_strides=(2048, 1024, 64),
                               v_strides=(2048, 1024, 64), out_strides=(2048, 512, 64), batch_size=2, num_q_heads=4, num_kv_heads=2,
                               q_len=8, kv_len=16, head_dim=64, dtype=L.BF16, softmax_scale=0.125)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


CROSS_BAD = [
    (dict(num_kv_heads=3), L.EINVAL), (dict(num_kv_heads=0), L.EINVAL), (dict(num_q_heads=0), L.EINVAL), (dict(head_dim=96), L.EINVAL),
    (dict(dtype=3), L.EINVAL), (dict(dtype=-1), L.EINVAL), (dict(softmax_scale=0.0), L.EINVAL), (dict(softmax_scale=-1.0), L.EINVAL),
    (dict(softmax_scale=math.nan), L.EINVAL), (dict(softmax_scale=math.inf), L.EINVAL), (dict(batch_size=-1), L.EINVAL),
    (dict(q_len=-1), L.EINVAL), (dict(kv_len=-1), L.EINVAL), (dict(q=None), L.EINVAL), (dict(k=None), L.EINVAL), (dict(v=None), L.EINVAL),
    (dict(out=None), L.EINVAL), (dict(q=0x1008), L.EALIGN), (dict(k=0x1002), L.EALIGN), (dict(out=0x1004), L.EALIGN),
    (dict(batch_size=70000), L.EINVAL), (dict(q_len=2 ** 30), L.EINVAL), (dict(kv_len=2 ** 30 + 5), L.EINVAL),
    (dict(q_strides=(2048, 512, 63)), L.EALIGN), (dict(k_strides=(2048, -1024, 64)), L.EALIGN), (dict(v_strides=(2044, 1024, 64)), L.EALIGN),
    (dict(out_strides=(0, 512, 64)), L.EALIGN), (dict(out_strides=(2048, 512, 32)), L.EALIGN), (dict(lse=0x1002), L.EALIGN),
    (dict(kv_lens=0x1001), L.EALIGN),
]


@pytest.mark.parametrize("kw,code", CROSS_BAD, ids=lambda x: str(x)[:40])
def test_cross_refusals(lib, kw, code):
    assert lib.cuda_llm_cross_attention(C.byref(cross(**kw)), None) == code
    assert lib.cuda_llm_last_cuda_error()


def test_nothing_to_do(lib):
    assert lib.cuda_llm_cross_attention(None, None) == L.EINVAL
    assert lib.cuda_llm_cross_attention(C.byref(cross(batch_size=0)), None) == L.OK
    assert lib.cuda_llm_cross_attention(C.byref(cross(q_len=0)), None) == L.OK
    assert lib.cuda_llm_cross_attention_wait_timeouts(None) == L.EINVAL
    assert lib.cuda_llm_kv_accumulate_weights(None, None) == L.EINVAL
    assert lib.cuda_llm_kv_accumulate_weights(C.byref(weights(num_seqs=0)), None) == L.OK
    assert lib.cuda_llm_kv_evict(None, None) == L.EINVAL
    assert lib.cuda_llm_kv_evict(C.byref(evict(num_seqs=0)), None) == L.OK


def weights(**kw):
    p = L.KvWeightsParams(query=0x1000, key_cache=0x2000, k_scale=0x3000, block_tables=0x4000, context_lens=0x5000, lse=0x6000, scores=0x7000,
                          score_strides=(512, 256), num_seqs=2, total_q=2, num_q_heads=4, num_kv_heads=2, head_dim=64, page_size=16,
                          max_blocks_per_seq=16, num_blocks=40, max_tokens=256, max_q_len=1, q_dtype=L.BF16, k_format=L.KV_FP8_E4M3,
                          scale_mode=L.SCALE_PER_TOKEN, is_causal=1, softmax_scale=0.125, decay=1.0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


WEIGHTS_BAD = [
    (dict(num_kv_heads=3), L.EINVAL), (dict(head_dim=80), L.EINVAL), (dict(page_size=8), L.EINVAL), (dict(q_dtype=7), L.EINVAL),
    (dict(k_format=L.KV_INT8), L.EINVAL), (dict(k_format=L.KV_F32), L.EINVAL), (dict(k_format=L.KV_FP4_E2M1), L.EINVAL),
    (dict(k_format=L.KV_F16), L.EINVAL), (dict(scale_mode=9), L.EINVAL), (dict(softmax_scale=0.0), L.EINVAL), (dict(decay=1.5), L.EINVAL),
    (dict(decay=-0.1), L.EINVAL), (dict(decay=math.nan), L.EINVAL), (dict(num_seqs=-1), L.EINVAL), (dict(total_q=3), L.EINVAL),
    (dict(num_blocks=0), L.EINVAL), (dict(key_cache=None), L.EINVAL), (dict(k_scale=None), L.EINVAL), (dict(lse=None), L.EINVAL),
    (dict(scores=None), L.EINVAL), (dict(key_cache=0x2008), L.EALIGN), (dict(query=0x1004), L.EALIGN), (dict(scores=0x7002), L.EALIGN),
    (dict(num_seqs=70000, total_q=70000), L.EINVAL),
]


@pytest.mark.parametrize("kw,code", WEIGHTS_BAD, ids=lambda x: str(x)[:40])
def test_weights_refusals(lib, kw, code):
    assert lib.cuda_llm_kv_accumulate_weights(C.byref(weights(**kw)), None) == code


def evict(**kw):
    p = L.KvEvictParams(scores=0x1000, new_scores=None, key_cache=0x2000, value_cache=0x3000, k_scale=0x4000, v_scale=0x5000,
                        block_tables=0x6000, new_block_tables=0x6000, context_lens=0x7000, new_context_lens=0x8000, kept=0x9000,
                        score_strides=(512, 256), num_seqs=2, num_kv_heads=2, head_dim=64, page_size=16, max_blocks_per_seq=16,
                        new_max_blocks_per_seq=16, num_blocks=40, max_tokens=256, k_format=L.KV_FP8_E4M3, v_format=L.KV_FP8_E4M3,
                        scale_mode=L.SCALE_PER_TOKEN, budget=64, sink=4, recent=16)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


EVICT_BAD = [
    (dict(num_kv_heads=0), L.EINVAL), (dict(head_dim=32), L.EINVAL), (dict(page_size=24), L.EINVAL), (dict(k_format=L.KV_INT8), L.EINVAL),
    (dict(k_format=L.KV_BF16), L.EINVAL), (dict(v_format=L.KV_F16), L.EINVAL), (dict(v_format=L.KV_FP4_E2M1), L.EINVAL),
    (dict(scale_mode=L.SCALE_PER_BLOCK), L.EINVAL), (dict(scale_mode=-1), L.EINVAL), (dict(budget=0), L.EINVAL), (dict(budget=-3), L.EINVAL),
    (dict(sink=-1), L.EINVAL), (dict(recent=-1), L.EINVAL), (dict(sink=40, recent=40), L.EINVAL), (dict(budget=2 ** 31 - 1, sink=2 ** 31 - 1, recent=1), L.EINVAL),
    (dict(max_tokens=L.EVICT_MAX_TOKENS + 1), L.EINVAL), (dict(num_blocks=0), L.EINVAL), (dict(num_seqs=70000), L.EINVAL),
    (dict(scores=None), L.EINVAL), (dict(kept=None), L.EINVAL), (dict(k_scale=None), L.EINVAL), (dict(new_context_lens=0x7000), L.EINVAL),
    (dict(new_max_blocks_per_seq=3), L.EINVAL), (dict(new_block_tables=0xa000, new_max_blocks_per_seq=3), L.EINVAL),
    (dict(key_cache=0x2004), L.EALIGN), (dict(kept=0x9002), L.EALIGN),
]


@pytest.mark.parametrize("kw,code", EVICT_BAD, ids=lambda x: str(x)[:40])
def test_evict_refusals(lib, kw, code):
    assert lib.cuda_llm_kv_evict(C.byref(evict(**kw)), None) == code
    assert lib.cuda_llm_last_cuda_error()


def test_python_layers_refuse_cpu_tensors(ext):
    q = torch.zeros(2, 4, 3, 64)
    k = torch.zeros(2, 2, 5, 64)
    kc = torch.zeros(4, 2, 64, 16, dtype=torch.uint8)
    sc = torch.zeros(4, 2, 16)
    bt = torch.zeros(2, 2, dtype=torch.int32)
    cl = torch.ones(2, dtype=torch.int32)
    scores = torch.zeros(2, 2, 32)
    for m in (ops, ext):
        with pytest.raises(RuntimeError, match="Inputs must be on CUDA"):
            m.cross_attention_forward(q, k, k)
        with pytest.raises(RuntimeError, match="Inputs must be on CUDA"):
            m.kv_cache_accumulate_weights(q[:, :, 0], kc, sc, bt, cl, torch.zeros(2, 4), scores)
        with pytest.raises(RuntimeError, match="Inputs must be on CUDA"):
            m.kv_cache_evict(scores, kc, kc, sc, sc, bt, cl, 8)


def test_extension_signatures(ext):
    for fn, names in ((ext.cross_attention_forward, ("q", "k", "v", "kv_lens", "softmax_scale", "return_lse")),
                      (ext.kv_cache_accumulate_weights, ("query", "key_cache", "k_scale", "block_tables", "context_lens", "lse", "scores", "softmax_scale",
                                                         "cu_q_lens", "max_q_len", "is_causal", "decay", "kv_format", "status")),
                      (ext.kv_cache_evict, ("scores", "key_cache", "value_cache", "k_scale", "v_scale", "block_tables", "context_lens", "budget", "sink",
                                            "recent", "new_block_tables", "new_scores", "kv_format", "status"))):
        for name in names:
            assert name + ":" in fn.__doc__, name


@pytest.mark.parametrize("strides", [(0, 256), (512, 0), (256, 256), (512, 255), (511, 256), (-512, 256)])
def test_score_rows_that_overlap(lib, strides):
    pair = (C.c_int64 * 2)(*strides)
    assert lib.cuda_llm_kv_accumulate_weights(C.byref(weights(score_strides=pair)), None) == L.EINVAL
    assert lib.cuda_llm_kv_evict(C.byref(evict(new_scores=0xb000, new_score_strides=(C.c_int64 * 2)(*[x // 4 for x in strides]))), None) == L.EINVAL


def test_limits_of_the_row_lengths(lib):
    wide = (C.c_int64 * 2)(2 ** 33, 2 ** 31)
    assert lib.cuda_llm_kv_accumulate_weights(C.byref(weights(max_tokens=2 ** 30 + 1, score_strides=wide)), None) == L.EINVAL
    assert lib.cuda_llm_kv_evict(C.byref(evict(budget=2 ** 30 + 1)), None) == L.EINVAL
    same = (C.c_int64 * 2)(1024, 512)
    assert lib.cuda_llm_kv_evict(C.byref(evict(new_scores=0x1000, new_score_strides=same)), None) == L.EINVAL
