"""Layouts that the cross-attention and cache-eviction entry points cannot address: refused by the C entries before any device is touched,
copied by the Python layers."""
import ctypes as C

import pytest
import torch

from cuda_b200 import _lib as L
from cuda_b200 import ops
from test_cross_evict_refusals_cpu import cross, evict, lib  # noqa: F401  (lib is a fixture)


# ---- one position that stands for all of them (a stride of 0): a tensor map cannot say so
@pytest.mark.parametrize("dtype", [L.F16, L.BF16])
@pytest.mark.parametrize("kw", [dict(q_strides=(2048, 512, 0)), dict(k_strides=(2048, 1024, 0)), dict(v_strides=(2048, 1024, 0)),
                                dict(q_strides=(2048, 512, 0), q_len=100), dict(k_strides=(0, 0, 0)), dict(v_strides=(0, 64, 0), q_len=100)], ids=str)
def test_position_stride_of_zero_is_refused_in_16_bits(lib, kw, dtype):  # noqa: F811
    assert lib.cuda_llm_cross_attention(C.byref(cross(dtype=dtype, **kw)), None) == L.EALIGN


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_python_copies_what_the_kernels_cannot_address(dtype):
    x = torch.randn(2, 3, 1, 64).to(dtype)
    spread = x.expand(2, 3, 5, 64)  # positions share one row
    got = ops._addressable(spread)
    assert torch.equal(got, spread)
    assert (got is spread) == (dtype == torch.float32) and (dtype == torch.float32 or got.stride(2) > 0)
    for fine in (x, torch.randn(1, 3, 5, 64).to(dtype).expand(2, 3, 5, 64), torch.randn(2, 1, 5, 64).to(dtype).expand(2, 3, 5, 64), spread[:, :, :1]):
        assert ops._addressable(fine) is fine  # batch rows and heads may share, a single position may carry any stride


# ---- scores compacted in place: a row is read to the end of its context while other rows are written
@pytest.mark.parametrize("strides,kw", [((200, 100), {}), ((512, 100), {}), ((100, 512), {}), ((400, 200), dict(budget=199)), ((512, 255), {}),
                                        ((240, 120), dict(max_tokens=121)), ((128, 64), dict(max_blocks_per_seq=5, new_max_blocks_per_seq=5))], ids=str)
def test_rows_of_scores_that_overlap_are_not_compacted_in_place(lib, strides, kw):  # noqa: F811
    pair = (C.c_int64 * 2)(*strides)
    assert lib.cuda_llm_kv_evict(C.byref(evict(new_scores=0x1000, score_strides=pair, new_score_strides=pair, **kw)), None) == L.EINVAL


@pytest.mark.parametrize("strides,kw", [((512, 256), {}), ((256, 512), {}), ((240, 120), dict(max_tokens=120)),
                                        ((160, 80), dict(max_blocks_per_seq=5, new_max_blocks_per_seq=5)), ((80, 1), dict(num_kv_heads=1, max_tokens=80))], ids=str)
def test_rows_of_scores_apart_may_be(lib, strides, kw):  # noqa: F811
    """Accepted as far as the device, which is not there."""
    if torch.cuda.is_available():
        pytest.skip("addresses are made up")
    pair = (C.c_int64 * 2)(*strides)
    assert lib.cuda_llm_kv_evict(C.byref(evict(new_scores=0x1000, score_strides=pair, new_score_strides=pair, **kw)), None) not in (L.EINVAL, L.EALIGN, L.OK)
