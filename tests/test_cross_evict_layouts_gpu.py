"""Cross attention and eviction on layouts beside the usual ones.  Formulas and tolerances are those of ``test_cross_attention_gpu``
and ``test_cache_eviction_gpu``."""
import importlib
import sys

import pytest
import torch

import test_cross_attention_gpu as X
from cuda_b200 import compat, ops

pytestmark = pytest.mark.gpu
DTYPES = ["bf16", "f16", "f32"]


@pytest.fixture(scope="module")
def ext():
    sys.path.insert(0, compat.PATH)
    try:
        return importlib.import_module("fused_online_softmax_cuda")
    finally:
        sys.path.remove(compat.PATH)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 20, 90])
@pytest.mark.parametrize("which", ["q", "k", "v", "qkv", "kv, all heads and rows too"])
def test_one_position_for_all(ext, which, sq, dtype):
    """Tensors expanded over their positions (a stride of 0) count as their contiguous copies."""
    dt, d, n = X.DTYPES[dtype], 64, 150
    q, k, v = X.make(2, 6, 3, sq, n, d, dt, seed=sq)
    if "q" in which:
        q = q[:, :, :1].expand(2, 6, sq, d)
    if "k" in which:
        k = k[:, :, -1:].expand(2, 3, n, d)
    if "v" in which:
        v = v[:, :, -1:].expand(2, 3, n, d)
    if "heads" in which:
        k, v = (x[1:, 2:, -1:].expand(2, 3, n, d) for x in (k, v))
    lens = torch.tensor([n, 77], dtype=torch.int32, device="cuda")
    want = ops.cross_attention_forward(q.contiguous(), k.contiguous(), v.contiguous(), lens, return_lse=True)
    X.check(*want, *X.formula(q, k, v, lens.tolist(), 0.125), dt, d, n)
    for m in (ops, ext):
        got = m.cross_attention_forward(q, k, v, lens, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_more_heads_than_a_grid_is_high():
    """30000 KV heads of three query heads, 33 rows each: the tensor-core kernel with one head per block."""
    q, k, v = X.make(1, 90000, 30000, 11, 5, 64, torch.bfloat16, seed=2)
    out, lse = ops.cross_attention_forward(q, k, v, return_lse=True)
    for h in (0, 13000, 29000):
        qh, kh, vh = q[:, 3 * h:3 * h + 3000], k[:, h:h + 1000], v[:, h:h + 1000]
        part = ops.cross_attention_forward(qh, kh, vh, return_lse=True)
        assert torch.equal(out[:, 3 * h:3 * h + 3000], part[0]) and torch.equal(lse[:, 3 * h:3 * h + 3000], part[1])
        X.check(*part, *X.formula(qh, kh, vh, None, 0.125), torch.bfloat16, 64, 5)


def test_count_of_timeouts_waits_for_side_streams():
    """It has to count what runs on any stream, also on one that does not wait for the default stream."""
    import ctypes
    from cuda_b200 import _lib as L
    side, n = torch.cuda.Stream(), ctypes.c_uint32(7)
    buf = torch.empty(2, 2 ** 28, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(100):  # a third of a millisecond each
            buf[0].copy_(buf[1])
    assert not side.query()
    assert L.load().cuda_llm_cross_attention_wait_timeouts(ctypes.byref(n)) == L.OK and n.value == 0
    assert side.query()


def test_rows_of_a_batch_do_not_feel_one_another():
    """The split over a cluster depends on the batch, so a row alone may differ in its last bits: each is within the tolerance of the formula."""
    for sq in (1, 33, 200):
        q, k, v = X.make(4, 8, 2, sq, 1777, 128, torch.bfloat16, seed=sq)
        lens = torch.tensor([1777, 900, 64, 1300], dtype=torch.int32, device="cuda")
        want = X.formula(q, k, v, lens.tolist(), 128 ** -0.5)
        X.check(*ops.cross_attention_forward(q, k, v, lens, return_lse=True), *want, torch.bfloat16, 128, 1777)
        for i in range(4):
            row = slice(i, i + 1)
            alone = ops.cross_attention_forward(q[row], k[row], v[row], lens[row], return_lse=True)
            X.check(*alone, *(x[row] if torch.is_tensor(x) else x for x in want), torch.bfloat16, 128, 1777)
