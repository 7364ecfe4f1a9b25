"""Accumulated weights where the queries brought none of the tokens (``keep_old``: an encoder's states in a paged cache).  The formula and
its tolerance are those of ``test_cache_eviction_gpu``; an old score adds one rounding of its product and of the sum, 2^-23 of it."""
import importlib
import math
import sys

import pytest
import torch

import test_cache_eviction_gpu as E
from cuda_b200 import compat, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ext():
    sys.path.insert(0, compat.PATH)
    try:
        return importlib.import_module("fused_online_softmax_cuda")
    finally:
        sys.path.remove(compat.PATH)


def expect(wl, lse, scores, causal, decay):
    got, tol = E.weights_formula(wl, lse, torch.zeros_like(scores), causal, 0.0)
    old = scores.double() * decay if decay else torch.zeros_like(scores, dtype=torch.float64)
    live = torch.arange(scores.shape[2], device="cuda").view(1, 1, -1) < wl.context_lens.view(-1, 1, 1)
    return torch.where(live, old + got, scores.double()), tol + 2.0 ** -23 * (old.abs() + got)


def check(wl, causal, decay):
    lse = E.true_lse(wl, causal)
    scores = torch.rand(wl.num_seqs, wl.num_kv_heads, wl.block_tables.shape[1] * wl.page_size, device="cuda")
    want, tol = expect(wl, lse, scores, causal, decay)
    if decay == 0:
        scores.fill_(math.nan)  # not read
    E.accumulate(wl, lse, scores, is_causal=causal, decay=decay, keep_old=True)
    for s in range(wl.num_seqs):
        n = int(wl.context_lens[s])
        assert ((scores[s, :, :n].double() - want[s, :, :n]).abs() <= tol[s, :, :n]).all(), s


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("decay", [1.0, 0.75, 0.0])
@pytest.mark.parametrize("q_lens", [None, [1, 3, 4, 2, 1], [40, 33, 1, 90, 64]])
@pytest.mark.parametrize("fmt", ["fp8_token", "mx8", "bf16"])
def test_old_scores_count_everywhere(fmt, q_lens, decay, causal):
    check(E.cache("w", lens=[333, 40, 1, 129, 2900], q_lens=q_lens, hq=8, hkv=2, d=128, page=16, fmt=fmt, seed=7), causal, decay)


@pytest.mark.parametrize("q_len,page", [(1, 16), (8, 32), (40, 64), (90, 16)])  # one and two blocks of rows, the window kernel (90)
def test_two_calls_add_up(q_len, page):
    """Every state holds the weight of both steps, the last ones too; an equal second step doubles all scores."""
    wl = E.cache("w", lens=[700, 5, 1500], q_lens=[q_len] * 3 if q_len <= 5 else [q_len, 5, q_len], hq=8, hkv=4, d=64, page=page, fmt="bf16", seed=q_len)
    scores = torch.zeros(3, 4, wl.block_tables.shape[1] * page, device="cuda")
    lse = E.true_lse(wl, False)
    E.accumulate(wl, lse, scores, is_causal=False, keep_old=True)
    first = scores.clone()
    E.accumulate(wl, lse, scores, is_causal=False, keep_old=True)
    assert torch.equal(scores, 2 * first)  # exact: doubling rounds nothing
    wl.query = torch.randn_like(wl.query)
    lse = E.true_lse(wl, False)
    want, tol = expect(wl, lse, scores, False, 1.0)
    E.accumulate(wl, lse, scores, is_causal=False, keep_old=True)
    for s, n in enumerate(wl.context_lens.tolist()):
        assert ((scores[s, :, :n].double() - want[s, :, :n]).abs() <= tol[s, :, :n]).all()


def test_both_python_layers(ext):
    wl = E.cache("w", lens=[70, 301], q_lens=[3, 2], hq=8, hkv=2, d=64, page=16, seed=3)
    lse = E.true_lse(wl, False)
    base = torch.rand(2, 2, wl.block_tables.shape[1] * 16, device="cuda")
    for keep in (False, True):
        got = [m.kv_cache_accumulate_weights(wl.query, wl.key_cache, wl.k_scale, wl.block_tables, wl.context_lens, lse, base.clone(), wl.softmax_scale,
                                             cu_q_lens=wl.cu_q_lens, max_q_len=wl.max_q_len, is_causal=False, decay=0.5, keep_old=keep) for m in (ops, ext)]
        assert torch.equal(*got)
        if keep:
            assert (got[0][0, :, 67:70] >= 0.5 * base[0, :, 67:70]).all()
            assert torch.equal(got[0][0, :, :67], before[0, :, :67])
        before = got[0]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens,declared", [(None, 1), ([1, 2, 4, 1], 4), ([8, 30, 5, 32], 32), ([8, 30, 5, 32], 1), ([60, 90, 40, 100], 100)])
@pytest.mark.parametrize("fmt,q_dtype", [("fp8_token", torch.bfloat16), ("fp8_token", torch.float16), ("fp8_head", torch.float32), ("mx8", torch.bfloat16),
                                         ("mx8", torch.float16), ("bf16", torch.bfloat16)])
def test_rows_that_saw_nothing_add_nothing(fmt, q_dtype, q_lens, declared, causal):
    """Rows with a log-sum-exp of -inf (the padding of a batch) count nothing, whatever their queries hold: the other rows' bits stay."""
    wl = E.cache("w", lens=[130, 2900, 333, 1500], q_lens=q_lens, hq=8, hkv=2, d=64, page=16, fmt=fmt, q_dtype=q_dtype, seed=5)
    wl.max_q_len = declared
    lse = E.true_lse(wl, causal)
    none = torch.rand(lse.shape, device="cuda") < 0.3
    none[-1], none[0, :4] = True, True  # a last row, a whole group
    lse[none] = -math.inf
    base = torch.rand(4, 2, wl.block_tables.shape[1] * 16, device="cuda")
    wl.query[none] = 0.0
    want = E.accumulate(wl, lse, base.clone(), is_causal=causal)
    for bad in (math.nan, math.inf, -math.inf):
        wl.query[none] = bad
        assert torch.equal(E.accumulate(wl, lse, base.clone(), is_causal=causal), want), bad


@pytest.mark.parametrize("q_lens", [None, [2, 1], [30, 9], [90, 70]])
@pytest.mark.parametrize("fmt", ["fp8_token", "mx8", "bf16"])
def test_keys_that_only_rows_that_saw_nothing_meet(fmt, q_lens):
    """Keys that are not finite where every row has a log-sum-exp of -inf: the old scores fade and nothing is added."""
    wl = E.cache("w", lens=[2900, 333], q_lens=q_lens, hq=8, hkv=2, d=128, page=16, fmt=fmt, seed=9)
    lse = torch.full((wl.query.shape[0], 8), -math.inf, device="cuda")
    for t in (0, 17, 300):
        page = wl.block_tables[:, t // 16].long()
        wl.key_cache[page, :, 3, t % 16] = math.nan if fmt == "bf16" else 0x7f
        if fmt == "bf16":
            wl.key_cache[page, :, 5, (t + 1) % 16] = math.inf
    base = torch.rand(2, 2, wl.block_tables.shape[1] * 16, device="cuda")
    got = E.accumulate(wl, lse, base.clone(), is_causal=False, decay=0.5, keep_old=True)
    for s, n in enumerate(wl.context_lens.tolist()):
        assert torch.equal(got[s, :, :n], 0.5 * base[s, :, :n]) and torch.equal(got[s, :, n:], base[s, :, n:])


@pytest.mark.parametrize("fmt", ["fp8_token", "mx8", "bf16"])
@pytest.mark.parametrize("group,n", [(4, 32), (1, 33), (5, 40)])
def test_log_sum_exp_of_a_window_from_one_decode(group, n, fmt):
    """The last n queries of two prompts in one decode: every 16 // group of them stand as a sequence of their own, with the same pages and
    the context up to them.  Each row's weights then add up to 1 within the tolerance of the decode's log-sum-exp, 1e-3."""
    wl = E.cache("w", lens=[700, 90], q_lens=[n, n], hq=2 * group, hkv=2, d=128, page=16, fmt=fmt, seed=n)
    step = 16 // group
    ends = [min(n, i + step) for i in range(0, n, step)]
    lens = torch.tensor([c - n + e for c in wl.context_lens.tolist() for e in ends], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0] + [s * n + e for s in range(2) for e in ends], dtype=torch.int32, device="cuda")
    tables = wl.block_tables.repeat_interleave(len(ends), 0).contiguous()
    if fmt == "bf16":
        _, lse = ops.paged_attention_forward(wl.query, wl.key_cache, wl.value_cache, tables, lens, wl.softmax_scale, cu_q_lens=cu, max_q_len=step,
                                             return_lse=True)
    else:
        _, lse = ops.fp8_paged_attention_forward(wl.query, wl.key_cache, wl.value_cache, wl.k_scale, wl.v_scale, tables, lens, wl.softmax_scale,
                                                 cu_q_lens=cu, max_q_len=step, return_lse=True)
    assert ((lse - E.true_lse(wl, True)).abs() < 1e-3).all()
    scores = E.accumulate(wl, lse, torch.zeros(2, 2, wl.block_tables.shape[1] * 16, device="cuda"))
    for s, c in enumerate(wl.context_lens.tolist()):
        assert ((scores[s, :, :c].sum(-1) - n * group).abs() < 1e-3 * n * group).all()
