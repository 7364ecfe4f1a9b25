"""Cross attention and eviction where a call is larger, busier or odder than usual: more sequences than a launch or a block holds,
more query rows than declared, offsets past 32 bits, non-finite scores, shared pages, many calls at once.  Formulas and
tolerances are those of ``test_cross_attention_gpu`` and ``test_cache_eviction_gpu``."""
import math

import pytest
import torch

import test_cache_eviction_gpu as E
import test_cross_attention_gpu as X
from cuda_b200 import _lib as L
from cuda_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = ["bf16", "f16", "f32"]


# ---- cross attention
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 40])
def test_more_sequences_than_threads_of_a_block(sq, dtype):
    b = 401
    lens = [(37 * i) % 70 for i in range(b)]
    q, k, v = X.make(b, 2, 1, sq, 67, 64, X.DTYPES[dtype], seed=sq)
    out, lse = ops.cross_attention_forward(q, k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"), return_lse=True)
    X.check(out, lse, *X.formula(q, k, v, lens, 0.125), q.dtype, 64, 67)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 20, 150])
@pytest.mark.parametrize("d", [64, 128])
def test_scores_that_are_not_finite(sq, d, dtype):
    """Row 0: one state scores -inf and weighs nothing; 1: all do, zeros; 2: one scores +inf, 3: one NaN: NaN."""
    q, k, v = X.make(4, 4, 2, sq, 200, d, X.DTYPES[dtype], seed=5)
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    k[0, :, 150, 0] = -math.inf
    k[1, :, :, 0] = -math.inf
    k[2, :, 7, 0] = math.inf
    k[3, :, 199, 3] = math.nan
    out, lse = ops.cross_attention_forward(q, k, v, return_lse=True)
    keep = [i for i in range(200) if i != 150]
    k[0, :, 150, 0] = 0.0
    want = X.formula(q[:1], k[:1, :, keep], v[:1, :, keep], None, 1 / math.sqrt(d))
    X.check(out[:1], lse[:1], *want, q.dtype, d, 200)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
    assert out[2:].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 70])
def test_states_past_two_to_the_31_elements(sq, dtype):
    """Two batch rows whose states lie 2^31 + 2^20 elements apart, K and V in one buffer."""
    dt, n, d = X.DTYPES[dtype], 130, 64
    far = 2 ** 31 + 2 ** 20
    buf = torch.empty(far + 2 * n * d, dtype=dt, device="cuda")
    k = buf.as_strided((2, 1, n, d), (far, n * d, d, 1))
    v = buf.as_strided((2, 1, n, d), (far, n * d, d, 1), n * d)
    q, k0, v0 = X.make(2, 2, 1, sq, n, d, dt, seed=3)
    k.copy_(k0)
    v.copy_(v0)
    assert k.data_ptr() == buf.data_ptr()
    out = ops.cross_attention_forward(q, k, v)
    assert torch.equal(out, ops.cross_attention_forward(q, k0, v0))
    X.check(out, None, *X.formula(q, k0, v0, None, 0.125), dt, d, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 90])
def test_shared_states_of_all_rows_and_heads(sq, dtype):
    """Beams: batch rows, heads or both with a stride of zero."""
    dt, d = X.DTYPES[dtype], 128
    q, k, v = X.make(5, 6, 3, sq, 190, d, dt, seed=9)
    for pick in ((slice(0, 1), slice(None)), (slice(None), slice(0, 1)), (slice(0, 1), slice(0, 1))):
        ke, ve = k[pick].expand(5, 3, 190, d), v[pick].expand(5, 3, 190, d)
        assert torch.equal(ops.cross_attention_forward(q, ke, ve), ops.cross_attention_forward(q, ke.contiguous(), ve.contiguous()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_calls_at_once_on_several_streams_and_graphs(dtype):
    dt = X.DTYPES[dtype]
    cases = [X.make(3, 8, 2, sq, 777, 128, dt, seed=sq) for sq in (1, 3, 33, 200)]
    want = [ops.cross_attention_forward(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    graphs, outs = [], []
    for c, s in zip(cases, streams):
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(ops.cross_attention_forward(*c))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, s, g in zip(cases, streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
                got.append(ops.cross_attention_forward(*c))
    torch.cuda.synchronize()
    for w, a, b in zip(want, outs, got):
        assert torch.equal(w, a) and torch.equal(w, b)


# ---- accumulated weights
@pytest.mark.parametrize("fmt", ["fp8_token", "mx8", "bf16"])
@pytest.mark.parametrize("q_lens", [[1, 40, 9, 2], [300, 5, 33, 1]])
@pytest.mark.parametrize("declared", [1, 4, 200])
def test_more_or_fewer_query_rows_than_declared(q_lens, declared, fmt):
    wl = E.cache("w", lens=[50, 170, 33, 90] if q_lens[0] == 1 else [310, 170, 33, 90], q_lens=q_lens, hq=8, hkv=2, d=128, page=16, fmt=fmt, seed=declared)
    wl.max_q_len = declared
    E.check_weights(wl)


@pytest.mark.parametrize("q_dtype", [torch.float16, torch.float32])
def test_rows_in_and_out_of_shared_memory(q_dtype):
    """A KV head's rows fit the block (128 of them) or do not, in turn, sequence after sequence."""
    E.check_weights(E.cache("w", lens=[200] * 6, q_lens=[32, 33, 31, 200, 1, 32], hq=8, hkv=2, d=64, page=64, q_dtype=q_dtype, seed=2))


@pytest.mark.parametrize("fmt", ["fp8_token", "fp8_head", "fp8_block", "mx8", "bf16", "f16"])
@pytest.mark.parametrize("d,page", [(64, 16), (64, 64), (128, 16), (128, 32), (128, 64)])
@pytest.mark.parametrize("q_len", [40, 90, 150])
def test_windows_of_a_prompt(fmt, d, page, q_len):
    """One, two and three blocks of 128 rows per KV head (40 to 150 queries of 4 heads), several tiles and heads for every CTA,
    sequences without queries, of one token, of fewer tokens than queries."""
    dt = torch.float16 if fmt == "f16" else torch.bfloat16
    E.check_weights(E.cache("w", lens=[2900, 260, 0, 1, 4100, 700, 257, q_len], q_lens=[q_len, q_len, 0, 1, q_len, 0, 33, q_len], hq=32, hkv=8, d=d, page=page,
                            fmt=fmt, q_dtype=dt, seed=d + page), causal=q_len != 90, decay=0.5)


@pytest.mark.parametrize("fmt", ["fp8_token", "fp8_block"])
def test_windows_of_a_prompt_in_other_layouts(fmt):
    """fp16 queries on 8-bit keys, a group that is no power of two, one KV head; a page that is not in the pool."""
    E.check_weights(E.cache("w", lens=[1500, 300], q_lens=[70, 64], hq=5, hkv=1, d=128, page=16, fmt=fmt, q_dtype=torch.float16, seed=3))
    wl = E.cache("w", lens=[1500, 900], q_lens=[70, 64], hq=12, hkv=4, d=64, page=32, fmt=fmt, seed=4)
    lse = E.true_lse(wl, True)
    base = torch.rand(2, 4, wl.block_tables.shape[1] * 32, device="cuda")
    fine = E.accumulate(wl, lse, base.clone())
    wl.block_tables[0, 7], wl.block_tables[1, 3] = -5, wl.key_cache.shape[0]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = E.accumulate(wl, lse, base.clone(), status=status)
    assert int(status) == L.ST_BAD_BLOCK
    fine[0, :, 7 * 32:8 * 32], fine[1, :, 3 * 32:4 * 32] = base[0, :, 7 * 32:8 * 32], base[1, :, 3 * 32:4 * 32]
    assert torch.equal(got, fine)


@pytest.mark.parametrize("ragged", [False, True])
def test_more_sequences_than_a_launch_holds(ragged):
    n = 2100
    lens = [(13 * i) % 50 for i in range(n)]
    wl = E.cache("w", lens=lens, q_lens=[(i % 3) for i in range(n)] if ragged else None, hq=2, hkv=2, d=64, page=16, seed=1)
    total = wl.query.shape[0]
    lse = torch.rand(total, 2, device="cuda") * 4
    base = torch.rand(n, 2, wl.block_tables.shape[1] * 16, device="cuda")
    got = E.accumulate(wl, lse, base.clone(), decay=0.5)
    for a in range(0, n, 700):  # the same in pieces
        piece = slice(a, a + 700)
        if ragged:
            cu, q, l = wl.cu_q_lens[a:a + 701].contiguous(), wl.query, lse
        else:
            cu, q, l = None, wl.query[piece].contiguous(), lse[piece].contiguous()
        part = ops.kv_cache_accumulate_weights(q, wl.key_cache, wl.k_scale, wl.block_tables[piece].contiguous(), wl.context_lens[piece].contiguous(), l,
                                               base[piece].clone(), wl.softmax_scale, cu_q_lens=cu, max_q_len=wl.max_q_len, decay=0.5)
        assert torch.equal(part, got[piece])


def _far_pool(wl, blocks):
    """The same cache in a pool of `blocks` pages, its pages the last of it."""
    n = wl.key_cache.shape[0]
    for name in ("key_cache", "value_cache", "k_scale", "v_scale"):
        t = getattr(wl, name)
        big = torch.empty((blocks, *t.shape[1:]), dtype=t.dtype, device="cuda")
        big[blocks - n:] = t
        setattr(wl, name, big)
    wl.block_tables += blocks - n
    return wl


def test_pages_past_two_to_the_32_bytes():
    def fresh():
        return E.cache("w", lens=[333, 64, 201], hq=8, hkv=2, d=128, page=64, seed=6)
    near, far = fresh(), _far_pool(fresh(), 2 ** 32 // (2 * 128 * 64) + 50)
    lse = E.true_lse(near, True)
    base = torch.rand(3, 2, near.block_tables.shape[1] * 64, device="cuda")
    a, b = E.accumulate(near, lse, base.clone()), E.accumulate(far, lse, base.clone())
    assert torch.equal(a, b)
    kept, _ = E.evict(near, a, 100, sink=2, recent=5)
    kept_far, _ = E.evict(far, b, 100, sink=2, recent=5)
    n = near.key_cache.shape[0]
    assert torch.equal(kept, kept_far)
    for x in ("key_cache", "value_cache", "k_scale", "v_scale"):
        assert E.same(getattr(near, x), getattr(far, x)[-n:]), x


def test_score_rows_that_overlap_are_refused():
    wl = E.cache("w", lens=[40, 40], hq=4, hkv=2, d=64, page=16, seed=1)
    row = torch.zeros(1, 1, 48, device="cuda")
    lse = torch.zeros(2, 4, device="cuda")
    with pytest.raises(RuntimeError):
        E.accumulate(wl, lse, row.expand(2, 2, 48))
    with pytest.raises(RuntimeError):
        E.evict(wl, torch.zeros(2, 2, 48, device="cuda"), 20, new_scores=row.expand(2, 2, 48))
    # read only, they may: every head keeps the same tokens
    kept, _ = E.evict(wl, torch.rand(1, 1, 48, device="cuda").expand(2, 2, 48), 20)
    assert torch.equal(kept[0, 0], kept[0, 1]) and torch.equal(kept[0], kept[1])


@pytest.mark.parametrize("q_lens", [None, [3, 40, 100]])
@pytest.mark.parametrize("hq", [2, 6, 16])
@pytest.mark.parametrize("fmt", ["bf16", "fp8_token", "mx8"])
def test_keys_that_are_not_finite(fmt, hq, q_lens):
    """A token that scores -inf in every row weighs nothing, one that is NaN becomes NaN, and no other token feels them."""
    wl = E.cache("w", lens=[70, 150, 333], q_lens=q_lens, hq=hq, hkv=2, d=64, page=16, fmt=fmt, seed=hq)
    wl.query[..., 0] = 1.0
    lse = E.true_lse(wl, True)
    base = torch.rand(3, 2, wl.block_tables.shape[1] * 16, device="cuda")
    fine = E.accumulate(wl, lse, base.clone())
    tokens = {0: 5, 1: 20, 2: 200}
    for s, t in tokens.items():
        page = int(wl.block_tables[s, t // 16])
        if fmt == "bf16":
            wl.key_cache[page, :, 0, t % 16] = -math.inf
        wl.key_cache[page, :, 3, t % 16 + 1] = math.nan if fmt == "bf16" else 0x7f
    got = E.accumulate(wl, lse, base.clone())
    same = torch.ones_like(base, dtype=torch.bool)
    for s, t in tokens.items():
        assert got[s, :, t + 1].isnan().all()
        same[s, :, t + 1] = False
        if fmt == "bf16":
            assert torch.equal(got[s, :, t], base[s, :, t])
            same[s, :, t] = False
    assert torch.equal(got[same], fine[same])


def test_all_kernels_at_once():
    """Windows, decode weights, prompt attention and eviction on four streams, three times over: the results of one at a time."""
    win = E.cache("w", lens=[3000, 1700], q_lens=[40, 33], hq=32, hkv=8, d=128, page=16, seed=1)
    dec = E.cache("w", lens=[900] * 8, hq=8, hkv=2, d=64, page=16, fmt="bf16", seed=2)
    evi = [E.cache("w", lens=[900, 1200], hq=8, hkv=2, d=64, page=16, seed=3) for _ in range(4)]
    lse = [E.true_lse(x, True) for x in (win, dec)]
    base = [torch.rand(x.num_seqs, x.num_kv_heads, x.block_tables.shape[1] * 16, device="cuda") for x in (win, dec, evi[0])]
    cross = X.make(2, 8, 2, 300, 900, 64, torch.bfloat16, seed=4)
    jobs = [lambda i: E.accumulate(win, lse[0], base[0].clone()), lambda i: E.accumulate(dec, lse[1], base[1].clone()),
            lambda i: ops.cross_attention_forward(*cross), lambda i: E.evict(evi[i], base[2], 500, sink=1, recent=9)[0]]
    want = [job(0) for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for i in range(1, 4):
        got = []
        for s, job in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(job(i))
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert torch.equal(w, g)
        assert E.same(evi[i].key_cache, evi[0].key_cache) and E.same(evi[i].v_scale, evi[0].v_scale)


# ---- eviction
@pytest.mark.parametrize("fmt,d", [("mx4v", 64), ("mx4v", 128), ("fp8_token", 64), ("f32", 64), ("bf16", 128)])
@pytest.mark.parametrize("page", [16, 64])
def test_several_runs_of_positions_in_place(fmt, d, page):
    wl = E.cache("e", lens=[9000, 4500, 4200], hq=1, hkv=1, d=d, page=page, fmt=fmt, seed=d)
    E.check_evict(wl, E.random_scores(wl, 3), 4300, sink=7, recent=31)


@pytest.mark.parametrize("page", [16, 64])
def test_kept_tokens_at_the_ends_of_a_long_row(page):
    """All kept tokens last, first, or alternating between far pages: the in-place move's longest and shortest ways."""
    wl = E.cache("e", lens=[7000] * 4, hq=2, hkv=1, d=64, page=page, seed=8)
    scores = torch.rand(4, 1, wl.block_tables.shape[1] * page, device="cuda")
    t = torch.arange(scores.shape[2], device="cuda")
    scores[0] += t > 4000
    scores[1] += t < 3000
    scores[2] += (t % page) == page - 1
    scores[3] += (t // page) % 2 == 1
    E.check_evict(wl, scores, 2999)


def test_scores_written_over_themselves_across_a_cluster():
    wl = E.cache("e", lens=[60000, 33000], hq=2, hkv=2, d=64, page=64, seed=12)
    E.check_evict(wl, E.random_scores(wl, 4, ties=True), 30000, sink=4, recent=100, scores_in_place=True)


def test_sequences_that_share_pages_leave_them_alone():
    """Two sequences with a common prefix evict into pages of their own."""
    wl = E.cache("e", lens=[500, 500], hq=2, hkv=2, d=64, page=16, seed=13)
    wl.block_tables[1, :20] = wl.block_tables[0, :20]
    E.check_evict(wl, E.random_scores(wl, 5), 300, sink=4, recent=16, in_place=False)


def test_budget_above_everything_and_narrow_rows():
    wl = E.cache("e", lens=[100, 0, 33], hq=2, hkv=2, d=64, page=16, seed=14)
    scores = E.random_scores(wl, 6)
    E.check_evict(wl, scores, 5000, sink=64, recent=64)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept, lens = E.evict(wl, scores[:, :, :50], 40, status=status)  # score rows end before the first sequence does
    assert lens.tolist() == [40, 0, 33] and int(status) == L.ST_BAD_CTX and int(kept[0].max()) < 50


def test_two_captured_evictions_at_once():
    """Each replay evicts a fresh copy of the same cache; nothing is shared between the graphs."""
    caches = [E.cache("g", lens=[900, 640, 1290], hq=8, hkv=2, d=64, page=16, seed=50 + i) for i in range(2)]
    start = [[x.clone() for x in (w.key_cache, w.value_cache, w.k_scale, w.v_scale)] for w in caches]
    scores = [E.random_scores(w, i) for i, w in enumerate(caches)]
    want = []
    for w, s, init in zip(caches, scores, start):
        kept, _ = E.evict(w, s, 300, sink=1, recent=3)
        want.append((kept, [x.clone() for x in (w.key_cache, w.value_cache, w.k_scale, w.v_scale)]))
    graphs, outs = [], []
    streams = [torch.cuda.Stream() for _ in caches]
    for w, s, st in zip(caches, scores, streams):
        st.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(E.evict(w, s, 300, sink=1, recent=3)[0])
        graphs.append(g)
    for _ in range(3):
        torch.cuda.synchronize()
        for w, init in zip(caches, start):
            for x, y in zip((w.key_cache, w.value_cache, w.k_scale, w.v_scale), init):
                x.copy_(y)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for w, k, (kept, state) in zip(caches, outs, want):
        assert torch.equal(k, kept)
        for x, y in zip((w.key_cache, w.value_cache, w.k_scale, w.v_scale), state):
            assert E.same(x, y)
