"""Accumulated attention weights of cached tokens and the eviction by them, against the formulas in 64 bits.

Tolerance of a weight: q (8 or 11 bits, or split into two 11-bit halves for fp32: 2^-22) times a code is exact in fp32, a sum of
D products carries at most (D + 4) 2^-24 of sum |q k|, the exponential 2^-21; the weights of R rows add at most R 2^-24.  With
L = scale * sum |q k| of a row that is a relative error of (D + 8) 2^-24 L + 2^-21 (+ 2^-21 L for fp32 queries) per weight, and
2^-24 of the old score."""
import math

import pytest
import torch

from cuda_b200 import _lib as L
from cuda_b200 import ops, workloads as W

pytestmark = pytest.mark.gpu


def cache(name, *, lens, hq, hkv, d, page, fmt="fp8_token", q_lens=None, q_dtype=torch.bfloat16, seed=0):
    mode = {"fp8_token": W.SCALE_PER_TOKEN, "fp8_head": W.SCALE_PER_HEAD, "fp8_block": W.SCALE_PER_BLOCK, "mx8": W.SCALE_MX_E8M0,
            "mx4v": W.SCALE_MX_E8M0}.get(fmt, W.SCALE_NONE)
    kw = {}
    if mode == W.SCALE_NONE:
        kw = dict(k_format=W.KV_F32, v_format=W.KV_F32, cache_dtype={"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[fmt])
    elif fmt == "mx4v":
        kw = dict(v_format=W.KV_FP4_E2M1)
    return W.build_workload(name, context_lens=lens, q_lens=q_lens, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, page_size=page,
                            q_dtype=q_dtype, scale_mode=mode, pool_factor=1.6, seed=seed, device="cuda", **kw)


def key_values(wl):
    """[num_blocks, Hkv, D, page] in 64 bits."""
    if wl.key_cache.dtype != torch.uint8:
        return wl.key_cache.double()
    x = wl.key_cache.view(torch.float8_e4m3fn).double()
    s = wl.k_scale
    if wl.k_scale_mode == W.SCALE_PER_HEAD:
        return x * s.double().view(1, -1, 1, 1)
    if wl.k_scale_mode == W.SCALE_PER_BLOCK:
        return x * s.double().view(*s.shape, 1, 1)
    if wl.k_scale_mode == W.SCALE_PER_TOKEN:
        return x * s.double().unsqueeze(2)
    return x * torch.exp2(s.double() - 127).repeat_interleave(32, dim=2)


def logits(wl, s, causal):
    """[q_len, Hq, ctx] in 64 bits (-inf where not seen) and sum |q k| scale."""
    ctx = int(wl.context_lens[s])
    a, b = (s, s + 1) if wl.cu_q_lens is None else (int(wl.cu_q_lens[s]), int(wl.cu_q_lens[s + 1]))
    group = wl.num_q_heads // wl.num_kv_heads
    pages = wl.block_tables[s, :(ctx + wl.page_size - 1) // wl.page_size].long()
    k = key_values(wl)[pages].permute(1, 0, 3, 2).reshape(wl.num_kv_heads, -1, wl.head_dim)[:, :ctx].repeat_interleave(group, 0)
    q = wl.query[a:b].double()
    x = torch.einsum("qhd,htd->qht", q, k) * wl.softmax_scale
    mag = torch.einsum("qhd,htd->qht", q.abs(), k.abs()) * wl.softmax_scale
    if causal:
        t = torch.arange(ctx, device=x.device)
        j = torch.arange(b - a, device=x.device).view(-1, 1, 1)
        x = torch.where(t < ctx - (b - a) + 1 + j, x, -math.inf)
    return x, mag, a, b


def weights_formula(wl, lse, scores, causal, decay):
    want, tol = scores.double().clone(), torch.zeros_like(scores, dtype=torch.float64)
    group = wl.num_q_heads // wl.num_kv_heads
    for s in range(wl.num_seqs):
        ctx = int(wl.context_lens[s])
        if ctx <= 0:
            continue
        x, mag, a, b = logits(wl, s, causal)
        p = torch.exp(x - lse[a:b].double().unsqueeze(-1))
        p = torch.where(lse[a:b].unsqueeze(-1) == -math.inf, 0.0, p)
        rel = (wl.head_dim + 8) * 2.0 ** -24 * mag + 2.0 ** -21 + (2.0 ** -21 * mag if wl.query.dtype == torch.float32 else 0) \
            + 2.0 ** -23 * lse[a:b].double().abs().nan_to_num(0, 0, 0).unsqueeze(-1)
        got = p.view(b - a, wl.num_kv_heads, group, ctx).sum(dim=(0, 2))
        off = (p * (rel + (b - a) * group * 2.0 ** -24)).view(b - a, wl.num_kv_heads, group, ctx).sum(dim=(0, 2))
        old = torch.where(torch.arange(ctx, device=got.device) < ctx - (b - a), scores[s, :, :ctx].double() * decay if decay else 0.0, 0.0)
        want[s, :, :ctx] = old + got
        tol[s, :, :ctx] = off + 2.0 ** -23 * (old.abs() + got) + 1e-37
    return want, tol


def true_lse(wl, causal):
    lse = torch.full((wl.query.shape[0], wl.num_q_heads), -math.inf, device="cuda")
    for s in range(wl.num_seqs):
        if int(wl.context_lens[s]) > 0:
            x, _, a, b = logits(wl, s, causal)
            lse[a:b] = torch.logsumexp(x, -1).float()
    return lse


def accumulate(wl, lse, scores, **kw):
    return ops.kv_cache_accumulate_weights(wl.query, wl.key_cache, wl.k_scale, wl.block_tables, wl.context_lens, lse, scores,
                                           wl.softmax_scale, cu_q_lens=wl.cu_q_lens, max_q_len=wl.max_q_len, **kw)


def check_weights(wl, causal=True, decay=1.0, extra=0):
    lse = true_lse(wl, causal)
    wide = torch.rand(wl.num_seqs, wl.num_kv_heads, wl.block_tables.shape[1] * wl.page_size + extra, device="cuda")
    scores = wide[:, :, :wide.shape[2] - extra]
    for s in range(wl.num_seqs):
        scores[s, :, max(0, int(wl.context_lens[s])):] = math.nan  # neither read nor written
        n = 1 if wl.cu_q_lens is None else int(wl.cu_q_lens[s + 1] - wl.cu_q_lens[s])
        scores[s, :, max(0, int(wl.context_lens[s]) - n):] = math.nan  # nor are the new tokens' read
    if decay == 0:
        scores.fill_(math.nan)
    want, tol = weights_formula(wl, lse, scores.nan_to_num(0.0), causal, decay)
    before = wide.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = accumulate(wl, lse, scores, is_causal=causal, decay=decay, status=status)
    assert got is scores and int(status) == 0
    for s in range(wl.num_seqs):
        n = max(0, int(wl.context_lens[s]))
        err = (got[s, :, :n].double() - want[s, :, :n]).abs()
        assert (err <= tol[s, :, :n]).all(), f"seq {s}: {float(err.max()):.3e}, {float((err / tol[s, :, :n].clamp_min(1e-300)).max()):.2f} of the tolerance"
        assert torch.equal(torch.nan_to_num(got[s, :, n:], 7.0), torch.nan_to_num(before[s, :, n:scores.shape[2]], 7.0))
    if extra:
        assert torch.equal(wide[:, :, -extra:], before[:, :, -extra:])
    return got


@pytest.mark.parametrize("fmt", ["fp8_token", "fp8_head", "fp8_block", "mx8", "bf16", "f16"])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("d", [64, 128])
def test_weights_formats(fmt, page, d):
    dt = torch.float16 if fmt == "f16" else torch.bfloat16
    check_weights(cache("w", lens=[0, 1, 15, 16, 17, 100, 333], hq=8, hkv=2, d=d, page=page, fmt=fmt, q_dtype=dt, seed=d + page), extra=3)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 8), (12, 12), (5, 1), (16, 2), (40, 8), (32, 1), (6, 3)])
@pytest.mark.parametrize("q_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_weights_head_layouts(hq, hkv, q_dtype):
    check_weights(cache("w", lens=[70, 301], hq=hq, hkv=hkv, d=128, page=16, q_dtype=q_dtype, seed=hq))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("decay", [1.0, 0.75, 0.0])
@pytest.mark.parametrize("fmt", ["fp8_token", "mx8", "bf16"])
def test_weights_query_lengths(causal, decay, fmt):
    """Query lengths of one, several, many rows, all of the context, and a single token of context."""
    check_weights(cache("w", lens=[40, 129, 300, 33, 1], q_lens=[1, 4, 37, 33, 1], hq=8, hkv=2, d=128, page=16, fmt=fmt, seed=4), causal, decay)


def test_weights_tiny_and_huge_queries():
    """bf16 queries far outside fp16's range, in both directions."""
    for gain in (1e-30, 1e-6, 3e4, 1e8):
        wl = cache("w", lens=[50, 200], hq=8, hkv=2, d=128, page=16, seed=6)
        wl.query = (wl.query.float() * gain).bfloat16()
        wl.softmax_scale = 0.1 / gain
        check_weights(wl)


def test_weights_sequence_without_queries_and_empty_rows():
    wl = cache("w", lens=[40, 60, 30], q_lens=[2, 1, 1], hq=4, hkv=2, d=64, page=16, seed=8)
    wl.cu_q_lens = torch.tensor([0, 2, 2, 4], dtype=torch.int32, device="cuda")  # the second has none, the third two
    wl.max_q_len = 2
    check_weights(wl, decay=0.5)
    lse = torch.full((4, 4), -math.inf, device="cuda")  # rows that saw nothing
    scores = torch.ones(3, 2, 64, device="cuda")
    accumulate(wl, lse, scores)
    assert torch.equal(scores[0, :, :40], torch.cat([torch.ones(2, 38), torch.zeros(2, 2)], 1).cuda())


def test_weights_sum_to_the_number_of_rows():
    """With the decode's own log-sum-exp the weights of a step add up to the heads of the group."""
    wl = cache("w", lens=[700, 90], hq=32, hkv=8, d=128, page=16, seed=11)
    _, lse = ops.run_workload(wl, return_lse=True)
    got = accumulate(wl, lse, torch.zeros(2, 8, wl.block_tables.shape[1] * 16, device="cuda"))
    # the decode rounds neither logits nor their sums below fp32: the sum is 1 within the tolerance of its log-sum-exp, 1e-3
    assert ((got.sum(-1) - 4).abs() < 4e-3).all()


def test_weights_findings():
    wl = cache("w", lens=[50, 60], hq=4, hkv=2, d=64, page=16, seed=12)
    lse = true_lse(wl, True)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    clean = accumulate(wl, lse, torch.zeros(2, 2, 64, device="cuda"), status=status)
    wl.block_tables[1, 2] = 10 ** 6
    got = accumulate(wl, lse, torch.full((2, 2, 64), 5.0, device="cuda"), status=status)
    assert int(status) == L.ST_BAD_BLOCK and (got[1, :, 32:48] == 5).all()
    assert torch.equal(got[0, :, :49] - 5, (clean[0, :, :49] + 5) - 5) or ((got[0, :, :49] - 5 - clean[0, :, :49]).abs() < 1e-6).all()
    wl.block_tables[1, 2] = 0
    wl.context_lens[0] = 65
    status.zero_()
    got = accumulate(wl, lse, torch.zeros(2, 2, 60, device="cuda"), status=status)
    assert int(status) & L.ST_BAD_CTX
    status.zero_()
    wl.context_lens[0] = 50
    wl.cu_q_lens = torch.tensor([0, 5, 2], dtype=torch.int32, device="cuda")
    got = accumulate(wl, lse, torch.ones(2, 2, 64, device="cuda"), status=status)
    assert int(status) == L.ST_BAD_QLEN and (got == 1).all()


# ------------------------------------------------------------------------------------------------ eviction
def select_formula(row, n, budget, sink, recent):
    if n <= budget:
        return list(range(n))
    must = set(range(min(sink, n))) | set(range(n - recent, n))
    rest = [t for t in range(n) if t not in must]
    rest.sort(key=lambda t: (-(row[t] if row[t] == row[t] else -math.inf), row[t] != row[t], t))
    return sorted(must | set(rest[:budget - len(must)]))


def gather(wl, table, h, tokens):
    """The bytes of the listed tokens of one KV head, K, V and scales."""
    t = torch.tensor(tokens, dtype=torch.long, device="cuda")
    blk, off = table[t // wl.page_size].long(), t % wl.page_size
    out = [wl.key_cache[blk, h, :, off], wl.value_cache[blk, h, :, off]]
    if wl.k_scale is not None and wl.k_scale.dim() == 3:
        out += [wl.k_scale[blk, h, off], wl.v_scale[blk, h, off]]
    elif wl.k_scale is not None and wl.k_scale.dim() == 4:
        out += [wl.k_scale[blk, h, :, off], wl.v_scale[blk, h, :, off]]
    return [x.clone() for x in out]


def evict(wl, scores, budget, **kw):
    return ops.kv_cache_evict(scores, wl.key_cache, wl.value_cache, wl.k_scale, wl.v_scale, wl.block_tables, wl.context_lens, budget, **kw)


def same(a, b):
    return a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def check_evict(wl, scores, budget, sink=0, recent=0, in_place=True, scores_in_place=False):
    lens = [max(0, int(n)) for n in wl.context_lens]
    page, pool = wl.page_size, wl.key_cache.shape[0]
    rows = scores.cpu()
    want = [[select_formula(rows[s, h].tolist(), lens[s], budget, sink, recent) for h in range(wl.num_kv_heads)] for s in range(wl.num_seqs)]
    held = [[gather(wl, wl.block_tables[s], h, want[s][h]) for h in range(wl.num_kv_heads)] for s in range(wl.num_seqs)]
    used = set()
    for s, n in enumerate(lens):
        used |= set(wl.block_tables[s, :(n + page - 1) // page].tolist())
    table = wl.block_tables
    if not in_place:
        width = (budget + page - 1) // page
        grown = pool + wl.num_seqs * width
        for name in ("key_cache", "value_cache", "k_scale", "v_scale"):
            t = getattr(wl, name)
            if t is not None and t.dim() > 1:
                setattr(wl, name, torch.cat([t, t[:1].expand(grown - pool, *t.shape[1:])]).contiguous())
        table = (pool + torch.randperm(grown - pool, device="cuda")).to(torch.int32).view(wl.num_seqs, width).contiguous()
    before = [None if t is None else t.clone() for t in (wl.key_cache, wl.value_cache, wl.k_scale, wl.v_scale)]
    given = scores.clone()
    new_scores = scores if scores_in_place else torch.full((wl.num_seqs, wl.num_kv_heads, budget + 5), 77.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept, new_lens = evict(wl, scores, budget, sink=sink, recent=recent, new_block_tables=None if in_place else table, new_scores=new_scores,
                           status=status)
    assert int(status) == 0
    assert new_lens.tolist() == [min(n, budget) for n in lens]
    written = [None if t is None else torch.zeros(t.shape, dtype=torch.bool, device="cuda") for t in before]
    for s in range(wl.num_seqs):
        for h in range(wl.num_kv_heads):
            w = want[s][h]
            assert kept[s, h].tolist() == w + [-1] * (budget - len(w)), (s, h)
            assert torch.equal(new_scores[s, h, :len(w)].nan_to_num(5.0), given[s, h, w].nan_to_num(5.0))
            tail = given[s, h, len(w):] if scores_in_place else torch.full((budget + 5 - len(w),), 77.0, device="cuda")
            assert torch.equal(new_scores[s, h, len(w):].nan_to_num(5.0), tail.nan_to_num(5.0))
            for x, y in zip(gather(wl, table[s], h, list(range(len(w)))), held[s][h]):
                assert same(x, y), (s, h)
            t = torch.arange(len(w), device="cuda")
            blk, off = table[s][t // page].long(), t % page
            for i, m in enumerate(written):
                if m is not None and m.dim() == 4:
                    m[blk, h, :, off] = True
                elif m is not None and m.dim() == 3:
                    m[blk, h, off] = True
    for t, b, m in zip((wl.key_cache, wl.value_cache, wl.k_scale, wl.v_scale), before, written):
        if t is not None:  # nothing else was written
            assert same(torch.where(m, torch.zeros_like(t.view(torch.uint8) if t.element_size() == 1 else t), t.view(torch.uint8) if t.element_size() == 1 else t),
                        torch.where(m, torch.zeros_like(b.view(torch.uint8) if b.element_size() == 1 else b), b.view(torch.uint8) if b.element_size() == 1 else b))
    return kept, new_lens


def random_scores(wl, seed=0, ties=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (wl.num_seqs, wl.num_kv_heads, wl.block_tables.shape[1] * wl.page_size)
    if ties:
        return torch.randint(0, 4, shape, generator=g, device="cuda").float()
    return torch.exp(torch.randn(shape, generator=g, device="cuda") * 2)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("fmt", ["fp8_token", "fp8_head", "mx8", "mx4v", "bf16", "f16", "f32"])
def test_evict_formats(fmt, page, in_place):
    for d in (64, 128):
        wl = cache("e", lens=[0, 1, 40, 41, 100, 333, 17], hq=4, hkv=2, d=d, page=page, fmt=fmt, seed=page + d)
        check_evict(wl, random_scores(wl, d), 40, sink=2, recent=7, in_place=in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (15, 0, 0), (16, 16, 0), (16, 0, 16), (17, 5, 5), (128, 0, 1), (299, 3, 3),
                                                (300, 0, 0), (511, 100, 411)])
def test_evict_budgets(budget, sink, recent, in_place):
    wl = cache("e", lens=[300, 512, 513, 299, 2], hq=3, hkv=3, d=64, page=16, seed=budget)
    check_evict(wl, random_scores(wl, budget, ties=budget % 2 == 1), budget, sink, recent, in_place)


@pytest.mark.parametrize("in_place", [True, False])
def test_evict_special_scores(in_place):
    """Infinities, NaN, zeros of both signs, subnormals, all scores alike; scores compacted in place."""
    wl = cache("e", lens=[200, 200, 200, 64], hq=2, hkv=2, d=64, page=16, seed=21)
    sc = random_scores(wl, 3)
    sc[0, 0, ::7], sc[0, 0, 3::7], sc[0, 0, 5::7] = math.inf, -math.inf, math.nan
    sc[0, 1] = math.nan
    sc[1, 0] = 0.0
    sc[1, 0, 1::2] = -0.0
    sc[1, 1] = torch.arange(sc.shape[2], device="cuda") * 1e-45
    sc[2, 0] = -sc[2, 0]
    sc[:, :, 200:] = math.inf  # behind every length
    check_evict(wl, sc, 50, 2, 9, in_place, scores_in_place=True)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("length,budget", [(5000, 1000), (70001, 9000), (140000, 139990)])
def test_evict_long_rows(length, budget, in_place):
    wl = cache("e", lens=[length, length // 3], hq=1, hkv=1, d=64, page=64, seed=5)
    check_evict(wl, random_scores(wl, 9), budget, 4, 100, in_place, scores_in_place=True)


def test_evict_heavy_ties_in_long_rows():
    wl = cache("e", lens=[30000, 12345], hq=2, hkv=2, d=64, page=16, seed=5)
    check_evict(wl, random_scores(wl, 9, ties=True), 7777, 0, 0)


def test_evict_strided_scores_and_findings():
    wl = cache("e", lens=[100, 90], hq=2, hkv=2, d=64, page=16, seed=31)
    big = random_scores(wl, 1)
    wide = torch.full((2, 2, 300), math.nan, device="cuda")
    wide[:, :, 100:100 + big.shape[2]] = big
    check_evict(wl, wide[:, :, 100:100 + big.shape[2]], 33)
    wl = cache("e", lens=[100, 90], hq=2, hkv=2, d=64, page=16, seed=31)
    sc = torch.arange(112, device="cuda").float().expand(2, 2, 112).contiguous()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    wl.block_tables[0, 6] = -1  # holds tokens 96..99, the best of sequence 0
    v = wl.value_cache.clone()
    kept, _ = evict(wl, sc, 8, status=status)
    assert int(status) == L.ST_BAD_BLOCK and kept[0, 0].tolist() == list(range(92, 100))
    b = int(wl.block_tables[0, 0])
    assert torch.equal(wl.value_cache[b, :, :, :4], v[int(wl.block_tables[0, 5]), :, :, 12:]) and torch.equal(wl.value_cache[b, :, :, 4:], v[b, :, :, 4:])
    status.zero_()
    wl.context_lens[1] = 10 ** 6
    kept, n = evict(wl, sc, 8, status=status)
    assert int(status) & L.ST_BAD_CTX and n.tolist() == [8, 8] and kept[1, 0].tolist() == list(range(104, 112))


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("fmt", ["fp8_token", "mx8", "bf16"])
def test_decode_accumulate_evict_decode(fmt):
    """A serving step as it is used: decode, accumulate, evict, decode on the smaller cache.  The second decode equals
    cross attention to exactly the kept tokens."""
    hq, hkv, d, page = 8, 2, 128, 16
    wl = cache("s", lens=[400, 90, 257], hq=hq, hkv=hkv, d=d, page=page, fmt=fmt, seed=2)
    wl.query = (wl.query.float() * 2).bfloat16()

    def decode():
        if fmt == "bf16":
            return ops.paged_attention_forward(wl.query, wl.key_cache, wl.value_cache, wl.block_tables, wl.context_lens, wl.softmax_scale, return_lse=True)
        return ops.run_workload(wl, return_lse=True)

    _, lse = decode()
    scores = torch.zeros(3, hkv, wl.block_tables.shape[1] * page, device="cuda")
    accumulate(wl, lse, scores)
    vals = [key_values(wl), None]
    keep_k, keep_v = wl.key_cache, wl.k_scale
    wl.key_cache, wl.k_scale = wl.value_cache, wl.v_scale
    vals[1] = key_values(wl)
    wl.key_cache, wl.k_scale = keep_k, keep_v
    kept, new_lens = evict(wl, scores, 128, sink=4, recent=16, new_scores=scores)
    k = torch.zeros(3, hkv, 128, d, device="cuda")
    v = torch.zeros_like(k)
    for s in range(3):
        for h in range(hkv):
            t = kept[s, h][kept[s, h] >= 0].long()
            blk = wl.block_tables[s][t // page].long()
            # pages already hold the kept tokens: the values come from the copies made before
            k[s, h, :len(t)], v[s, h, :len(t)] = vals[0][blk, h, :, t % page].float(), vals[1][blk, h, :, t % page].float()
    wl.context_lens = new_lens
    out, lse2 = decode()
    want, want_lse = ops.cross_attention_forward(wl.query.float().unsqueeze(2), k, v, new_lens, wl.softmax_scale, return_lse=True)
    assert (out.float() - want[:, :, 0]).abs().max() < 2e-2 and (lse2 - want_lse[:, :, 0]).abs().max() < 2e-3
    accumulate(wl, lse2, scores)  # the next step adds to the compacted scores


def test_graph_side_stream_and_extension():
    import sys
    import cuda_b200.compat
    sys.path.insert(0, cuda_b200.compat.PATH)
    try:
        import fused_online_softmax_cuda as ext
    finally:
        sys.path.remove(cuda_b200.compat.PATH)
    def fresh():
        return cache("g", lens=[300, 64, 129], hq=8, hkv=2, d=64, page=16, seed=41)
    wl = fresh()
    lse = true_lse(wl, True)
    base = torch.rand(3, 2, wl.block_tables.shape[1] * 16, device="cuda")
    want = accumulate(wl, lse, base.clone())
    kept, lens = evict(wl, want, 100, sink=1, recent=3)
    w2 = fresh()
    got = ext.kv_cache_accumulate_weights(w2.query, w2.key_cache, w2.k_scale, w2.block_tables, w2.context_lens, lse, base.clone(), w2.softmax_scale)
    k2, l2 = ext.kv_cache_evict(got, w2.key_cache, w2.value_cache, w2.k_scale, w2.v_scale, w2.block_tables, w2.context_lens, 100, sink=1, recent=3)
    assert torch.equal(got, want) and torch.equal(kept, k2) and torch.equal(lens, l2) and torch.equal(w2.key_cache, wl.key_cache)
    w3 = fresh()
    sc = base.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        accumulate(w3, lse, sc)
        k3, l3 = evict(w3, sc, 100, sink=1, recent=3)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(k3, kept) and torch.equal(l3, lens) and same(w3.value_cache, wl.value_cache) and same(w3.k_scale, wl.k_scale)  # unused slots hold NaN
    w4 = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s4 = accumulate(w4, lse, base.clone())
        k4, _ = evict(w4, s4, 100, sink=1, recent=3)
    torch.cuda.synchronize()
    assert torch.equal(s4, want) and torch.equal(k4, kept) and torch.equal(w4.value_cache, wl.value_cache)
