"""Cross attention to an encoder's states against the formula in 64 bits.

Tolerances.  16-bit types: the output is rounded once (half a step, eps / 2 relative) and the weights are rounded to the
same type before the second product, eps / 2 relative to each weight, so relative to the sum of |weight * value| over a
row; sums are in 32 bits (2^-24 per addition, a tenth of that) and the exponential is good to 1e-4.  Hence
|error| <= (eps / 2) |out| + (eps / 2 + 1.5e-4) sum_t p_t |v_t|.  fp32: logits of magnitude <= 40 carry a relative error of
(D + 2) 2^-24, which the exponential turns into an absolute error of the weight's logarithm: (D + 2) 2^-24 * sum|q k| scale,
bounded here by measuring sum|q k| scale itself; sums over n states add at most n 2^-24 relative, on
sum_t p_t |v_t|."""
import math

import pytest
import torch

from cuda_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def formula(q, k, v, lens, scale):
    """out, lse, sum p |v| and the largest sum |q k| scale, all in 64 bits."""
    b, hq, sq, d = q.shape
    group = hq // k.shape[1]
    out = torch.zeros(b, hq, sq, d, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full((b, hq, sq), -math.inf, dtype=torch.float64, device=q.device)
    big = 0.0
    for i in range(b):
        n = k.shape[2] if lens is None else max(0, min(int(lens[i]), k.shape[2]))
        if n == 0:
            continue
        kk = k[i, :, :n].double().repeat_interleave(group, 0)
        vv = v[i, :, :n].double().repeat_interleave(group, 0)
        s = q[i].double() @ kk.transpose(1, 2) * scale
        big = max(big, float((q[i].double().abs() @ kk.abs().transpose(1, 2)).max()) * scale)
        lse[i] = torch.logsumexp(s, -1)
        p = torch.softmax(s, -1)
        out[i], mag[i] = p @ vv, p @ vv.abs()
    return out, lse, mag, big


def check(got, lse, want, want_lse, mag, big, dtype, d, n):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    logit = (d + 4) * 2.0 ** -24 * max(big, 1.0)
    if dtype == torch.float32:
        tol = mag * (2 * logit + (n + 8) * 2.0 ** -24) + 1e-30
    else:
        half = torch.finfo(dtype).eps / 2
        tol = half * want.abs() + (half + 1.5e-4 + 2 * logit + n * 2.0 ** -25) * mag + (2.0 ** -24 if dtype == torch.float16 else 0)
    assert (err <= tol).all(), f"error {float(err.max()):.3e}, {float((err / tol.clamp_min(1e-300)).max()):.2f} of the tolerance"
    if lse is not None:
        fine = torch.isfinite(want_lse)
        assert torch.equal(fine, torch.isfinite(lse)) and (lse[~fine] == -math.inf).all()
        # the sum behind the log is of unrounded weights: relative error as above, absolute after the log
        tol = logit + (n + 8) * 2.0 ** -24 + want_lse.abs() * 2.0 ** -22 + (0 if dtype == torch.float32 else 1.5e-4)
        assert ((lse.double() - want_lse).abs() <= tol)[fine].all(), float((lse.double() - want_lse)[fine].abs().max())


def make(b, hq, hkv, sq, skv, d, dtype, layout="bhsd", seed=0, gain=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(h, n):
        x = torch.randn((b, h, n, d) if layout == "bhsd" else (b, n, h, d), generator=g, device="cuda")
        return x if layout == "bhsd" else x.transpose(1, 2)
    return (t(hq, sq) * gain).to(dtype), t(hkv, skv).to(dtype), t(hkv, skv).to(dtype)


SHAPES = [  # b, hq, hkv, sq, skv, d
    (1, 1, 1, 1, 1, 64), (2, 4, 4, 1, 17, 64), (3, 8, 2, 1, 130, 128), (2, 8, 8, 3, 64, 128), (1, 16, 2, 2, 1000, 128),
    (2, 5, 1, 7, 65, 64), (2, 12, 4, 33, 129, 128), (1, 8, 8, 128, 128, 64), (2, 4, 2, 200, 77, 128), (1, 7, 7, 129, 640, 64),
    (1, 16, 1, 40, 300, 128), (2, 32, 8, 1, 2111, 128), (1, 8, 1, 65, 511, 64), (1, 24, 2, 19, 257, 128), (9, 2, 1, 16, 63, 64),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(shape, dtype):
    b, hq, hkv, sq, skv, d = shape
    q, k, v = make(*shape, DTYPES[dtype], seed=sum(shape))
    scale = 1 / math.sqrt(d)
    out, lse = ops.cross_attention_forward(q, k, v, return_lse=True)
    check(out, lse, *formula(q, k, v, None, scale), q.dtype, d, skv)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("sq", [1, 5, 70, 300])
@pytest.mark.parametrize("d", [64, 128])
def test_lengths_with_nan_behind_them(sq, d, dtype):
    """Lengths of zero, one, tile edges and beyond the buffer; NaN and infinities behind every length."""
    skv = 321
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 320, 321, 400, -3]
    q, k, v = make(len(lens), 4, 2, sq, skv, d, DTYPES[dtype], seed=sq + d)
    kl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = formula(q, k, v, lens, 1 / math.sqrt(d))
    for i, n in enumerate(lens):
        n = max(0, min(n, skv))
        k[i, :, n:], v[i, :, n:] = math.nan, math.nan
        v[i, :, n:n + 1] = math.inf
    out, lse = ops.cross_attention_forward(q, k, v, kl, return_lse=True)
    check(out, lse, *want, q.dtype, d, skv)
    assert (out[0] == 0).all() and (out[-1] == 0).all() and (lse[0] == -math.inf).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("sq", [1, 90])
def test_strides(sq, dtype):
    """The projections' own layout, a slice of a wider buffer, states shared by all batch rows and heads, a misaligned view."""
    dt, d, scale = DTYPES[dtype], 128, 0.07
    q, k, v = make(3, 8, 2, sq, 200, d, dt, layout="bshd", seed=3)
    out = ops.cross_attention_forward(q, k, v, softmax_scale=scale)
    assert out.stride() == q.stride()
    want = formula(q, k, v, None, scale)
    check(out, None, *want, dt, d, 200)
    wide = torch.randn(3, 2, 400, 2 * d, device="cuda").to(dt)
    ks, vs = wide[:, :, 100:300, :d], wide[:, :, 50:250, d:]
    check(ops.cross_attention_forward(q, ks, vs, softmax_scale=scale), None, *formula(q, ks, vs, None, scale), dt, d, 200)
    ke, ve = k[:1].expand(3, -1, -1, -1), v[:1, :1].expand(3, 2, -1, -1)
    check(ops.cross_attention_forward(q, ke, ve, softmax_scale=scale), None, *formula(q, ke, ve, None, scale), dt, d, 200)
    qe = q[:1].expand(3, -1, -1, -1)
    check(ops.cross_attention_forward(qe, k, v, softmax_scale=scale), None, *formula(qe, k, v, None, scale), dt, d, 200)
    odd = torch.randn(3 * 2 * 200 * d + 1, device="cuda").to(dt)[1:].view(3, 2, 200, d)
    check(ops.cross_attention_forward(q, odd, v, softmax_scale=scale), None, *formula(q, odd, v, None, scale), dt, d, 200)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("sq", [1, 100])
def test_large_logits_and_constant_rows(sq, dtype):
    """One state far above the others (weight exactly one), equal logits (the mean), logits far below zero."""
    dt, d = DTYPES[dtype], 64
    q = torch.ones(1, 2, sq, d, device="cuda").to(dt)
    k = torch.zeros(1, 2, 150, d, device="cuda").to(dt)
    v = torch.randn(1, 2, 150, d, device="cuda").to(dt)
    k[0, 0, 97] = 30.0
    k[0, 1] = -30.0
    out, lse = ops.cross_attention_forward(q, k, v, softmax_scale=1.0, return_lse=True)
    assert torch.equal(out[0, 0], v[0, 0, 97].expand(sq, d))
    want = formula(q, k, v, None, 1.0)
    check(out, lse, *want, dt, d, 150)


def test_repeats_are_bit_identical_and_independent_of_the_batch():
    q, k, v = make(4, 8, 2, 1, 1777, 128, torch.bfloat16)
    lens = torch.tensor([1777, 900, 64, 1300], dtype=torch.int32, device="cuda")
    a = ops.cross_attention_forward(q, k, v, lens)
    assert torch.equal(a, ops.cross_attention_forward(q, k, v, lens))


def test_empty_sizes():
    for b, sq, skv in ((0, 3, 5), (2, 0, 5), (2, 3, 0)):
        q = torch.randn(b, 4, sq, 64, device="cuda").bfloat16()
        k = torch.randn(b, 2, skv, 64, device="cuda").bfloat16()
        out, lse = ops.cross_attention_forward(q, k, k, return_lse=True)
        assert out.shape == q.shape and (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("sq", [1, 130])
def test_side_stream_and_graph(sq):
    """A call on a side stream, and a captured call replayed on new inputs while eager calls run."""
    q, k, v = make(2, 8, 2, sq, 600, 128, torch.bfloat16)
    lens = torch.tensor([600, 77], dtype=torch.int32, device="cuda")
    want = ops.cross_attention_forward(q, k, v, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.cross_attention_forward(q, k, v, lens)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.cross_attention_forward(q, k, v, lens)
    q2, k2, v2 = make(2, 8, 2, sq, 600, 128, torch.bfloat16, seed=9)
    q.copy_(q2), k.copy_(k2), v.copy_(v2)
    lens.copy_(torch.tensor([0, 599], dtype=torch.int32))
    graph.replay()
    eager = ops.cross_attention_forward(q2, k2, v2, lens)
    torch.cuda.synchronize()
    assert torch.equal(out, eager)


def test_extension_gives_the_same_bits():
    import sys
    import cuda_b200.compat
    sys.path.insert(0, cuda_b200.compat.PATH)
    try:
        import fused_online_softmax_cuda as ext
    finally:
        sys.path.remove(cuda_b200.compat.PATH)
    for sq in (1, 130):
        q, k, v = make(2, 8, 2, sq, 300, 64, torch.float16, layout="bshd")
        lens = torch.tensor([211, 300], dtype=torch.int32, device="cuda")
        a, la = ops.cross_attention_forward(q, k, v, lens, 0.1, return_lse=True)
        b, lb = ext.cross_attention_forward(q, k, v, lens, 0.1, return_lse=True)
        assert torch.equal(a, b) and torch.equal(la, lb) and a.stride() == b.stride()


def test_no_wait_ran_out():
    import ctypes
    from cuda_b200 import _lib as L
    n = ctypes.c_uint32(7)
    assert L.load().cuda_llm_cross_attention_wait_timeouts(ctypes.byref(n)) == L.OK and n.value == 0
