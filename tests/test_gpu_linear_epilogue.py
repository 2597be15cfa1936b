"""The products with bias, activation and residual in their epilogue (gemm_bias_act,
w8a8_block_int8_matmul_bias_act, w8a8_block_fp8_matmul_bias_act) against their definition in 64
bits.

The shape sweeps use whole numbers and power-of-two scales, for which every product, partial sum
and scaled sum is exact in fp32 whatever the order, so the kernel's output must EQUAL the exact
value rounded once to the output type. The gated activations and real-valued inputs are held to
bounds written beside them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import tileops_b200 as tob
from tileops_b200 import _epilogue, _lib

pytestmark = pytest.mark.gpu

F64 = torch.float64
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def act64(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * (1 + torch.tanh((2 / np.pi) ** 0.5 * (v + 0.044715 * v ** 3)))
    return v


def ints(gen, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=gen, dtype=torch.int64)


def exact_dense(a, b, bias, act, res):
    v = a.to(F64) @ b.to(F64)
    if bias is not None:
        v = v + bias.to(F64)
    v = act64(v, act)
    return v if res is None else v + res.to(F64)


# One token to several tiles; sizes below, at and past a tile; nothing divisible by anything.
DENSE_SHAPES = [
    (1, 1, 1), (1, 64, 64), (1, 4096, 256), (2, 8, 8), (3, 5, 7), (15, 130, 65), (16, 128, 64),
    (17, 136, 72), (31, 200, 33), (33, 1000, 1000), (64, 192, 512), (65, 264, 264),
    (100, 257, 129), (127, 513, 640), (128, 384, 64), (129, 129, 129), (200, 512, 1024),
    (255, 1024, 512), (256, 2560, 256), (257, 72, 2048), (300, 776, 320), (513, 1544, 200),
]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", DENSE_SHAPES)
def test_dense_exact(cuda, dt, m, n, k):
    gen = torch.Generator().manual_seed(m * 7 + n * 3 + k)
    a = ints(gen, -3, 3, m, k).to(dt).to(cuda)
    b = ints(gen, -2, 2, k, n).to(dt).to(cuda)
    bias = ints(gen, -8, 8, n).to(dt).to(cuda)
    res = ints(gen, -8, 8, m, n).to(dt).to(cuda)
    for kw in ({}, {"bias": bias}, {"residual": res}, {"bias": bias, "act": "relu", "residual": res}):
        y = tob.gemm_bias_act(a, b, **kw)
        assert y.shape == (m, n) and y.dtype == dt
        want = exact_dense(a, b, kw.get("bias"), kw.get("act"), kw.get("residual")).to(dt)
        assert torch.equal(y, want), kw.keys()


def w8a8_exact(a, b, a_s, b_s, bn, bk, bias, act, res):
    m, k = a.shape
    n = b.shape[0]
    ka = torch.arange(k, device=a.device) // bk
    nb = torch.arange(n, device=a.device) // bn
    af = a.to(F64) * a_s.to(F64)[:, ka]
    bf = b.to(F64) * b_s.to(F64)[nb][:, ka]
    return exact_dense(af, bf.t(), bias, act, res)


W8A8_SHAPES = [
    (1, 1, 1), (1, 128, 128), (1, 1000, 512), (5, 24, 48), (16, 256, 1024), (17, 144, 160),
    (33, 130, 257), (64, 512, 384), (65, 320, 2048), (100, 1003, 515), (128, 128, 128),
    (129, 272, 272), (200, 1024, 640), (256, 2560, 512), (257, 80, 1024), (300, 333, 1111),
    (600, 1288, 256),
]


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("scales", ["channel", "tensor", "block128", "block256", "wide_n", "odd_n",
                                    "bk64"])
@pytest.mark.parametrize("m,n,k", W8A8_SHAPES)
def test_w8a8_exact(cuda, codes, scales, m, n, k):
    gen = torch.Generator().manual_seed(m * 7 + n * 3 + k)
    bn, bk = {"channel": (1, k), "tensor": (n, k), "block128": (128, 128), "block256": (256, 256),
              "wide_n": (n, 128), "odd_n": (48, 128), "bk64": (64, 64)}[scales]
    hi = 127 if codes == "int8" else 8
    cast = torch.int8 if codes == "int8" else torch.float8_e4m3fn
    hi_b = 3 if codes == "int8" else 8
    a = ints(gen, -hi, hi, m, k).float().to(cast).to(cuda)
    b = ints(gen, -hi_b, hi_b, n, k).float().to(cast).to(cuda)
    kt, nt = -(-k // bk), -(-n // bn)
    a_s = torch.exp2(ints(gen, -1, 0, m, kt).float()).to(cuda)
    b_s = torch.exp2(ints(gen, -1, 0, nt, kt).float()).to(cuda)
    op = (tob.w8a8_block_int8_matmul_bias_act if codes == "int8"
          else tob.w8a8_block_fp8_matmul_bias_act)
    for i, dt in enumerate((torch.bfloat16, torch.float16, torch.float32)):
        bias = ints(gen, -8, 8, n).to(dt).to(cuda)
        res = ints(gen, -8, 8, m, n).to(dt).to(cuda)
        kw = [{"act": "relu", "bias": bias, "residual": res}, {"bias": bias}, {"residual": res}][i]
        y = op(a, b, a_s, b_s, [bn, bk], output_dtype=dt, **kw)
        assert y.shape == (m, n) and y.dtype == dt
        want = w8a8_exact(a, b, a_s, b_s, bn, bk, kw.get("bias"), kw.get("act"),
                          kw.get("residual")).to(dt)
        assert torch.equal(y, want), (dt, list(kw))


@pytest.mark.parametrize("m,n,k", [(65, 9600, 96), (80, 20000, 64), (128, 7200, 160),
                                   (145, 2240, 1300), (162, 3520, 1280), (129, 190, 2100)])
def test_tile_choices(cuda, m, n, k):
    """Half-empty pairs of wide outputs, and few tiles of some more than 64 tokens with K split."""
    test_dense_exact(cuda, torch.bfloat16, m, n, k)
    for codes in ("int8", "e4m3"):
        for scales in ("channel", "block128", "odd_n"):
            test_w8a8_exact(cuda, codes, scales, m, n, k)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (40, 333, 777), (300, 1024, 512)])
def test_dense_activations(cuda, act, dt, m, n, k):
    """Real values. |acc error| <= k 2^-23 sum|ab| (one rounding, or truncation, of at most 2^-23
    per addition); silu and gelu have slopes within 1.13; sigmoid's exponential and division are
    within 4e-6; one rounding of the result."""
    gen = torch.Generator().manual_seed(m + n + k)
    a = torch.randn(m, k, generator=gen).to(dt).to(cuda)
    b = (torch.randn(k, n, generator=gen) * 2 * k ** -0.5).to(dt).to(cuda)
    bias = torch.randn(n, generator=gen).to(dt).to(cuda)
    res = torch.randn(m, n, generator=gen).to(dt).to(cuda)
    y = tob.gemm_bias_act(a, b, bias, act=act, residual=res).to(F64)
    want = exact_dense(a, b, bias, act, res)
    acc = k * 2.0 ** -23 * (a.to(F64).abs() @ b.to(F64).abs())
    pre = exact_dense(a, b, bias, None, None)
    tol = HALF_STEP[dt] * want.abs() * 1.01 + 1.13 * acc + 4e-6 * (pre.abs() + res.to(F64).abs() + 1)
    assert bool(((y - want).abs() <= tol).all())


@pytest.mark.parametrize("scales", ["channel", "block"])
@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("m,n,k", [(1, 640, 2048), (50, 200, 500), (384, 768, 1024)])
def test_w8a8_activations(cuda, scales, codes, m, n, k):
    """As above; the scales add at most three roundings per term."""
    gen = torch.Generator().manual_seed(m + n + k)
    cast = torch.int8 if codes == "int8" else torch.float8_e4m3fn
    a = (torch.randn(m, k, generator=gen) * 40).clamp(-127, 127).round().to(cast).to(cuda)
    b = (torch.randn(n, k, generator=gen) * 40).clamp(-127, 127).round().to(cast).to(cuda)
    bn, bk = (1, k) if scales == "channel" else (128, 128)
    a_s = ((0.5 + torch.rand(m, -(-k // bk), generator=gen)) / 40).to(cuda)
    b_s = ((0.5 + torch.rand(-(-n // bn), -(-k // bk), generator=gen)) / (40 * k ** 0.5)).to(cuda)
    res = torch.randn(m, n, generator=gen).bfloat16().to(cuda)
    bias = torch.randn(n, generator=gen).bfloat16().to(cuda)
    op = (tob.w8a8_block_int8_matmul_bias_act if codes == "int8"
          else tob.w8a8_block_fp8_matmul_bias_act)
    for act in ("silu", "gelu"):
        y = op(a, b, a_s, b_s, [bn, bk], bias, act=act, residual=res,
               output_dtype=torch.bfloat16).to(F64)
        want = w8a8_exact(a, b, a_s, b_s, bn, bk, bias, act, res)
        pre = w8a8_exact(a, b, a_s, b_s, bn, bk, bias, None, None)
        mass = w8a8_exact(a.float().abs(), b.float().abs(), a_s, b_s, bn, bk, None, None, None)
        tol = 2.0 ** -8 * want.abs() * 1.01 + 1.13 * (k + 3) * 2.0 ** -23 * mass \
            + 4e-6 * (pre.abs() + res.to(F64).abs() + 1)
        assert bool(((y - want).abs() <= tol).all()), act


@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(3, 96, 64), (130, 264, 136), (300, 640, 192)])
def test_layouts_and_alignment(cuda, dt, m, n, k):
    """Strided rows of A, residual and out; operands one element off their alignment; transposed
    residual and out; nothing outside the output's rows is touched."""
    gen = torch.Generator().manual_seed(m + n)
    a0 = ints(gen, -3, 3, m, k).to(dt).to(cuda)
    b0 = ints(gen, -2, 2, k, n).to(dt).to(cuda)
    r0 = ints(gen, -8, 8, m, n).to(dt).to(cuda)
    bias0 = ints(gen, -8, 8, n).to(dt).to(cuda)
    want = exact_dense(a0, b0, bias0, None, r0).to(dt)

    def off(t, by):  # the same values at a storage offset
        flat = torch.zeros(t.numel() + by, dtype=t.dtype, device=cuda)
        flat[by:] = t.reshape(-1)
        return flat[by:].view(t.shape)

    for by in (1, 2, 4):
        y = tob.gemm_bias_act(off(a0, by), off(b0, by), off(bias0, by), residual=off(r0, by))
        assert torch.equal(y, want), by
    for pad in (1, 8):
        wide_a = torch.zeros(m, k + pad, dtype=dt, device=cuda)
        wide_a[:, :k] = a0
        wide_r = torch.zeros(m, n + pad, dtype=dt, device=cuda)
        wide_r[:, pad:] = r0
        wide_o = torch.full((m, n + 2 * pad), 7, dtype=dt, device=cuda)
        o = wide_o[:, pad:pad + n]
        assert tob.gemm_bias_act(wide_a[:, :k], b0, bias0, residual=wide_r[:, pad:], out=o) is o
        assert torch.equal(o, want)
        assert bool((wide_o[:, :pad] == 7).all()) and bool((wide_o[:, pad + n:] == 7).all())
    ot = torch.empty(n, m, dtype=dt, device=cuda).t()
    rt = r0.t().contiguous().t()
    assert tob.gemm_bias_act(a0, b0.t().contiguous().t(), bias0, residual=rt, out=ot) is ot
    assert torch.equal(ot, want)
    # broadcast residual and bias views
    row = r0[:1].expand(m, n)
    one = bias0[:1].expand(n)
    assert torch.equal(tob.gemm_bias_act(a0, b0, one, residual=row),
                       exact_dense(a0, b0, one, None, row).to(dt))


@pytest.mark.parametrize("by", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("m,n,k", [(2, 130, 96), (70, 256, 128), (260, 520, 160)])
def test_w8a8_byte_alignment(cuda, by, m, n, k):
    gen = torch.Generator().manual_seed(by + m)
    a0 = ints(gen, -127, 127, m, k).to(torch.int8)
    b0 = ints(gen, -3, 3, n, k).to(torch.int8)
    one_m, one_n = torch.ones(m, 1, device=cuda), torch.ones(n, 1, device=cuda)
    want = (a0.to(F64) @ b0.to(F64).t()).float().to(cuda)

    def off(t):
        flat = torch.zeros(t.numel() + by, dtype=t.dtype, device=cuda)
        flat[by:] = t.reshape(-1).to(cuda)
        return flat[by:].view(t.shape)

    y = tob.w8a8_block_int8_matmul_bias_act(off(a0), off(b0), one_m, one_n, [1, k],
                                            output_dtype=torch.float32)
    assert torch.equal(y, want)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 512), (48, 300, 200), (300, 512, 256)])
def test_in_place_residual(cuda, m, n, k):
    gen = torch.Generator().manual_seed(3)
    a = ints(gen, -3, 3, m, k).to(torch.bfloat16).to(cuda)
    b = ints(gen, -2, 2, k, n).to(torch.bfloat16).to(cuda)
    r = ints(gen, -8, 8, m, n).to(torch.bfloat16).to(cuda)
    want = exact_dense(a, b, None, None, r).to(torch.bfloat16)
    assert tob.gemm_bias_act(a, b, residual=r, out=r) is r
    assert torch.equal(r, want)


def test_leading_dimensions_and_empty(cuda):
    a = torch.ones(2, 3, 32, dtype=torch.int8, device=cuda)
    b = torch.ones(5, 32, dtype=torch.int8, device=cuda)
    a_s, b_s = torch.ones(2, 3, 1, device=cuda), torch.ones(5, 1, device=cuda)
    res = torch.full((2, 3, 5), 1.5, device=cuda, dtype=torch.float16)
    y = tob.w8a8_block_int8_matmul_bias_act(a, b, a_s, b_s, [1, 32], residual=res)
    assert y.shape == (2, 3, 5) and bool((y == 33.5).all())
    e = torch.empty(0, 8, device=cuda)
    assert tob.gemm_bias_act(e, torch.ones(8, 4, device=cuda)).shape == (0, 4)
    assert tob.gemm_bias_act(torch.ones(4, 8, device=cuda), torch.empty(8, 0, device=cuda)).shape \
        == (4, 0)
    # K = 0: the epilogue of zeros
    z = torch.empty(3, 0, device=cuda, dtype=torch.float16)
    bias = torch.tensor([-1.0, 2.0], device=cuda, dtype=torch.float16)
    y = tob.gemm_bias_act(z, torch.empty(0, 2, device=cuda, dtype=torch.float16), bias, act="relu",
                          residual=torch.ones(3, 2, device=cuda, dtype=torch.float16))
    assert y.tolist() == [[1.0, 3.0]] * 3


@pytest.mark.parametrize("m", [1, 20, 300])
def test_non_finite_values_stay_in_their_row_and_column(cuda, m):
    """A NaN or infinity in one row of A or one column of B marks that row / column alone, and
    silu and gelu take +inf to inf, NaN to NaN."""
    n, k = 264, 200
    a = torch.ones(m, k, dtype=torch.bfloat16, device=cuda)
    b = torch.ones(k, n, dtype=torch.bfloat16, device=cuda)
    b[7, 5] = float("nan")
    b[k - 1, n - 1] = float("inf")
    a[m - 1, 3] = 2.0
    for act in (None, "relu", "silu", "gelu"):
        y = tob.gemm_bias_act(a, b, act=act)
        assert bool(torch.isnan(y[:, 5]).all()) and bool(torch.isposinf(y[:, n - 1]).all())
        keep = [j for j in range(n) if j not in (5, n - 1)]
        assert bool(torch.isfinite(y[:, keep]).all())


def test_side_stream_and_graph(cuda):
    """The call runs on the current stream, and a captured call replays on new inputs."""
    gen = torch.Generator().manual_seed(11)
    a = torch.empty(24, 256, dtype=torch.bfloat16, device=cuda)
    b = ints(gen, -2, 2, 256, 300).to(torch.bfloat16).to(cuda)
    out = torch.empty(24, 300, dtype=torch.bfloat16, device=cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.fill_(1)
        tob.gemm_bias_act(a, b, act="relu", out=out)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tob.gemm_bias_act(a, b, act="relu", out=out)
    for seed in (1, 2):
        src = ints(torch.Generator().manual_seed(seed), -3, 3, 24, 256).to(torch.bfloat16).to(cuda)
        a.copy_(src)
        g.replay()
        assert torch.equal(out, exact_dense(src, b, None, "relu", None).to(torch.bfloat16))


def test_two_streams_at_once(cuda):
    """Calls in flight on two streams share nothing."""
    gen = torch.Generator().manual_seed(12)
    a = [ints(gen, -3, 3, 16, 4096).to(torch.float16).to(cuda) for _ in range(2)]
    b = [ints(gen, -2, 2, 4096, 1024).to(torch.float16).to(cuda) for _ in range(2)]
    want = [exact_dense(a[i], b[i], None, None, None).half() for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(tob.gemm_bias_act(a[i], b[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in outs[i]:
            assert torch.equal(y, want[i])


def test_repeatable(cuda):
    """Equal inputs give equal bits, whatever the split of K."""
    gen = torch.Generator().manual_seed(13)
    for m, n, k in ((1, 4096, 4096), (100, 512, 8192), (600, 512, 1024)):
        a = torch.randn(m, k, generator=gen).bfloat16().to(cuda)
        b = torch.randn(k, n, generator=gen).bfloat16().to(cuda)
        first = tob.gemm_bias_act(a, b, act="gelu")
        assert all(torch.equal(tob.gemm_bias_act(a, b, act="gelu"), first) for _ in range(5))


def test_launch_overlap(cuda):
    """With launch overlap on, a chain of products equals the chain with it off."""
    gen = torch.Generator().manual_seed(14)
    ws = [(torch.randn(512, 512, generator=gen) / 22).half().to(cuda) for _ in range(6)]
    x0 = torch.randn(4, 512, generator=gen).half().to(cuda)

    def chain():
        x = x0
        for w in ws:
            x = tob.gemm_bias_act(x, w, act="silu", residual=x)
        return x

    want = chain()
    prev = tob.set_launch_overlap(True)
    try:
        got = [chain() for _ in range(4)]
    finally:
        tob.set_launch_overlap(prev)
    assert all(torch.equal(y, want) for y in got)


def test_offsets_past_32_bits(cuda):
    """An output of more than 2^31 elements, with its residual."""
    m, n, k = 66000, 33000, 16
    a = torch.ones(m, k, dtype=torch.bfloat16, device=cuda)
    a *= (torch.arange(m, device=cuda) % 7 - 3).to(torch.bfloat16)[:, None]
    b = torch.ones(k, n, dtype=torch.bfloat16, device=cuda)
    b *= (torch.arange(n, device=cuda) % 5 - 2).to(torch.bfloat16)
    res = (torch.arange(n, device=cuda) % 3).to(torch.bfloat16).expand(m, n).contiguous()
    y = tob.gemm_bias_act(a, b, residual=res, out=res)
    for rows in (slice(0, 40), slice(65040, 65110), slice(m - 40, m)):
        want = (k * a[rows, :1].float() * b[:1].float()
                + (torch.arange(n, device=cuda) % 3).float()).bfloat16()
        assert torch.equal(y[rows], want)


# Many tokens, nothing aligned: operands copied to aligned rows, outputs written row by row.
RAGGED_SHAPES = [(129, 4097, 65), (200, 3001, 1000), (300, 9001, 777), (777, 2049, 1531),
                 (513, 5003, 72), (1025, 1030, 33)]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", RAGGED_SHAPES)
def test_dense_exact_many_tokens_ragged(cuda, dt, m, n, k):
    gen = torch.Generator(device=cuda).manual_seed(m + n + k)

    def ri(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=gen, device=cuda).to(dt)

    a, b, bias, res = ri(-3, 3, m, k), ri(-2, 2, k, n), ri(-8, 8, n), ri(-8, 8, m, n)
    want = exact_dense(a, b, bias, "relu", res).to(dt)
    assert torch.equal(tob.gemm_bias_act(a, b, bias, act="relu", residual=res), want)
    out = res.clone()
    assert tob.gemm_bias_act(a, b, bias, act="relu", residual=out, out=out) is out
    assert torch.equal(out, want)
    # only A, only B off alignment; an aligned product into unaligned rows
    flat = torch.zeros(m * k + 1, dtype=dt, device=cuda)
    flat[1:] = a.reshape(-1)
    assert torch.equal(tob.gemm_bias_act(flat[1:].view(m, k), b), exact_dense(a, b, None, None, None).to(dt))
    k8, n8 = k // 8 * 8, n // 8 * 8
    wide = torch.full((m, n8 + 3), 7, dtype=dt, device=cuda)
    tob.gemm_bias_act(a[:, :k8].contiguous(), b[:k8, :n8].contiguous(), out=wide[:, 1:n8 + 1])
    assert torch.equal(wide[:, 1:n8 + 1], exact_dense(a[:, :k8], b[:k8, :n8], None, None, None).to(dt))
    assert bool((wide[:, 0] == 7).all()) and bool((wide[:, n8 + 1:] == 7).all())


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("scales", ["channel", "block128"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", RAGGED_SHAPES)
def test_w8a8_exact_many_tokens_ragged(cuda, codes, scales, dt, m, n, k):
    gen = torch.Generator(device=cuda).manual_seed(m + n + k)
    bn, bk = (1, k) if scales == "channel" else (128, 128)
    hi, hi_b = (127, 3) if codes == "int8" else (8, 8)
    cast = torch.int8 if codes == "int8" else torch.float8_e4m3fn

    def ri(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=gen, device=cuda).float()

    a, b = ri(-hi, hi, m, k).to(cast), ri(-hi_b, hi_b, n, k).to(cast)
    a_s, b_s = torch.exp2(ri(-1, 0, m, -(-k // bk))), torch.exp2(ri(-1, 0, -(-n // bn), -(-k // bk)))
    bias, res = ri(-8, 8, n).to(dt), ri(-8, 8, m, n).to(dt)
    op = (tob.w8a8_block_int8_matmul_bias_act if codes == "int8"
          else tob.w8a8_block_fp8_matmul_bias_act)
    y = op(a, b, a_s, b_s, [bn, bk], bias, act="relu", residual=res, output_dtype=dt)
    assert torch.equal(y, w8a8_exact(a, b, a_s, b_s, bn, bk, bias, "relu", res).to(dt))


def test_workspace_of_the_c_entries(cuda):
    """Scratch for aligned copies: asked for exactly when a row is not 16-byte aligned, refused when
    short, unaligned or missing, with nothing launched."""
    m, n, k = 30, 1001, 333
    a, b = torch.ones(m, k, device=cuda).half(), torch.ones(k, n, device=cuda).half()
    c = torch.full((m, n), 7.0, device=cuda, dtype=torch.float16)
    lib, f16 = _lib.load(), _lib.DTYPE_CODES[torch.float16]
    need = lib.to_gemm_bias_act_workspace_size(a.data_ptr(), k, b.data_ptr(), f16, m, n, k)
    assert need == m * 768 + k * 2048  # rows of 666 and 2002 bytes, padded to 128
    assert need == (_epilogue.padded(m, 2 * k, a.data_ptr(), 2 * k)
                    + _epilogue.padded(k, 2 * n, b.data_ptr(), 2 * n))
    assert lib.to_gemm_bias_act_workspace_size(1024, 336, 1024, f16, m, 1000, 333) == 0
    assert lib.to_w8a8_gemm_bias_act_workspace_size(1024, 1024, m, n, 336, 336) == 0
    assert lib.to_w8a8_gemm_bias_act_workspace_size(1024, 1024, m, n, k, k) == (m + n) * 384
    buf = torch.empty(need + 16, dtype=torch.uint8, device=cuda)

    def call(ws, size):
        return lib.to_gemm_bias_act(a.data_ptr(), k, b.data_ptr(), None, 0, None, n, c.data_ptr(), n,
                                    f16, m, n, k, ws, size, _lib.stream_ptr())

    assert call(None, 0) == _lib.TO_ENOSPACE and call(buf.data_ptr(), need - 1) == _lib.TO_ENOSPACE
    assert call(buf.data_ptr() + 8, need) == _lib.TO_EINVAL
    assert bool((c == 7).all())
    assert call(buf.data_ptr(), need) == _lib.TO_OK
    assert bool((c == k).all())


# Many tokens: several tiles per CTA pair, ragged last tiles, K of one slice, of an odd number of
# slices, of no whole slice; tile widths chosen by the number of tiles.
LARGE_SHAPES = [
    (256, 11008, 512), (257, 9480, 192), (512, 4096, 128), (1000, 6152, 320), (1024, 5120, 136),
    (2048, 2304, 1024), (2500, 4104, 72), (4100, 2048, 64), (300, 28672, 256), (9000, 640, 200),
]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", LARGE_SHAPES)
def test_dense_exact_many_tokens(cuda, dt, m, n, k):
    gen = torch.Generator(device=cuda).manual_seed(m + n + k)

    def ri(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=gen, device=cuda).to(dt)

    a, b, bias, res = ri(-3, 3, m, k), ri(-2, 2, k, n), ri(-8, 8, n), ri(-8, 8, m, n)
    assert torch.equal(tob.gemm_bias_act(a, b), exact_dense(a, b, None, None, None).to(dt))
    want = exact_dense(a, b, bias, "relu", res).to(dt)
    y = tob.gemm_bias_act(a, b, bias, act="relu", residual=res)
    assert torch.equal(y, want)
    wide = torch.full((m, n + 16), 7, dtype=dt, device=cuda)
    wide[:, 8:n + 8] = res
    o = wide[:, 8:n + 8]
    assert tob.gemm_bias_act(a, b, bias, act="relu", residual=o, out=o) is o
    assert torch.equal(o, want)
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, n + 8:] == 7).all())


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("scales", ["channel", "tensor", "block128", "wide_n", "block256"])
@pytest.mark.parametrize("m,n,k", LARGE_SHAPES)
def test_w8a8_exact_many_tokens(cuda, codes, scales, m, n, k):
    gen = torch.Generator(device=cuda).manual_seed(m + n + k)
    k = -(-k // 16) * 16
    bn, bk = {"channel": (1, k), "tensor": (n, k), "block128": (128, 128), "wide_n": (n, 128),
              "block256": (256, 256)}[scales]
    hi = 127 if codes == "int8" else 8
    hi_b = 3 if codes == "int8" else 8
    cast = torch.int8 if codes == "int8" else torch.float8_e4m3fn

    def ri(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=gen, device=cuda).float()

    a, b = ri(-hi, hi, m, k).to(cast), ri(-hi_b, hi_b, n, k).to(cast)
    kt, nt = -(-k // bk), -(-n // bn)
    a_s, b_s = torch.exp2(ri(-1, 0, m, kt)), torch.exp2(ri(-1, 0, nt, kt))
    bias, res = ri(-8, 8, n).bfloat16(), ri(-8, 8, m, n).bfloat16()
    op = (tob.w8a8_block_int8_matmul_bias_act if codes == "int8"
          else tob.w8a8_block_fp8_matmul_bias_act)
    y = op(a, b, a_s, b_s, [bn, bk], bias, act="relu", residual=res, output_dtype=torch.bfloat16)
    want = w8a8_exact(a, b, a_s, b_s, bn, bk, bias, "relu", res).bfloat16()
    assert torch.equal(y, want)
    y = op(a, b, a_s, b_s, [bn, bk], output_dtype=torch.float16)
    assert torch.equal(y, w8a8_exact(a, b, a_s, b_s, bn, bk, None, None, None).half())
