"""add_rms_norm_group_quant against its definition in 64 bits.

Bounds. d = (cols / 32 + 24) 2^-24 covers the fp32 sum of squares (every thread of a row's team of
at least 32 adds at most cols / 32 terms, then ten pairwise steps; half of it reaches rstd) and the
roundings of h, rstd, the two products, the maximum's division and the quotient's division.
A scale is off by at most d relatively. A code stands for a value within half a step of the exact
one: e4m3 2^-4 relatively (2^-10 scale units below its normal range), int8 half a unit, plus what d
moves."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import tileops_b200 as tob

pytestmark = pytest.mark.gpu

F64 = torch.float64
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def definition(x, w, r, g, codes, eps=1e-6, qeps=1e-10):
    h = x.to(F64) if r is None else x.to(F64) + r.to(F64)
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.to(F64)
    qmax = 448.0 if codes == torch.float8_e4m3fn else 127.0
    yg = y.reshape(*y.shape[:-1], y.shape[-1] // g, g)
    s = yg.abs().amax(-1).clamp(min=qeps) / qmax
    return h, y, s


def check(x, w, r, g, codes, got, **kw):
    h, y, s = definition(x, w, r, g, codes, **kw)
    cols = x.shape[-1]
    d = (cols / 32 + 24) * 2.0 ** -24
    q, sc = got[0], got[1]
    assert q.shape == x.shape and q.dtype == codes and sc.shape == s.shape
    assert bool(((sc.to(F64) - s).abs() <= d * s).all())
    sx = sc.to(F64).repeat_interleave(g, -1)
    v = q.to(torch.float32).to(F64) * sx
    tol = 2.0 ** -4 * y.abs() + 2.0 ** -10 * sx if codes == torch.float8_e4m3fn else 0.5 * sx
    # At the top of the range the code is qmax itself whatever d does to the quotient.
    assert bool(((v - y).abs() <= tol * (1 + 1e-9) + 4 * d * y.abs()).all())
    if r is not None:
        assert got[2].dtype == x.dtype
        tol_h = HALF_STEP[x.dtype] * h.abs() * (1 + 1e-6) + 2.0 ** -24 * h.abs() + 2.0 ** -25 * 2.0 ** -14
        assert bool(((got[2].to(F64) - h).abs() <= tol_h).all())


CASES = [
    # rows, cols, group: one row, warps sharing a block, every group form, odd columns, rows longer
    # than the registers of a block (> 32768 columns in 16 bits, > 8192 unaligned)
    (1, 4096, 128), (1, 32, 32), (3, 8, 8), (5, 256, 64), (7, 1024, 1024), (9, 384, 96),
    (2, 5120, 5120), (33, 11008, 11008), (4, 1001, 1001), (6, 1001, 7), (5, 999, 333), (17, 36, 4),
    (1, 1, 1), (300, 512, 128), (2, 40960, 128), (2, 40960, 40960), (3, 40960, 5120), (2, 9999, 9999),
    (2, 9999, 99), (13, 768, 256), (4, 2048, 512), (1000, 128, 16), (3, 16384, 128), (2, 65, 13),
]


@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols,g", CASES)
def test_definition(cuda, codes, dt, rows, cols, g):
    gen = torch.Generator().manual_seed(rows * 31 + cols + g)
    x = torch.randn(rows, cols, generator=gen).to(dt).to(cuda)
    r = (torch.randn(rows, cols, generator=gen) * 3).to(dt).to(cuda)
    w = (1 + 0.3 * torch.randn(cols, generator=gen)).to(dt).to(cuda)
    check(x, w, None, g, codes, tob.add_rms_norm_group_quant(x, w, g, dtype=codes))
    got = tob.add_rms_norm_group_quant(x, w, g, r, dtype=codes)
    check(x, w, r, g, codes, got)


@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols,g", [
    # rows past a few per SM run on persistent blocks: a last block part full, one and several rows
    # per block, columns that leave threads idle, rows of one and of two blocks' shared memory
    (593, 256, 256), (1201, 384, 128), (777, 1024, 64), (650, 5120, 5120), (700, 11008, 128),
    (601, 16384, 16384), (600, 8192, 8192), (2000, 32, 32), (3000, 64, 16),
])
def test_many_rows(cuda, codes, dt, rows, cols, g):
    gen = torch.Generator(device=cuda).manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=gen, device=cuda).to(dt)
    r = (torch.randn(rows, cols, generator=gen, device=cuda) * 3).to(dt)
    w = (1 + 0.3 * torch.randn(cols, generator=gen, device=cuda)).to(dt)
    x[7] = 0
    x[11, 3] = float("inf")
    keep = [i for i in range(rows) if i != 11]
    q, s = tob.add_rms_norm_group_quant(x, w, g, dtype=codes)
    check(x[keep], w, None, g, codes, (q[keep], s[keep]))
    assert bool(torch.isnan(s[11, 3 // g]))
    r[11] = -x[11].clamp(max=1)
    x[11, 3] = 1
    want = tob.add_rms_norm_group_quant(x, w, g, r, dtype=codes)
    check(x, w, r, g, codes, want)
    wide = torch.full((rows, cols + 8), 7, dtype=dt, device=cuda)
    wide[:, 8:] = r
    got = tob.add_rms_norm_group_quant(x, w, g, wide[:, 8:], dtype=codes, residual_out=wide[:, 8:])
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    assert bool((wide[:, :8] == 7).all())


@pytest.mark.parametrize("cols,g", [(512, 128), (512, 512), (480, 96), (333, 111), (40960, 128),
                                    (40960, 40960), (40960, 5120)])
@pytest.mark.parametrize("into", ["x", "residual"])
def test_residual_in_place(cuda, cols, g, into):
    gen = torch.Generator().manual_seed(cols)
    x = torch.randn(6, cols, generator=gen).bfloat16().to(cuda)
    r = torch.randn(6, cols, generator=gen).bfloat16().to(cuda)
    w = torch.rand(cols, generator=gen).bfloat16().to(cuda)
    want = tob.add_rms_norm_group_quant(x, w, g, r)
    x2, r2 = x.clone(), r.clone()
    dst = x2 if into == "x" else r2
    q, s, h = tob.add_rms_norm_group_quant(x2, w, g, r2, residual_out=dst)
    assert h is dst
    assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8))
    assert torch.equal(s, want[1]) and torch.equal(h, want[2])
    assert torch.equal((r2 if into == "x" else x2), (r if into == "x" else x))


@pytest.mark.parametrize("g", [128, 640])
def test_layouts(cuda, g):
    """Strided rows, a storage offset, leading dimensions, a transposed x, an expanded residual and
    a strided residual_out whose other columns stay as they were."""
    cols = 640
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(2, 5, cols, generator=gen).bfloat16().to(cuda)
    r = torch.randn(2, 5, cols, generator=gen).bfloat16().to(cuda)
    w = torch.rand(cols, generator=gen).bfloat16().to(cuda)

    # Alignment decides the loads and with them the order of the row's sum, so layouts agree
    # within the definition's bound and not bit for bit.
    def same(got):
        check(x, w, r, g, torch.float8_e4m3fn, got)

    for pad in (1, 8):
        wide = torch.zeros(2, 5, cols + pad, dtype=torch.bfloat16, device=cuda)
        wide[..., pad:] = x
        out = torch.full((2, 5, cols + 2 * pad), 7, dtype=torch.bfloat16, device=cuda)
        view = out[..., pad:pad + cols]
        got = tob.add_rms_norm_group_quant(wide[..., pad:], w, g, r, residual_out=view)
        assert got[2] is view
        same(got)
        assert bool((out[..., :pad] == 7).all()) and bool((out[..., pad + cols:] == 7).all())
    flat = torch.zeros(x.numel() + 3, dtype=torch.bfloat16, device=cuda)
    flat[3:] = x.reshape(-1)
    same(tob.add_rms_norm_group_quant(flat[3:].view(x.shape), w, g, r))
    same(tob.add_rms_norm_group_quant(x.transpose(0, 1).contiguous().transpose(0, 1), w, g, r))
    row = r[:1, :1].expand(2, 5, cols)
    check(x, w, row, g, torch.float8_e4m3fn, tob.add_rms_norm_group_quant(x, w, g, row))


def test_scale_options(cuda):
    """Power-of-two scales and the column-major layout, as per_token_group_quant_fp8 has them."""
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(12, 512, generator=gen).bfloat16().to(cuda)
    w = torch.rand(512, generator=gen).bfloat16().to(cuda)
    q0, s0 = tob.add_rms_norm_group_quant(x, w, 128)
    q1, s1 = tob.add_rms_norm_group_quant(x, w, 128, use_ue8m0=True)
    assert bool((torch.log2(s1) == torch.log2(s1).round()).all())
    assert bool((s1 >= s0).all()) and bool((s1 < 2 * s0 * (1 + 1e-6)).all())
    q2, s2 = tob.add_rms_norm_group_quant(x, w, 128, column_major_scales=True)
    assert torch.equal(q2.view(torch.uint8), q0.view(torch.uint8))
    # the layout per_token_group_quant_fp8 gives the same scales
    lay = s0.reshape(-1).reshape(4, 12).t().contiguous()
    assert torch.equal(s2, lay)


@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("cols,g", [(512, 128), (512, 512), (480, 96), (333, 111)])
def test_rows_that_are_not_numbers(cuda, codes, cols, g):
    """A row of zeros, a NaN, an infinity, subnormals: each in its own row, the others untouched."""
    x = torch.ones(6, cols, dtype=torch.bfloat16, device=cuda)
    x[1] = 0
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    x[4] = 1e-39
    w = torch.ones(cols, dtype=torch.bfloat16, device=cuda)
    q, s = tob.add_rms_norm_group_quant(x, w, g, dtype=codes)
    qmax = 448.0 if codes == torch.float8_e4m3fn else 127.0
    qf = q.float()
    for row in (0, 5):
        assert bool((qf[row] == qmax).all())
        torch.testing.assert_close(s[row], torch.full_like(s[row], 1 / qmax), rtol=1e-5, atol=0)
    assert bool((qf[1] == 0).all())
    # the IEEE quotient (torch on the GPU multiplies by a reciprocal)
    floor = float(np.float32(1e-10) / np.float32(qmax))
    assert bool((s[1] == floor).all())
    assert bool(torch.isnan(s[2]).all())
    assert bool(torch.isnan(qf[2]).all()) if codes != torch.int8 else bool((q[2] == 0).all())
    # mean of squares infinite: finite values become 0, the infinity NaN, in its group alone
    assert bool(torch.isnan(s[3, 4 // g])) and int(torch.isnan(s[3]).sum()) == 1
    assert bool((s[4] > 0).all()) and bool(torch.isfinite(s[4]).all())


def test_graph_stream_and_empty(cuda):
    x = torch.randn(4, 512, device=cuda).half()
    r = torch.randn(4, 512, device=cuda).half()
    w = torch.ones(512, device=cuda).half()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        tob.add_rms_norm_group_quant(x, w, 128, r)
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, s, h = tob.add_rms_norm_group_quant(x, w, 128, r)
    x.copy_(torch.randn(4, 512, device=cuda).half())
    g.replay()
    want = tob.add_rms_norm_group_quant(x, w, 128, r)
    assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8))
    assert torch.equal(s, want[1]) and torch.equal(h, want[2])
    q, s = tob.add_rms_norm_group_quant(torch.empty(0, 512, device=cuda).half(), w, 128)
    assert q.shape == (0, 512) and s.shape == (0, 4)


@pytest.mark.parametrize("tokens", [1, 19, 300])
@pytest.mark.parametrize("codes,bs", [("e4m3", "block"), ("int8", "channel")])
def test_mlp_block(cuda, tokens, codes, bs):
    """The operators together, as a pre-norm MLP block runs them: norm + quantiser, up projection
    with bias and gelu, quantiser, down projection with bias added to the residual stream in place;
    then the unquantised head. Against 64 bits on the codes the kernels chose: with the quantisers'
    outputs taken as given, what is left are fp32 sums (k 2^-23 of the absolute products), the
    activation (slope 1.13) and one rounding per output."""
    d, f, v = 512, 1280, 300
    gen = torch.Generator().manual_seed(tokens)
    cast = torch.float8_e4m3fn if codes == "e4m3" else torch.int8
    amp = 100 if codes == "e4m3" else 40

    def weight(n, k):
        q = (torch.randn(n, k, generator=gen) * amp).clamp(-127, 127).round().to(cast).to(cuda)
        shape = (-(-n // 128), -(-k // 128)) if bs == "block" else (n, 1)
        return q, ((0.5 + torch.rand(*shape, generator=gen)) / (amp * k ** 0.5)).to(cuda)

    up, up_s = weight(f, d)
    down, down_s = weight(d, f)
    b1 = torch.randn(f, generator=gen).bfloat16().to(cuda)
    b2 = torch.randn(d, generator=gen).bfloat16().to(cuda)
    head = (torch.randn(d, v, generator=gen) * d ** -0.5).bfloat16().to(cuda)
    w = (1 + 0.1 * torch.randn(d, generator=gen)).bfloat16().to(cuda)
    x = torch.randn(tokens, d, generator=gen).bfloat16().to(cuda)
    stream = torch.randn(tokens, d, generator=gen).bfloat16().to(cuda)
    op = (tob.w8a8_block_fp8_matmul_bias_act if codes == "e4m3"
          else tob.w8a8_block_int8_matmul_bias_act)
    quant = tob.per_token_group_quant_fp8 if codes == "e4m3" else tob.per_token_group_quant_int8

    def grp(k):
        return 128 if bs == "block" else k

    def block(k):
        return [128, 128] if bs == "block" else [1, k]

    stream0 = stream.clone()
    q, s, h = tob.add_rms_norm_group_quant(x, w, grp(d), stream, dtype=cast, residual_out=stream)
    check(x, w, stream0, grp(d), cast, (q, s, h))
    mid = op(q, up, s, up_s, block(d), b1, act="gelu", output_dtype=torch.bfloat16)
    qm, sm = quant(mid, grp(f))
    before = h.clone()
    y = op(qm, down, sm, down_s, block(f), b2, residual=h, out=h, output_dtype=torch.bfloat16)
    assert y is h
    logits = tob.gemm_bias_act(y, head)

    def deq(c, sc, bn, bk):
        n, k = c.shape
        rows = torch.arange(n, device=cuda) // bn
        return c.float().to(F64) * sc.to(F64)[rows][:, torch.arange(k, device=cuda) // bk]

    def near(got, pre, mass, k, extra, act=None):
        want = pre
        if act:
            want = 0.5 * pre * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (pre + 0.044715 * pre ** 3)))
        want = want + extra
        tol = 2.0 ** -8 * want.abs() * 1.01 + 1.13 * (k + 3) * 2.0 ** -23 * mass \
            + 4e-6 * (pre.abs() + 1 + (extra.abs() if torch.is_tensor(extra) else 0))
        assert bool(((got.to(F64) - want).abs() <= tol).all())

    bn, bk = block(d)
    a64, u64 = deq(q, s, 1, bk), deq(up, up_s, bn, bk)
    near(mid, a64 @ u64.t() + b1.to(F64), a64.abs() @ u64.abs().t(), d, 0.0, act="gelu")
    bn, bk = block(f)
    m64, d64 = deq(qm, sm, 1, bk), deq(down, down_s, bn, bk)
    near(y, m64 @ d64.t() + b2.to(F64), m64.abs() @ d64.abs().t(), f, before.to(F64))
    near(logits, y.to(F64) @ head.to(F64), y.to(F64).abs() @ head.to(F64).abs(), d, 0.0)
