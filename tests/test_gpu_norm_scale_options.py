"""add_rms_norm_group_quant with power-of-two scales and with column-major scales: the codes and the
scales against 64 bits, in every form the groups take."""

from __future__ import annotations

import pytest
import torch

import tileops_b200 as tob
from test_gpu_norm_quant import check, definition

pytestmark = pytest.mark.gpu

F64 = torch.float64
FORMS = [(5, 512, 128), (300, 512, 16), (7, 640, 640), (4, 480, 96), (3, 333, 111), (2, 9999, 99),
         (9, 20480, 128), (400, 8192, 256), (64, 12288, 128), (6, 36, 4)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols,g", FORMS)
def test_power_of_two_scales(cuda, dt, residual, rows, cols, g):
    """d = (cols / 32 + 24) 2^-24 bounds the relative error of y and of max|y| / 448 (see
    test_gpu_norm_quant). The scale is 2^k with 2^k >= max|y| / 448 and 2^(k-1) below it, up to d and
    to the rounding of log2 (|log2| < 32: half a step of it is 2^-20, a factor of 2^-20). A code
    stands for a value within half an e4m3 step of y, 2^-4 relatively or 2^-10 scale units."""
    gen = torch.Generator(device=cuda).manual_seed(rows + cols + g)
    x = torch.randn(rows, cols, generator=gen, device=cuda).to(dt)
    r = (torch.randn(rows, cols, generator=gen, device=cuda) * 3).to(dt) if residual else None
    w = (1 + 0.3 * torch.randn(cols, generator=gen, device=cuda)).to(dt)
    x[rows - 1] = 0
    if residual:
        r[rows - 1] = 0
    q, s = tob.add_rms_norm_group_quant(x, w, g, r, use_ue8m0=True)[:2]
    _, y, exact = definition(x, w, r, g, torch.float8_e4m3fn)
    d = (cols / 32 + 24) * 2.0 ** -24 + 2.0 ** -20
    s64 = s.to(F64)
    assert bool((torch.frexp(s)[0] == 0.5).all())
    assert bool((s64 >= exact * (1 - d)).all()) and bool((s64 / 2 <= exact * (1 + d)).all())
    sx = s64.repeat_interleave(g, -1)
    v = q.to(torch.float32).to(F64) * sx
    tol = 2.0 ** -4 * y.abs() + 2.0 ** -10 * sx
    assert bool(((v - y).abs() <= tol * (1 + 1e-9) + 4 * d * y.abs()).all())


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("ue8m0", [False, True])
@pytest.mark.parametrize("rows,cols,g", FORMS + [(1, 512, 128), (5, 512, 512)])
def test_column_major_scales(cuda, residual, ue8m0, rows, cols, g):
    """The codes of the row-major call, and its scales in the layout of per_token_group_quant_fp8."""
    gen = torch.Generator(device=cuda).manual_seed(rows + cols + g)
    x = torch.randn(rows, cols, generator=gen, device=cuda).bfloat16()
    r = torch.randn(rows, cols, generator=gen, device=cuda).bfloat16() if residual else None
    w = (1 + 0.3 * torch.randn(cols, generator=gen, device=cuda)).bfloat16()
    want = tob.add_rms_norm_group_quant(x, w, g, r, use_ue8m0=ue8m0)
    got = tob.add_rms_norm_group_quant(x, w, g, r, use_ue8m0=ue8m0, column_major_scales=True)
    if not ue8m0:
        check(x, w, r, g, torch.float8_e4m3fn, want)
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))
    assert torch.equal(got[1], want[1].reshape(-1).reshape(cols // g, rows).t().contiguous())
    # the same layout, from the quantiser that stands beside this one
    p0 = tob.per_token_group_quant_fp8(x, g)[1]
    p1 = tob.per_token_group_quant_fp8(x, g, column_major_scales=True)[1]
    assert torch.equal(p1, p0.reshape(-1).reshape(cols // g, rows).t().contiguous())
    assert got[1].shape == p1.shape and got[1].stride() == p1.stride()
