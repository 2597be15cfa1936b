"""Tensors seen as rows with a pitch: what the facade hands the kernels as a row stride, and what it
calls an overlap, for views whose leading dimensions have size 1 (the [batch, 1, width] of a decode
step)."""

from __future__ import annotations

import pytest
import torch

import tileops_b200 as tob
from tileops_b200.fused import _overlap, _row_stride

Z = torch.zeros


@pytest.mark.parametrize("t,want", [
    (Z(4, 1, 128)[..., :64], 128), (Z(4, 1, 128)[..., 64:], 128), (Z(2, 4, 1, 128)[..., :64], 128),
    (Z(4, 1, 1, 128)[..., :64], 128), (Z(1, 4, 128)[..., :64], 128), (Z(1, 1, 128)[..., :64], 64),
    (Z(2, 3, 128)[..., :64], 128), (Z(2, 6, 128)[:, :3, :64], None), (Z(2, 6, 128)[:, :1, :64], 768),
    (Z(4, 64), 64), (Z(4, 1, 64), 64), (Z(64), 64), (Z(1, 64), 64), (Z(1, 64).expand(4, 64), None),
    (Z(4, 1, 1).expand(4, 3, 1), None), (Z(8, 3, 4).transpose(0, 1), None), (Z(8, 4).t(), None),
    (Z(4, 1, 64).expand(4, 2, 64), None), (Z(5, 1)[::2], 2), (Z(2, 3, 1, 8)[:, ::3], 24),
])
def test_row_stride(t, want):
    got = _row_stride(t)
    assert got == want
    if got is not None:  # the rows it names are the tensor's
        t.copy_(torch.arange(t.numel()).view(t.shape))
        cols = t.shape[-1]
        rows = t.numel() // cols
        seen = torch.as_strided(t, (rows, cols), (got, 1), t.storage_offset())
        assert torch.equal(seen.reshape(-1), t.reshape(-1))


def test_overlap_of_one_token_slices():
    for wide in (Z(4, 1, 128), Z(2, 4, 1, 128), Z(4, 1, 1, 128), Z(4, 128)):
        lo, hi = wide[..., :64], wide[..., 64:]
        assert not _overlap(lo, hi) and not _overlap(hi, lo)
        assert _overlap(lo, wide[..., 63:127]) and _overlap(lo, lo)


def sliced(rows, cols, dt, device, fill=None):
    """[rows, 1, cols] in the second half of [rows, 1, 2 cols] of sevens; and the whole."""
    wide = torch.full((rows, 1, 2 * cols), 7, dtype=dt, device=device)
    if fill is not None:
        wide[..., cols:] = fill
    return wide[..., cols:], wide


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(4, 64), (3, 1000), (300, 256)])
def test_norm_of_one_token_slices(cuda, dt, rows, cols):
    gen = torch.Generator().manual_seed(rows + cols)
    x0 = torch.randn(rows, 1, cols, generator=gen).to(dt).to(cuda)
    r0 = torch.randn(rows, 1, cols, generator=gen).to(dt).to(cuda)
    w = torch.rand(cols, generator=gen).to(dt).to(cuda)
    want = tob.add_rms_norm_group_quant(x0, w, cols, r0)
    x, _ = sliced(rows, cols, dt, cuda, x0)
    r = sliced(rows, cols, dt, cuda, r0)[0]
    for residual, (out, whole) in [(r0, sliced(rows, cols, dt, cuda)), (r, sliced(rows, cols, dt, cuda)),
                                   (r, (r, r._base))]:
        q, s, h = tob.add_rms_norm_group_quant(x, w, cols, residual, residual_out=out)
        assert h is out and torch.equal(out, want[2])
        assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8))
        assert torch.equal(s, want[1])
        assert bool((whole[..., :cols] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,n,k", [(4, 64, 64), (5, 100, 48), (300, 264, 128)])
def test_products_of_one_token_slices(cuda, dt, rows, n, k):
    gen = torch.Generator().manual_seed(rows + n)
    a = torch.randint(-9, 10, (rows, 1, k), generator=gen).to(torch.int8).to(cuda)
    b = torch.randint(-3, 4, (n, k), generator=gen).to(torch.int8).to(cuda)
    one_m, one_n = torch.ones(rows, 1, 1, device=cuda), torch.ones(n, 1, device=cuda)
    r0 = torch.randint(-8, 9, (rows, 1, n), generator=gen).to(dt).to(cuda)
    want = (a.double() @ b.double().t() + r0.double()).to(dt)
    r, _ = sliced(rows, n, dt, cuda, r0)
    out, whole = sliced(rows, n, dt, cuda)
    y = tob.w8a8_block_int8_matmul_bias_act(a, b, one_m, one_n, [1, k], residual=r, out=out,
                                            output_dtype=dt)
    assert y is out and torch.equal(out, want) and bool((whole[..., :n] == 7).all())
    tob.w8a8_block_int8_matmul_bias_act(a, b, one_m, one_n, [1, k], residual=r, out=r,
                                        output_dtype=dt)
    assert torch.equal(r, want)


@pytest.mark.gpu
def test_gated_activations_of_one_token_slices(cuda):
    gen = torch.Generator().manual_seed(1)
    u = torch.randn(6, 1, 512, generator=gen).half().to(cuda)
    gate, up = u[..., :256], u[..., 256:]
    out, whole = sliced(6, 256, torch.float16, cuda)
    want = tob.silu_and_mul(gate.contiguous(), up.contiguous())
    assert torch.equal(tob.silu_and_mul(gate, up, out=out), want)
    assert bool((whole[..., :256] == 7).all())
    q, s = tob.act_and_mul_group_quant(gate, up, 128)
    q0, s0 = tob.act_and_mul_group_quant(gate.contiguous(), up.contiguous(), 128)
    assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s, s0)


def test_in_place_through_another_view():
    """One row of a wide buffer, as a slice and as an unsqueezed row: the strides of the size-1
    dimension differ, the memory does not. What is allowed goes on to the check for a GPU."""
    buf, w = Z(5, 16), Z(4, 4)
    row, again = buf[:1, :4], buf[0, :4][None]
    assert row.stride() != again.stride()
    a = Z(1, 4)
    with pytest.raises(TypeError, match="CUDA"):
        tob.gemm_bias_act(a, w, residual=row, out=again)
    with pytest.raises(TypeError, match="CUDA"):
        tob.add_rms_norm_group_quant(a, Z(4), 4, row, residual_out=again)
    with pytest.raises(ValueError, match="partly overlaps"):
        tob.gemm_bias_act(a, w, residual=row, out=buf[:1, 1:5])
