"""Fused operators whose offsets pass 2^31, and block widths of every kind on the folding tiles."""

from __future__ import annotations

import pytest
import torch

import tileops_b200 as tob
from test_gpu_norm_quant import check

pytestmark = pytest.mark.gpu

F64 = torch.float64


@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8])
def test_norm_past_2_31_elements(cuda, codes):
    rows, cols, g = 270000, 8192, 128
    gen = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(1, cols, generator=gen, device=cuda).bfloat16().expand(rows, cols).contiguous()
    x *= (1 + torch.arange(rows, device=cuda) % 5).bfloat16()[:, None]
    r = torch.randn(1, cols, generator=gen, device=cuda).bfloat16().expand(rows, cols).contiguous()
    w = torch.rand(cols, generator=gen, device=cuda).bfloat16()
    keep = [0, 1, 4095, 131071, 262143, 262144, 262145, rows - 2, rows - 1]
    r0 = r[keep].clone()
    q, s, h = tob.add_rms_norm_group_quant(x, w, g, r, dtype=codes, residual_out=r)
    check(x[keep], w, r0, g, codes, (q[keep], s[keep], h[keep]))


@pytest.mark.parametrize("m,n,k", [(70000, 8, 32001), (40, 70000, 32001)])
def test_copies_past_2_31_bytes(cuda, m, n, k):
    """An operand of more than 2^31 bytes whose rows are copied to aligned ones."""
    a = (torch.arange(m, device=cuda) % 5 - 2).to(torch.int8)[:, None].expand(m, k).contiguous()
    b = (torch.arange(n, device=cuda) % 3 - 1).to(torch.int8)[:, None].expand(n, k).contiguous()
    a[:, -1], b[:, -1] = 1, 1
    y = tob.w8a8_block_int8_matmul_bias_act(a, b, torch.ones(m, 1, device=cuda),
                                            torch.ones(n, 1, device=cuda), [1, k],
                                            output_dtype=torch.float32)
    want = ((k - 1) * a[:, :1].float() * b[:, :1].float().t() + 1)
    assert torch.equal(y, want)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("bn", [32, 64, 96, 160, 192, 224, 352])
@pytest.mark.parametrize("m,n,k,bk", [(2000, 2304, 700, 128), (1000, 4100, 1100, 256),
                                      (700, 5000, 400, 384), (3000, 1000, 900, 640)])
def test_block_widths(cuda, codes, bn, m, n, k, bk):
    gen = torch.Generator(device=cuda).manual_seed(m + bn)

    def ri(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=gen, device=cuda)

    a, b = ri(-8, 8, m, k), ri(-8, 8, n, k)
    kt, nt = -(-k // bk), -(-n // bn)
    a_s, b_s = torch.exp2(ri(-2, 0, m, kt).float()), torch.exp2(ri(-2, 0, nt, kt).float())
    op = (tob.w8a8_block_int8_matmul_bias_act if codes == torch.int8
          else tob.w8a8_block_fp8_matmul_bias_act)
    y = op(a.float().to(codes), b.float().to(codes), a_s, b_s, [bn, bk], output_dtype=torch.float32)
    kb = torch.arange(k, device=cuda) // bk
    nb = torch.arange(n, device=cuda) // bn
    want = (a.to(F64) * a_s.to(F64)[:, kb]) @ (b.to(F64) * b_s.to(F64)[nb][:, kb]).t()
    assert torch.equal(y, want.float())
