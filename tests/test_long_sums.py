"""int8 products whose sums do not fit int32: 131072 products of -128 are 2^31."""

from __future__ import annotations

import pytest
import torch

import tileops_b200 as tob
from tileops_b200 import _lib


def test_long_blocks_of_the_simt_tiles_are_refused():
    """Before any device work, so it holds without a GPU."""
    lib = _lib.load()
    f32, p = _lib.DTYPE_CODES[torch.float32], 1 << 20

    def call(fn, k, bk):
        return fn(p, p, p, p, None, 0, None, 2, p, 2, f32, 2, 2, k, 1, bk, None, 0, None)

    assert call(lib.to_w8a8_i8_gemm_bias_act, 400000, 131072 + 64) == _lib.TO_EUNSUPPORTED
    assert "131071" in _lib.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("k", [131072, 131073, 262144 + 80])
@pytest.mark.parametrize("m,n,bn", [(1, 5, 1), (3, 130, 1), (70, 200, 1), (70, 200, 200),
                                    (2000, 640, 640)])
def test_sums_past_int32(cuda, m, n, bn, k):
    """One K block, rows and columns of one value each: every partial sum over whole slices is a
    multiple of 2^12 (the last ragged slice of 2^5) below 2^33 with at most 24 significant bits, so
    fp32 holds it exactly and the result equals the product's value rounded once."""
    av = torch.tensor([-128, 127, 64], device=cuda)[torch.arange(m, device=cuda) % 3]
    bv = torch.tensor([-128, 32], device=cuda)[torch.arange(n, device=cuda) % 2]
    a = av.to(torch.int8)[:, None].expand(m, k).contiguous()
    b = bv.to(torch.int8)[:, None].expand(n, k).contiguous()
    a_s = torch.full((m, 1), 0.5, device=cuda)
    b_s = torch.full((-(-n // bn), 1), 2.0 ** -10, device=cuda)
    y = tob.w8a8_block_int8_matmul_bias_act(a, b, a_s, b_s, [bn, k], output_dtype=torch.float32)
    want = (av[:, None].double() * bv.double() * k * 2.0 ** -11).float()
    assert torch.equal(y, want)
