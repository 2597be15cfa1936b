"""add_rms_norm_group_quant where the rows decide how many threads hold one: a row to an SM, two, and
more, at columns on both sides of what a block holds (1024, 1536 and 2048 packs of 16 bytes)."""

from __future__ import annotations

import pytest
import torch

import tileops_b200 as tob
from test_gpu_norm_quant import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 147, 149, 297])
@pytest.mark.parametrize("cols", [4104, 8192, 8200, 11008, 12288, 12296, 16384, 16392])
def test_few_rows(cuda, codes, dt, rows, cols):
    gen = torch.Generator(device=cuda).manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=gen, device=cuda).to(dt)
    r = (torch.randn(rows, cols, generator=gen, device=cuda) * 3).to(dt)
    w = (1 + 0.3 * torch.randn(cols, generator=gen, device=cuda)).to(dt)
    for g in (8, cols):
        want = tob.add_rms_norm_group_quant(x, w, g, r, dtype=codes)
        check(x, w, r, g, codes, want)
        h = r.clone()
        got = tob.add_rms_norm_group_quant(x, w, g, h, dtype=codes, residual_out=h)
        assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))
        assert torch.equal(got[1], want[1]) and torch.equal(h, want[2])
