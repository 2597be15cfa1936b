"""Dimensions whose tiles or strides would pass 2^31 in the kernels' 32-bit indexes are refused by the
C entries, before any device work."""

from __future__ import annotations

import pytest
import torch

from tileops_b200 import _lib

TOP = 2 ** 31 - 1
P = 1 << 20


@pytest.mark.parametrize("m,n,k", [(TOP, 8, 8), (8, TOP, 8), (8, 8, TOP), (TOP - 1000, 8, 8),
                                   (8, 8, TOP - 1000), (8, TOP - 1000, 8)])
def test_products(m, n, k):
    lib = _lib.load()
    for dt in (torch.float16, torch.float32):
        code = _lib.DTYPE_CODES[dt]
        assert lib.to_gemm_bias_act(P, k, P, None, 0, None, 0, P, n, code, m, n, k, None, 0,
                                    None) == _lib.TO_EINVAL
    for fn in (lib.to_w8a8_i8_gemm_bias_act, lib.to_w8a8_fp8_gemm_bias_act):
        for bk in (128, 64, k):
            assert fn(P, P, P, P, None, 0, None, 0, P, n, 0, m, n, k, 1, bk, None, 0,
                      None) == _lib.TO_EINVAL


@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [TOP, TOP - 1, TOP - 600, TOP - 1000])
def test_norm(dt, cols):
    lib = _lib.load()
    for group in (cols, 1):
        assert lib.to_add_rms_norm_group_quant(
            P, cols, None, 0, P, _lib.DTYPE_CODES[dt], 1, cols, group, 1e-6, 1e-10, 0, 0,
            _lib.DTYPE_CODES[torch.int8], P, P, None, 0, None) == _lib.TO_EINVAL
