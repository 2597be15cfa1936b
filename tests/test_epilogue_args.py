"""Refusals of the fused norm quantiser and of the products with an epilogue: raised before any
device work, so they hold on CPU tensors too; and the C entries' own checks, which launch nothing."""

from __future__ import annotations

import pytest
import torch

import tileops_b200 as tob
from tileops_b200 import _lib

Z = torch.zeros


@pytest.mark.parametrize("err,match,args,kw", [
    (ValueError, "2-D", (Z(3), Z(3, 4)), {}),
    (ValueError, "incompatible", (Z(2, 3), Z(4, 5)), {}),
    (TypeError, "dtypes must match", (Z(2, 3), Z(3, 4).half()), {}),
    (ValueError, "Unsupported dtype", (Z(2, 3).int(), Z(3, 4).int()), {}),
    (ValueError, "act must be", (Z(2, 3), Z(3, 4)), {"act": "tanh"}),
    (ValueError, "bias.shape", (Z(2, 3), Z(3, 4), Z(3)), {}),
    (ValueError, "bias.shape", (Z(2, 3), Z(3, 4), Z(1, 4)), {}),
    (TypeError, "bias.dtype", (Z(2, 3), Z(3, 4), Z(4).half()), {}),
    (ValueError, "residual.shape", (Z(2, 3), Z(3, 4)), {"residual": Z(4)}),
    (TypeError, "residual.dtype", (Z(2, 3), Z(3, 4)), {"residual": Z(2, 4).half()}),
    (ValueError, "out.shape", (Z(2, 3), Z(3, 4)), {"out": Z(4, 2)}),
    (TypeError, "out.dtype", (Z(2, 3), Z(3, 4)), {"out": Z(2, 4).half()}),
    (TypeError, "CUDA", (Z(2, 3), Z(3, 4)), {"act": "silu"}),
])
def test_gemm_bias_act_refusals(err, match, args, kw):
    with pytest.raises(err, match=match):
        tob.gemm_bias_act(*args, **kw)


@pytest.mark.parametrize("fp8", [False, True])
def test_w8a8_bias_act_refusals(fp8):
    op = tob.w8a8_block_fp8_matmul_bias_act if fp8 else tob.w8a8_block_int8_matmul_bias_act
    cast = torch.float8_e4m3fn if fp8 else torch.int8
    a, b = Z(2, 8).to(cast), Z(3, 8).to(cast)
    a_s, b_s = Z(2, 1), Z(3, 1)
    for err, match, args, kw in [
        (ValueError, "length 2", (a, b, a_s, b_s, [1]), {}),
        (ValueError, "K mismatch", (a, Z(3, 9).to(cast), a_s, b_s, [1, 8]), {}),
        (TypeError, "must be", (Z(2, 8), Z(3, 8), a_s, b_s, [1, 8]), {}),
        (ValueError, "K must be positive", (Z(2, 0).to(cast), Z(3, 0).to(cast), a_s, b_s, [1, 8]), {}),
        (ValueError, "contiguous", (a, Z(8, 3).to(cast).t(), a_s, b_s, [1, 8]), {}),
        (ValueError, "As shape", (a, b, Z(2, 2), b_s, [1, 8]), {}),
        (ValueError, "Bs shape", (a, b, a_s, Z(2, 1), [1, 8]), {}),
        (TypeError, "output_dtype", (a, b, a_s, b_s, [1, 8]), {"output_dtype": torch.int32}),
        (ValueError, "act must be", (a, b, a_s, b_s, [1, 8]), {"act": "swish"}),
        (ValueError, "bias.shape", (a, b, a_s, b_s, [1, 8], Z(2).half()), {}),
        (TypeError, "bias.dtype", (a, b, a_s, b_s, [1, 8], Z(3)), {}),
        (ValueError, "residual.shape", (a, b, a_s, b_s, [1, 8]), {"residual": Z(3, 2).half()}),
        (TypeError, "out.dtype", (a, b, a_s, b_s, [1, 8]), {"out": Z(2, 3)}),
        (TypeError, "CUDA", (a, b, a_s, b_s, [1, 8]), {}),
    ]:
        with pytest.raises(err, match=match):
            op(*args, **kw)


def test_overlaps_are_refused():
    """An output over an operand, or part of the residual, would be read after it is written. What
    is allowed goes on to the next check, that the tensors are on a GPU."""
    buf, w, wide = Z(9, 4), Z(4, 4), Z(8, 12)
    x, r = buf[:8], Z(8, 4)

    def gemm(a, out, residual=None, bias=None, b=w):
        return tob.gemm_bias_act(a, b, bias, residual=residual, out=out)

    for args in [(x, x), (x, buf[1:])]:
        with pytest.raises(ValueError, match="overlaps an input"):
            gemm(*args)
    with pytest.raises(ValueError, match="overlaps an input"):
        gemm(Z(4, 4), w)
    with pytest.raises(ValueError, match="overlaps an input"):
        gemm(r, x, bias=buf[3])
    with pytest.raises(ValueError, match="partly overlaps"):
        gemm(r, x, residual=buf[1:])
    with pytest.raises(ValueError, match="partly overlaps"):
        gemm(Z(4, 4), x[:4], residual=x[:4].t())
    with pytest.raises(ValueError, match="partly overlaps"):
        gemm(r, wide[:, 2:6], residual=wide[:, :4])
    for args in [(r, x, x), (r, x, buf[:8]), (wide[:, :4], wide[:, 4:8], wide[:, 8:]), (r, x, Z(8, 4))]:
        with pytest.raises(TypeError, match="CUDA"):
            gemm(*args)
    a8 = Z(8, 8, dtype=torch.int8)
    out = a8.view(torch.float16)  # [8, 4] over the operand's memory
    with pytest.raises(ValueError, match="overlaps an input"):
        tob.w8a8_block_int8_matmul_bias_act(a8, Z(4, 8, dtype=torch.int8), Z(8, 1), Z(4, 1), [1, 8],
                                            out=out)

    def norm(x, r, out, w=Z(4)):
        return tob.add_rms_norm_group_quant(x, w, 4, r, residual_out=out)

    for args in [(x, r, buf[1:]), (r, x, buf[1:])]:
        with pytest.raises(ValueError, match="partly overlaps"):
            norm(*args)
    with pytest.raises(ValueError, match="overlaps an input"):
        norm(r, Z(8, 4), x, buf[2])
    for args in [(x, r, x), (x, r, r), (x, x, x), (wide[:, :4], wide[:, 4:8], wide[:, 8:])]:
        with pytest.raises(TypeError, match="CUDA"):
            norm(*args)


def test_fnuz_operands_are_refused():
    a = Z(2, 8).to(torch.float8_e4m3fnuz)
    with pytest.raises(NotImplementedError, match="e4m3fn"):
        tob.w8a8_block_fp8_matmul_bias_act(a, a, Z(2, 1), Z(2, 1), [1, 8])


@pytest.mark.parametrize("err,match,args,kw", [
    (ValueError, "weight.shape", (Z(2, 8), Z(4), 4), {}),
    (ValueError, "weight.shape", (Z(()), Z(1), 1), {}),
    (ValueError, "divisible", (Z(2, 8), Z(8), 3), {}),
    (ValueError, "divisible", (Z(2, 8), Z(8), 0), {}),
    (TypeError, "codes must be", (Z(2, 8), Z(8), 4), {"dtype": torch.float8_e5m2}),
    (ValueError, "FP8 options", (Z(2, 8), Z(8), 4), {"dtype": torch.int8, "use_ue8m0": True}),
    (ValueError, "2-D", (Z(2, 2, 8), Z(8), 4), {"column_major_scales": True}),
    (ValueError, "residual.shape", (Z(2, 8), Z(8), 4, Z(8)), {}),
    (TypeError, "residual.dtype", (Z(2, 8), Z(8), 4, Z(2, 8).half()), {}),
    (TypeError, "weight.dtype", (Z(2, 8), Z(8).half(), 4), {}),
    (ValueError, "needs a residual", (Z(2, 8), Z(8), 4), {"residual_out": Z(2, 8)}),
    (ValueError, "residual_out.shape", (Z(2, 8), Z(8), 4, Z(2, 8)), {"residual_out": Z(8, 2)}),
    (ValueError, "quant_eps", (Z(2, 8), Z(8), 4), {"quant_eps": 0.0}),
    (ValueError, "quant_eps", (Z(2, 8), Z(8), 4), {"quant_eps": float("nan")}),
    (ValueError, "quant_eps", (Z(2, 8), Z(8), 4), {"quant_eps": float("inf")}),
    (ValueError, "eps", (Z(2, 8), Z(8), 4), {"eps": -1e-6}),
    (ValueError, "eps", (Z(2, 8), Z(8), 4), {"eps": float("nan")}),
    (TypeError, "CUDA", (Z(2, 8), Z(8), 4), {}),
])
def test_norm_quant_refusals(err, match, args, kw):
    with pytest.raises(err, match=match):
        tob.add_rms_norm_group_quant(*args, **kw)


def test_c_entries_check_before_they_launch():
    lib = _lib.load()
    f16 = _lib.DTYPE_CODES[torch.float16]

    def gemm(m, n, k, act=0, dtype=f16, lda=8, ldr=8, ldc=8, p=1 << 20):
        return lib.to_gemm_bias_act(p, lda, p, None, act, None, ldr, p, ldc, dtype, m, n, k, None, 0, None)

    assert gemm(-1, 4, 4) == _lib.TO_EINVAL
    assert gemm(0, 4, 4) == _lib.TO_OK and gemm(4, 0, 4) == _lib.TO_OK
    assert gemm(2, 8, 8, act=9) == _lib.TO_EINVAL
    assert gemm(2, 8, 8, dtype=_lib.DTYPE_CODES[torch.int8]) == _lib.TO_EUNSUPPORTED
    assert gemm(2, 8, 8, lda=7) == _lib.TO_EINVAL and gemm(2, 8, 8, ldc=7) == _lib.TO_EINVAL
    assert gemm(2, 8, 8, p=None) == _lib.TO_EINVAL
    for fn in (lib.to_w8a8_i8_gemm_bias_act, lib.to_w8a8_fp8_gemm_bias_act):
        def w8a8(m, n, k, bn=1, bk=8, act=0, p=1 << 20, fn=fn):
            return fn(p, p, p, p, None, act, None, n, p, n, f16, m, n, k, bn, bk, None, 0, None)

        assert w8a8(2, 2, 0) == _lib.TO_EINVAL and w8a8(2, 2, 8, bk=0) == _lib.TO_EINVAL
        assert w8a8(0, 2, 8) == _lib.TO_OK
        assert w8a8(2, 2, 8, act=-1) == _lib.TO_EINVAL and w8a8(2, 2, 8, p=None) == _lib.TO_EINVAL

    def norm(rows, cols, g, qd=torch.int8, ue=0, ldx=8, p=1 << 20, eps=1e-6, qe=1e-10):
        return lib.to_add_rms_norm_group_quant(p, ldx, None, 0, p, f16, rows, cols, g, eps, qe,
                                               ue, 0, _lib.DTYPE_CODES[qd], p, p, None, 0, None)

    assert norm(2, 8, 3) == _lib.TO_EINVAL and norm(2, 8, 0) == _lib.TO_EINVAL
    assert norm(2, 8, 8, ldx=4) == _lib.TO_EINVAL and norm(2, 8, 8, ue=1) == _lib.TO_EINVAL
    assert norm(2, 8, 8, qd=torch.float16) == _lib.TO_EUNSUPPORTED
    nan = float("nan")
    assert norm(2, 8, 8, qe=0.0) == _lib.TO_EINVAL and norm(2, 8, 8, qe=nan) == _lib.TO_EINVAL
    assert norm(2, 8, 8, eps=-1.0) == _lib.TO_EINVAL and norm(2, 8, 8, eps=nan) == _lib.TO_EINVAL
    assert norm(0, 8, 8) == _lib.TO_OK and norm(2, 8, 8, p=None) == _lib.TO_EINVAL
