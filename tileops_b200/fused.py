"""Gated activations of an MLP block, as in the reference's ``tileops.fused``
(tileops/fused.py:97-114): ``silu_and_mul(a, b)`` = ``silu(a) * b`` and ``gelu_and_mul(a, b)`` =
``gelu(a, tanh approximation) * b``, element-wise over same-shaped tensors, with the
reference's argument names, ``out=`` keyword and validation (ValueError for shapes and devices,
TypeError for dtypes).

Inputs may be strided views whose last dimension is contiguous (for example the gate and up
halves ``u[:, :F]`` and ``u[:, F:]`` of a fused gate_up output): the kernel reads them in place.
Other layouts are made contiguous first. An ``out`` that the kernel cannot write in place (a
transposed view, say) receives a copy of the result and is returned, as in the reference.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_ROWS = torch.contiguous_format
_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _validate_fused(a: torch.Tensor, b: torch.Tensor, out: Optional[torch.Tensor],
                    op: str) -> None:
    # Same checks, order and messages as tileops/fused.py:34-64.
    if a.shape != b.shape:
        raise ValueError(f"{op}: shape mismatch — a.shape={a.shape}, b.shape={b.shape}")
    if a.dtype != b.dtype:
        raise TypeError(f"{op}: dtype mismatch — a.dtype={a.dtype}, b.dtype={b.dtype}")
    if a.device != b.device:
        raise ValueError(f"{op}: device mismatch — a.device={a.device}, b.device={b.device}")
    if out is not None:
        if out.shape != a.shape:
            raise ValueError(f"{op}: out.shape={out.shape} != input shape {a.shape}")
        if out.dtype != a.dtype:
            raise TypeError(f"{op}: out.dtype={out.dtype} != input dtype {a.dtype}")
        if out.device != a.device:
            raise ValueError(f"{op}: out.device={out.device} != input device {a.device}")


def _row_stride(t: torch.Tensor) -> Optional[int]:
    """Row stride of ``t`` seen as [numel / last, last] with a contiguous last dimension, or
    None when it cannot be seen that way without a copy."""
    if t.dim() == 0:
        return 1
    cols = t.shape[-1]
    if cols > 1 and t.stride(-1) != 1:
        return None
    if t.numel() == 0:
        return cols
    # The leading dimensions must collapse into one row index. Those of size 1 have no say: the
    # pitch of [4, 1, 128][..., :64] is 128.
    ld = outer = None
    for i in range(t.dim() - 2, -1, -1):
        n, step = t.shape[i], t.stride(i)
        if n == 1:
            continue
        if ld is None:
            ld = step
        elif step != outer:
            return None
        outer = step * n
    if ld is None:  # one row
        return cols
    return ld if ld >= cols else None


def _act_mul(op: str, entry: str, a: torch.Tensor, b: torch.Tensor,
             out: Optional[torch.Tensor]) -> torch.Tensor:
    _validate_fused(a, b, out, op)
    _lib.ensure_device(a, op)
    if a.dtype not in _DTYPES:
        raise TypeError(f"{op}: unsupported dtype {a.dtype} (float32, float16 and bfloat16 are "
                        "supported)")
    cols = a.shape[-1] if a.dim() > 0 else 1
    rows = a.numel() // cols if cols else 0
    lda = _row_stride(a)
    if lda is None:
        a = a.contiguous()
        lda = cols
    ldb = _row_stride(b)
    if ldb is None:
        b = b.contiguous()
        ldb = cols
    dst = out
    ldc = _row_stride(out) if out is not None else None
    if ldc is None:
        dst = torch.empty(a.shape, dtype=a.dtype, device=a.device)
        ldc = cols
    if a.numel():
        _lib.call(entry, a.data_ptr(), b.data_ptr(), dst.data_ptr(), _lib.DTYPE_CODES[a.dtype],
                  rows, cols, lda, ldb, ldc, _lib.stream_ptr())
    if out is not None and dst is not out:
        out.copy_(dst)
        return out
    return dst


def silu_and_mul(a: torch.Tensor, b: torch.Tensor, *,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``silu(a) * b`` element-wise (same shapes) -- tileops/fused.py:97."""
    return _act_mul("silu_and_mul", "to_silu_and_mul", a, b, out)


def gelu_and_mul(a: torch.Tensor, b: torch.Tensor, *,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``gelu(a) * b`` with the tanh GELU approximation -- tileops/fused.py:107."""
    return _act_mul("gelu_and_mul", "to_gelu_and_mul", a, b, out)


def act_and_mul_group_quant(a: torch.Tensor, b: torch.Tensor, group_size: int, *,
                            act: str = "silu", dtype: Optional[torch.dtype] = None,
                            eps: float = 1e-10, column_major_scales: bool = False,
                            use_ue8m0: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Library extension (no reference counterpart): ``silu_and_mul(a, b)`` (or gelu with
    ``act="gelu"``) quantised per token group -- ``per_token_group_quant_fp8`` of it
    (tileops/quant_fp8.py:83; dtype ``torch.float8_e4m3fn``, the default) or
    ``per_token_group_quant_int8`` (tileops/quant_int8.py:109; dtype ``torch.int8``) -- in one
    kernel that never writes the activation. Returns the same ``(q, scales)`` as the two ops
    run one after the other, bit for bit: the input of a W8A8 down projection straight from
    the gate and up halves of the gate_up output."""
    op = "act_and_mul_group_quant"
    _validate_fused(a, b, None, op)
    if act not in ("silu", "gelu"):
        raise ValueError(f"{op}: act must be 'silu' or 'gelu' (got {act!r})")
    dtype = torch.float8_e4m3fn if dtype is None else dtype
    if dtype not in (torch.float8_e4m3fn, torch.int8):
        raise TypeError(f"{op}: codes must be torch.float8_e4m3fn or torch.int8 (got {dtype})")
    if dtype == torch.int8 and (use_ue8m0 or column_major_scales):
        raise ValueError(f"{op}: use_ue8m0 and column_major_scales are FP8 options")
    _lib.ensure_device(a, op)
    if a.dtype not in _DTYPES:
        raise TypeError(f"{op}: unsupported dtype {a.dtype} (float32, float16 and bfloat16 are "
                        "supported)")
    if a.dim() == 0 or a.shape[-1] % group_size != 0:
        raise ValueError(f"the last dimension of `a` must be divisible by `group_size` "
                         f"{group_size}")
    if column_major_scales and a.dim() != 2:
        raise ValueError(f"{op}: column_major_scales needs 2-D inputs")
    cols = a.shape[-1]
    rows = a.numel() // cols if cols else 0
    lda, ldb = _row_stride(a), _row_stride(b)
    if lda is None:
        a, lda = a.contiguous(), cols
    if ldb is None:
        b, ldb = b.contiguous(), cols
    q = torch.empty(a.shape, dtype=dtype, device=a.device)
    groups = cols // group_size
    s = torch.empty(*a.shape[:-1], groups, dtype=torch.float32, device=a.device)
    if a.numel():
        _lib.call("to_act_and_mul_group_quant", a.data_ptr(), b.data_ptr(),
                  _lib.DTYPE_CODES[a.dtype], rows, cols, lda, ldb, 0 if act == "silu" else 1,
                  group_size, eps, 1 if use_ue8m0 else 0, 1 if column_major_scales else 0,
                  _lib.DTYPE_CODES[dtype], q.data_ptr(), s.data_ptr(), _lib.stream_ptr())
    return q, s


def _refuse(op: str, name: str, t: torch.Tensor, dtype: torch.dtype,
            device: torch.device) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{op}: {name}.dtype={t.dtype} != x.dtype={dtype}")
    raise TypeError(f"{op}: all tensors must be on {device} ({name} is on {t.device})")


def _span(t: torch.Tensor) -> int:
    """Bytes from the first element of ``t`` to the end of its last."""
    if t.is_contiguous():
        return t.numel() * t.element_size()
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors share memory; column slices of the same rows do not."""
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + _span(a) <= pb or pb + _span(b) <= pa:
        return False
    la, lb = _row_stride(a), _row_stride(b)
    if la is not None and lb is not None and a.dim() > 1 and b.dim() > 1:
        pitch = la * a.element_size()
        if pitch == lb * b.element_size() and pitch > 0:
            off = (pb - pa) % pitch
            return (off < a.shape[-1] * a.element_size() or
                    off + b.shape[-1] * b.element_size() > pitch)
    return True


def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether element i of both is the same memory; a dimension of size 1 has any stride."""
    return a.data_ptr() == b.data_ptr() and all(
        n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def _refuse_overlap(op: str, name: str, out: torch.Tensor, same: tuple, others: tuple) -> None:
    """An output may be one of ``same``, in its layout, and shares memory with nothing else the
    kernel reads."""
    for t in same:
        if t is not None and t is not out and _overlap(out, t) and not _same_layout(out, t):
            raise ValueError(f"{op}: {name} partly overlaps an input it may only replace whole")
    for t in others:
        if t is not None and _overlap(out, t):
            raise ValueError(f"{op}: {name} overlaps an input")


def add_rms_norm_group_quant(x: torch.Tensor, weight: torch.Tensor, group_size: int,
                             residual: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                             dtype: Optional[torch.dtype] = None, quant_eps: float = 1e-10,
                             column_major_scales: bool = False, use_ue8m0: bool = False,
                             residual_out: Optional[torch.Tensor] = None):
    """Library extension (no reference counterpart): the residual's addition, a root-mean-square
    norm and the per-token-group quantiser in one kernel -- the input of a W8A8 linear straight
    from the residual stream:

        h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight        (over the last dimension)
        scale = max(max|y|, quant_eps) / qmax per group,  q = code(y / scale)

    ``dtype`` torch.float8_e4m3fn (default; qmax 448, optionally power-of-two scales) or
    torch.int8 (qmax 127); ``group_size`` divides the last dimension and may be all of it. All of
    it is fp32: unlike an unfused chain, y is not rounded to ``x.dtype`` before it is quantised.
    ``x``, ``weight`` (one per column) and ``residual`` share a dtype (float32, float16, bfloat16).

    Returns ``(q, scales)``, or ``(q, scales, h)`` with a residual, h rounded to ``x.dtype``:
    written to ``residual_out`` when given, which may be ``x`` or ``residual`` itself. A row with
    a NaN has NaN scales, e4m3 NaN codes and int8 zeros; a row of zeros has codes 0 and scales
    quant_eps / qmax (with ``eps`` 0 it is 0 / 0: NaN). The mean of squares is fp32: values beyond
    about 1e19 overflow it, and their row's codes become 0."""
    op = "add_rms_norm_group_quant"
    if x.dim() == 0 or weight.shape != x.shape[-1:]:
        raise ValueError(f"{op}: weight.shape={tuple(weight.shape)} does not match the last "
                         f"dimension of x {tuple(x.shape)}")
    cols = x.shape[-1]
    if group_size <= 0 or cols % group_size != 0:
        raise ValueError(f"{op}: the last dimension of `x` {cols} must be divisible by "
                         f"`group_size` {group_size}")
    if not (1e-35 <= quant_eps < 3e38) or not 0.0 <= eps < 3e38:
        raise ValueError(f"{op}: eps={eps} must be at least 0 and quant_eps={quant_eps} at least "
                         "1e-35 (a scale is a normal number)")
    if dtype is None:
        dtype = torch.float8_e4m3fn
    code = 4 if dtype == torch.float8_e4m3fn else 3
    if code == 3:
        if dtype != torch.int8:
            raise TypeError(f"{op}: codes must be torch.float8_e4m3fn or torch.int8 (got {dtype})")
        if use_ue8m0 or column_major_scales:
            raise ValueError(f"{op}: use_ue8m0 and column_major_scales are FP8 options")
    if column_major_scales and x.dim() != 2:
        raise ValueError(f"{op}: column_major_scales needs a 2-D input")
    xd, device = x.dtype, x.device
    if weight.dtype != xd or weight.device != device:
        _refuse(op, "weight", weight, xd, device)
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"{op}: residual.shape={tuple(residual.shape)} != "
                             f"x.shape={tuple(x.shape)}")
        if residual.dtype != xd or residual.device != device:
            _refuse(op, "residual", residual, xd, device)
    if residual_out is not None:
        if residual is None:
            raise ValueError(f"{op}: residual_out needs a residual")
        if residual_out.shape != x.shape:
            raise ValueError(f"{op}: residual_out.shape={tuple(residual_out.shape)} != "
                             f"x.shape={tuple(x.shape)}")
        if residual_out.dtype != xd or residual_out.device != device:
            _refuse(op, "residual_out", residual_out, xd, device)
        _refuse_overlap(op, "residual_out", residual_out, (x, residual), (weight,))
    idx = _lib.ensure_device(x, op)
    if xd not in _DTYPES:
        raise TypeError(f"{op}: unsupported dtype {xd} (float32, float16 and bfloat16 are "
                        "supported)")
    rows = x.numel() // cols if cols else 0
    ldx = ldr = ldh = cols
    if not x.is_contiguous():
        ldx = _row_stride(x)
        if ldx is None:
            x, ldx = x.contiguous(), cols
    q = torch.empty_like(x, dtype=dtype, memory_format=_ROWS)
    dst = None
    if residual is not None:
        if not residual.is_contiguous():
            ldr = _row_stride(residual)
            if ldr is None:
                residual, ldr = residual.contiguous(), cols
        if residual_out is not None:
            ldh = cols if residual_out.is_contiguous() else _row_stride(residual_out)
        if residual_out is None or ldh is None:
            dst, ldh = torch.empty_like(x, memory_format=_ROWS), cols
        else:
            dst = residual_out
    if not weight.is_contiguous():
        weight = weight.contiguous()
    s = torch.empty((*x.shape[:-1], cols // group_size), dtype=torch.float32, device=device)
    _lib.call("to_add_rms_norm_group_quant", x.data_ptr(), ldx, _lib.ptr(residual), ldr,
              weight.data_ptr(), _lib.DTYPE_CODES[xd], rows, cols, group_size, eps, quant_eps,
              1 if use_ue8m0 else 0, 1 if column_major_scales else 0, code, q.data_ptr(),
              s.data_ptr(), _lib.ptr(dst), ldh, _lib.stream_ptr(idx))
    if residual is None:
        return q, s
    if residual_out is not None and dst is not residual_out:
        residual_out.copy_(dst)
        dst = residual_out
    return q, s, dst


__all__ = ["act_and_mul_group_quant", "add_rms_norm_group_quant", "gelu_and_mul", "silu_and_mul"]
