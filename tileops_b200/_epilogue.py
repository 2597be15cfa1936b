"""Argument checks shared by the products with bias, activation and residual in their epilogue
(``gemm_bias_act``, ``w8a8_block_int8_matmul_bias_act``, ``w8a8_block_fp8_matmul_bias_act``).

A decode step makes several such calls per layer on kernels of a few microseconds, so the common
case (contiguous operands) does nothing but compare."""

from __future__ import annotations

from typing import Optional

import torch

from .fused import _refuse_overlap, _row_stride

ACT_CODES = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


def _refuse(op: str, name: str, t: torch.Tensor, dtype: torch.dtype, device: torch.device) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{op}: {name}.dtype={t.dtype} != output dtype {dtype}")
    raise TypeError(f"{op}: all tensors must be on {device} ({name} is on {t.device})")


def check(op: str, shape: tuple, n: int, dtype: torch.dtype, device: torch.device,
          bias: Optional[torch.Tensor], act: Optional[str], residual: Optional[torch.Tensor],
          out: Optional[torch.Tensor], reads: tuple) -> int:
    """Checks the epilogue's operands against an output of ``shape`` (last dimension ``n``) and
    returns the activation's code; ``reads``: the product's operands, which ``out`` must not
    overlap. Raised before any device work."""
    try:
        code = ACT_CODES[act]
    except (KeyError, TypeError):
        code = None
    if code is None:
        raise ValueError(f"{op}: act must be None, 'relu', 'silu' or 'gelu' (got {act!r})")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"{op}: bias.shape={tuple(bias.shape)} != ({n},)")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"{op}: residual.shape={tuple(residual.shape)} != {tuple(shape)}")
    if out is not None and out.shape != shape:
        raise ValueError(f"{op}: out.shape={tuple(out.shape)} != {tuple(shape)}")
    if bias is not None and (bias.dtype != dtype or bias.device != device):
        _refuse(op, "bias", bias, dtype, device)
    if residual is not None and (residual.dtype != dtype or residual.device != device):
        _refuse(op, "residual", residual, dtype, device)
    if out is not None and (out.dtype != dtype or out.device != device):
        _refuse(op, "out", out, dtype, device)
    if out is not None:
        _refuse_overlap(op, "out", out, (residual,), (*reads, bias))
    return code


def prepare(shape: tuple, n: int, like: torch.Tensor, dtype: torch.dtype,
            bias: Optional[torch.Tensor], residual: Optional[torch.Tensor],
            out: Optional[torch.Tensor]):
    """``(bias, residual, ldr, dst, ldc)``: the tensors the kernel reads and writes, rows strided
    as they are where their last dimension is contiguous, copied otherwise. ``dst`` is ``out`` or,
    where the kernel cannot write that in place, a fresh tensor to copy into it (finish)."""
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    ldr = n
    if residual is not None and not residual.is_contiguous():
        ldr = _row_stride(residual)
        if ldr is None:
            residual, ldr = residual.contiguous(), n
    if out is not None:
        ldc = n if out.is_contiguous() else _row_stride(out)
        if ldc is not None:
            return bias, residual, ldr, out, ldc
    return bias, residual, ldr, like.new_empty(shape, dtype=dtype), n


def padded(rows: int, row_bytes: int, address: int, pitch: int) -> int:
    """Bytes of the aligned copy of an operand, 0 if its rows are 16-byte aligned already; the
    operands' sum is what the library's workspace queries return."""
    return rows * ((row_bytes + 127) // 128 * 128) if (address | pitch) & 15 else 0


def copies(nbytes: int, like: torch.Tensor) -> torch.Tensor:
    """Scratch for aligned copies of operands, allocated for this call alone: it can be as large as
    the weights."""
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device)


def finish(dst: torch.Tensor, out: Optional[torch.Tensor]) -> torch.Tensor:
    if out is not None and dst is not out:
        out.copy_(dst)
        return out
    return dst


__all__ = ["ACT_CODES", "check", "copies", "finish", "padded", "prepare"]
