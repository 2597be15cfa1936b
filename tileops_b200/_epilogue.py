"""Argument checks shared by the products with bias, activation and residual in their epilogue
(``gemm_bias_act``, ``w8a8_block_int8_matmul_bias_act``, ``w8a8_block_fp8_matmul_bias_act``)."""

from __future__ import annotations

from typing import Optional

import torch

from .fused import _row_stride

ACT_CODES = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


def check(op: str, shape: tuple, n: int, dtype: torch.dtype, device: torch.device,
          bias: Optional[torch.Tensor], act: Optional[str], residual: Optional[torch.Tensor],
          out: Optional[torch.Tensor]) -> int:
    """Checks the epilogue's operands against an output of ``shape`` (last dimension ``n``) and
    returns the activation's code. Raised before any device work."""
    if act not in ACT_CODES:
        raise ValueError(f"{op}: act must be None, 'relu', 'silu' or 'gelu' (got {act!r})")
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"{op}: bias.shape={tuple(bias.shape)} != ({n},)")
    for name, t in (("residual", residual), ("out", out)):
        if t is not None and tuple(t.shape) != tuple(shape):
            raise ValueError(f"{op}: {name}.shape={tuple(t.shape)} != {tuple(shape)}")
    for name, t in (("bias", bias), ("residual", residual), ("out", out)):
        if t is None:
            continue
        if t.dtype != dtype:
            raise TypeError(f"{op}: {name}.dtype={t.dtype} != output dtype {dtype}")
        if t.device != device:
            raise TypeError(f"{op}: all tensors must be on {device} ({name} is on {t.device})")
    return ACT_CODES[act]


def prepare(shape: tuple, n: int, dtype: torch.dtype, device: torch.device,
            bias: Optional[torch.Tensor], residual: Optional[torch.Tensor],
            out: Optional[torch.Tensor]):
    """``(bias, residual, ldr, dst, ldc)``: the tensors the kernel reads and writes, rows strided
    as they are where their last dimension is contiguous, copied otherwise. ``dst`` is ``out`` or,
    where the kernel cannot write that in place, a fresh tensor to copy into it (finish)."""
    if bias is not None and n > 1 and bias.stride(0) != 1:
        bias = bias.contiguous()
    ldr = 0
    if residual is not None:
        ldr = _row_stride(residual)
        if ldr is None:
            residual, ldr = residual.contiguous(), n
    ldc = None if out is None else _row_stride(out)
    if ldc is None:
        return bias, residual, ldr, torch.empty(shape, dtype=dtype, device=device), n
    return bias, residual, ldr, out, ldc


def finish(dst: torch.Tensor, out: Optional[torch.Tensor]) -> torch.Tensor:
    if out is not None and dst is not out:
        out.copy_(dst)
        return out
    return dst


__all__ = ["ACT_CODES", "check", "finish", "prepare"]
