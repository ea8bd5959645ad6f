"""Activations that keep their input in 8 bits for the backward pass: half the memory of 16 bits, or a third of what a gated
activation's input and result take.

The result is computed from the 16-bit input.  Kept are e4m3 values with one fp32 scale per row and 128 columns (the form of
``moe_explore.functional.fp8.quantize_rows``); the gradient is the activation's at these values.  No reference counterpart.
"""
from __future__ import annotations

import torch

from moe_explore import _native
from moe_explore.functional.activation import is_glu
from moe_explore.functional.fp8 import DTYPE, _dense, blocks


def kept_columns(columns: int) -> int:
    """Columns of the 8-bit rows that keep ``columns``: rows are 16-byte aligned."""
    return (columns + 15) // 16 * 16


class _ActivationFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, act):
        z = _dense(x.reshape(-1, x.size(-1)))
        rows, columns = z.shape
        h = torch.empty(rows, columns // 2 if is_glu(act) else columns, dtype=x.dtype, device=x.device)
        q = torch.empty(rows, kept_columns(columns), dtype=DTYPE, device=x.device)
        scales = torch.empty(rows, blocks(columns), dtype=torch.float32, device=x.device)
        _native.act_f8_forward(z, h, q, scales, act)
        ctx.save_for_backward(q, scales)
        ctx.act, ctx.shape = act, x.shape
        return h.view(*x.shape[:-1], h.size(1))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, scales = ctx.saved_tensors
        with _native.on_device_of(q):
            dh = _dense(grad.reshape(-1, grad.size(-1)))
            dz = torch.empty(dh.size(0), ctx.shape[-1], dtype=grad.dtype, device=grad.device)
            _native.act_f8_backward(q, scales, dh, dz, ctx.act)
        return dz.view(ctx.shape), None


def activation_fp8(x: torch.Tensor, act) -> torch.Tensor:
    """``activation(x, act)`` of 16-bit ``x`` [..., columns] (gated: gate and up columns in turn, the result has half as many) that
    keeps ``x`` in 8 bits for its gradient.  The result has a multiple of 8 columns."""
    _native.require_cuda(x)
    act = None if act is None else str(act)
    if act not in _native.ACT_CODES:
        raise ValueError(f"Unsupported activation: {act!r}")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"activation_fp8 takes bf16 or fp16, got {x.dtype}")
    per_column = 2 if is_glu(act) else 1
    if x.dim() < 1 or x.size(-1) == 0 or x.size(-1) % (8 * per_column) != 0:
        raise ValueError(f"columns come in multiples of {8 * per_column} for {act!r}, got {tuple(x.shape)}")
    _native.refuse_tracing()
    with _native.on_device_of(x):
        if _native.needs_gradient(x):
            return _ActivationFp8.apply(x, act)
        z = _dense(x.reshape(-1, x.size(-1)))
        h = torch.empty(z.size(0), z.size(1) // per_column, dtype=x.dtype, device=x.device)
        _native.act_f8_forward(z, h, None, None, act)
        return h.view(*x.shape[:-1], h.size(1))
