"""Root-mean-square norm with the residual's addition, in 16 bits (differentiable) and in 8 bits.

``h = x + residual`` (rounded to the rows' dtype: the stream as the next layer reads it), ``y = h / sqrt(mean(h^2) + eps) *
weight``.  No reference counterpart (its layer begins behind the norm).
"""
from __future__ import annotations

import torch

from moe_explore import _native
from moe_explore.functional.fp8 import BLOCK, DTYPE, Fp8Rows


def _checked(x, weight, residual):
    _native.require_cuda(x, weight, residual)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"rms_norm takes bf16 or fp16 rows, got {x.dtype}")
    if x.dim() < 1 or weight.shape != x.shape[-1:] or weight.dtype not in (x.dtype, torch.float32) or weight.device != x.device:
        raise ValueError(f"weight is [{x.size(-1) if x.dim() else 0}] in the rows' dtype or fp32, on their device")
    if residual is not None and (residual.shape != x.shape or residual.dtype is not x.dtype or residual.device != x.device):
        raise ValueError("residual is like x")


def _rows(x):
    """[..., d] as rows [R, d] that the kernels can read: dense columns, 16-byte aligned rows."""
    if x.dim() == 2 and x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x   # (a multiple of 8 columns is checked behind; a single row's stride, whatever it is, is not looked at)
    x = x.reshape(-1, x.size(-1))
    if x.stride(1) != 1 or x.size(0) != 1 and x.stride(0) % 8 != 0 or x.data_ptr() % 16 != 0:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _aligned(weight):
    weight = weight.contiguous()
    return weight if weight.data_ptr() % 16 == 0 else weight.clone()


def _forward(x, weight, residual, eps, with_rstd):
    """(y, h or None, 1 / root mean square of the rows or None)"""
    rows = _rows(x)
    y = torch.empty(rows.shape, dtype=x.dtype, device=x.device)
    h = None if residual is None else torch.empty_like(y)
    rstd = torch.empty(rows.size(0), dtype=torch.float32, device=x.device) if with_rstd else None
    _native.rms_norm(rows, None if residual is None else _rows(residual), _aligned(weight), eps, h=h, y=y, rstd=rstd)
    return _like(y, x), None if h is None else _like(h, x), rstd


def _like(rows, x):
    return rows if x.dim() == 2 else rows.view(x.shape)


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, rstd = _forward(x, weight, residual, eps, any(ctx.needs_input_grad))
        ctx.set_materialize_grads(False)
        ctx.has_residual = residual is not None
        if residual is None:
            ctx.save_for_backward(x, weight, rstd)
            return y
        ctx.save_for_backward(h, weight, rstd)
        return y, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:   # only the sum was used
            return dh, None, dh if ctx.has_residual else None, None
        with _native.on_device_of(h):
            dx, dw = _native.rms_norm_backward(_rows(dy).contiguous(), None if dh is None else _rows(dh).contiguous(), _rows(h),
                                               _aligned(weight), rstd)
        dx = _like(dx, h)
        return dx, dw, dx if ctx.has_residual else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor = None):
    """``y`` like ``x`` [..., d]; with ``residual``: (y, x + residual).  ``weight`` [d] in the rows' dtype or fp32.  Differentiable in
    all three; d a multiple of 8."""
    _checked(x, weight, residual)
    _native.refuse_tracing()
    with _native.on_device_of(x):
        if not _native.needs_gradient(x, weight, residual):
            y, h, _ = _forward(x, weight, residual, float(eps), False)
            return y if residual is None else (y, h)
        return _RMSNorm.apply(x, weight, residual, float(eps))


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor = None, with_rows: bool = False):
    """The norm's result in 8 bits (``Fp8Rows``), for the 8-bit products of a serving pass: ``rows``, then, with ``with_rows``, the
    same result in 16 bits (what a router reads), then, with ``residual``, ``x + residual``.  No gradient; d a multiple of 16."""
    _checked(x, weight, residual)
    _native.refuse_tracing()
    if _native.needs_gradient(x, weight, residual):
        raise RuntimeError("rms_norm_fp8 has no backward pass: call it under torch.no_grad(), or train with rms_norm")
    d = x.size(-1)
    if d % 16 != 0:
        raise ValueError(f"8-bit rows have a multiple of 16 columns, got {d}")
    with _native.on_device_of(x):
        rows = _rows(x)
        num_rows, device = rows.size(0), x.device
        q = torch.empty(num_rows, d, dtype=DTYPE, device=device)
        scales = torch.empty(num_rows, -(-d // BLOCK), dtype=torch.float32, device=device)
        y = torch.empty_like(rows, memory_format=torch.contiguous_format) if with_rows else None
        h = torch.empty_like(rows, memory_format=torch.contiguous_format) if residual is not None else None
        _native.rms_norm(rows, None if residual is None else _rows(residual), _aligned(weight), float(eps), h=h, y=y, q=q, scales=scales)
    if y is None and h is None:
        return Fp8Rows(q, scales, x.dtype)
    out = (Fp8Rows(q, scales, x.dtype),)
    if y is not None:
        out += (_like(y, x),)
    return out if h is None else out + (_like(h, x),)
