"""Weights in 4 bits -- values of 0 to 15 with a 16-bit scale, and where wanted a zero point, per row and group of 32, 64 or 128
columns -- and their products with a few 16-bit rows, for serving.

Element [n, k] of a weight [N, K] (K contiguous, as checkpoints store a linear layer) is ``(value - zero) * scale``; without zero points
zero is 8.  Products multiply the exact ``value - zero`` and add in fp32, group by group, times the scale.  The values are laid out once for
the kernels (``pack_int4``): tiles of 16 rows, cut into steps of 128 columns.  Nothing here has a backward pass.  No reference counterpart.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from moe_explore import _native
from moe_explore.functional.activation import is_glu
from moe_explore.functional.fp8 import _dense

TILE = 16      # rows
STEP = 128     # columns
GROUPS = (32, 64, 128)


def _up(n: int, of: int) -> int:
    return -(-n // of)


@dataclass
class Int4Weight:
    """Weights [..., n, k] in 4 bits, laid out by ``pack_int4``."""
    data: torch.Tensor     # uint8 [..., tiles, steps, bytes of a block]: 1024 of values, then scales, then zeros
    n: int
    k: int
    group: int
    dtype: torch.dtype     # of the scales, and of the rows: bf16 or fp16
    zeros: bool            # whether there are zero points

    @property
    def per_step(self) -> int:
        return STEP // self.group

    @property
    def block(self) -> int:
        return 1024 + TILE * self.per_step * (3 if self.zeros else 2)

    def checked(self, dims: int, what: str) -> "Int4Weight":
        """``dims``: axes in front of the matrix."""
        data = self.data
        _native.require_cuda(data)
        if self.group not in GROUPS or data.dim() != dims + 3 or data.dtype is not torch.uint8 or self.dtype not in (torch.bfloat16, torch.float16) or \
                data.shape[dims:] != (_up(self.n, TILE), _up(self.k, STEP), self.block):
            raise ValueError(f"{what} is an Int4Weight of pack_int4 with {dims} axes in front of the matrix, got {data.dtype} {tuple(data.shape)} for "
                             f"[{self.n}, {self.k}] in groups of {self.group} with scales in {self.dtype}")
        if not data.is_contiguous() or data.data_ptr() % 16 != 0:
            raise ValueError(f"{what}: the data of an Int4Weight are contiguous and 16-byte aligned, as pack_int4 makes them")
        return self

    def unpack(self):
        """(values uint8 [..., N, K / 2] two per byte, scales [..., N, groups], zeros or None): what ``pack_int4`` was given."""
        lead, tiles, steps, n = self.data.shape[:-3], self.data.size(-3), self.data.size(-2), TILE * self.per_step
        words = self.data[..., :1024].reshape(*lead, tiles, steps, 2, 8, 4, 4, 4)   # half, row, t, i, byte
        b0, b1, b2, b3 = words.unbind(-1)
        four = torch.stack(((b0 & 15) | (b2 << 4), (b0 >> 4) | (b2 & 240), (b1 & 15) | (b3 << 4), (b1 >> 4) | (b3 & 240)), -1)
        d = len(lead)
        rows = four.permute(*range(d), d, d + 2, d + 3, d + 1, d + 5, d + 4, d + 6).reshape(*lead, tiles * TILE, steps * STEP // 2)
        scales = self.data[..., 1024:1024 + 2 * n].contiguous().view(self.dtype)
        zeros = self.data[..., 1024 + 2 * n:] if self.zeros else None
        groups = _up(self.k, self.group)

        def flat(t):
            if t is None:
                return None
            t = t.reshape(*lead, tiles, steps, TILE, self.per_step).transpose(-3, -2)
            return t.reshape(*lead, tiles * TILE, steps * self.per_step)[..., :self.n, :groups].contiguous()
        return rows[..., :self.n, :self.k // 2].contiguous(), flat(scales), flat(zeros)

    def dequantize(self) -> torch.Tensor:
        """fp32 [..., N, K]."""
        values, scales, zeros = self.unpack()
        wide = lambda t: t.float().repeat_interleave(self.group, -1)[..., :self.k]
        whole = torch.stack((values & 15, values >> 4), -1).flatten(-2).float()
        return (whole - (8.0 if zeros is None else wide(zeros))) * wide(scales)


def pack_int4(values: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor = None, *, group: int = 128) -> Int4Weight:
    """``values`` uint8 [..., N, K / 2], two columns per byte, the even one in the low half; ``scales`` (bf16 or fp16) and ``zeros`` (uint8,
    0 to 15) [..., N, ceil(K / group)].  N and K multiples of 8.  Done once, when a model is loaded."""
    if group not in GROUPS:
        raise ValueError(f"groups are of 32, 64 or 128 columns, got {group}")
    if values.dim() < 2 or values.dtype is not torch.uint8:
        raise ValueError(f"values are uint8 [..., N, K / 2], got {values.dtype} {tuple(values.shape)}")
    *lead, n, half = values.shape
    k = 2 * half
    if n == 0 or k == 0 or n % 8 != 0 or k % 8 != 0:
        raise ValueError(f"N and K are multiples of 8, got {n} and {k}")
    want = (*lead, n, _up(k, group))
    if scales.dtype not in (torch.bfloat16, torch.float16) or tuple(scales.shape) != want or scales.device != values.device:
        raise ValueError(f"scales are bf16 or fp16 {want} on the device of the values, got {scales.dtype} {tuple(scales.shape)}")
    if zeros is not None and (zeros.dtype is not torch.uint8 or tuple(zeros.shape) != want or zeros.device != values.device):
        raise ValueError(f"zeros are uint8 {want} on the device of the values, got {zeros.dtype} {tuple(zeros.shape)}")
    if zeros is not None and bool((zeros > 15).any()):
        raise ValueError(f"zeros are 0 to 15, got {int(zeros.max())}")
    tiles, steps, per_step, d = _up(n, TILE), _up(k, STEP), STEP // group, len(lead)
    pad = torch.nn.functional.pad
    p = pad(values.detach(), (0, steps * STEP // 2 - half, 0, tiles * TILE - n))
    p = p.reshape(*lead, tiles, 2, 8, steps, 4, 4, 4)                               # half, row, step, i, t, byte
    p = p.permute(*range(d), d, d + 3, d + 1, d + 2, d + 5, d + 4, d + 6)           # tile, step, half, row, t, i, byte
    p0, p1, p2, p3 = p.unbind(-1)
    data = torch.stack(((p0 & 15) | (p1 << 4), (p2 & 15) | (p3 << 4), (p0 >> 4) | (p1 & 240), (p2 >> 4) | (p3 & 240)), -1)

    def laid(t):
        t = pad(t.detach(), (0, steps * per_step - t.size(-1), 0, tiles * TILE - n))
        t = t.reshape(*lead, tiles, TILE, steps, per_step).transpose(-3, -2).contiguous()
        return t.view(torch.uint8).reshape(*lead, tiles, steps, -1)
    blocks = [data.reshape(*lead, tiles, steps, 1024), laid(scales)] + ([] if zeros is None else [laid(zeros)])
    return Int4Weight(torch.cat(blocks, -1), n, k, group, scales.dtype, zeros is not None)


def quantize_int4(weight: torch.Tensor, group: int = 128, zeros: bool = False, dtype: torch.dtype = None) -> Int4Weight:
    """Weights [..., N, K] (16 or 32 bits) in 4 bits, detached, scales in ``dtype`` (the weights', bf16 for fp32 ones): to nearest, with
    ``zeros`` over each group's range, else symmetrically.  Torch operations in fp32: done once, when a model is loaded."""
    values, scales, points = _quantized(weight, group, zeros, dtype)
    return pack_int4(values, scales, points, group=group)


def _quantized(weight, group, zeros, dtype):
    if group not in GROUPS:
        raise ValueError(f"groups are of 32, 64 or 128 columns, got {group}")
    dtype = dtype if dtype is not None else weight.dtype if weight.dtype in (torch.bfloat16, torch.float16) else torch.bfloat16
    w = weight.detach().float()
    k = w.size(-1)
    if w.dim() < 2 or k % 8 != 0 or w.size(-2) % 8 != 0:
        raise ValueError(f"weights are [..., N, K] with N and K multiples of 8, got {tuple(weight.shape)}")
    groups = _up(k, group)
    w = torch.nn.functional.pad(w, (0, groups * group - k)).unflatten(-1, (groups, group))
    least = float(torch.finfo(dtype).tiny)
    if zeros:
        low, high = w.amin(-1).clamp_max(0), w.amax(-1).clamp_min(0)
        scales = ((high - low) / 15).clamp_min(least).to(dtype)
        points = (-low / scales.float()).round().clamp(0, 15)
    else:
        scales = (w.abs().amax(-1) / 7).clamp_min(least).to(dtype)
        points = torch.full_like(scales, 8.0, dtype=torch.float32)
    q = ((w / scales.float()[..., None]).round() + points[..., None]).clamp(0, 15).to(torch.uint8).flatten(-2)[..., :k]
    return q[..., 0::2] | (q[..., 1::2] << 4), scales, points.to(torch.uint8) if zeros else None


def pack_experts_int4(up, down, activation, *, group: int = 128):
    """``Int4ExpertParams`` of (values, scales, zeros or None) triples as ``pack_int4`` takes them: ``up`` [E, 2, I, d] (gate, up) for gated
    activations, else [E, 1, I, d]; ``down`` [E, d, I]."""
    from moe_explore.params import Int4ExpertParams

    activation = None if activation is None else str(activation)
    if activation not in _native.ACT_CODES:
        raise ValueError(f"Unsupported activation: {activation!r}")
    gates = 2 if is_glu(activation) else 1
    if up[0].dim() != 4 or up[0].size(1) != gates or down[0].dim() != 3 or up[0].size(2) % 8 != 0:
        raise ValueError(f"up is [E, {gates}, I, d] and down [E, d, I] for {activation!r} with I a multiple of 8, got {tuple(up[0].shape)}, "
                         f"{tuple(down[0].shape)} (values: two columns per byte)")

    def rows(t):   # eight rows of the gate, eight of the up matrix in turn: a tile holds both halves of its eight results
        if t is None:
            return None
        e, _, inter, cols = t.shape
        return t.view(e, gates, inter // 8, 8, cols).transpose(1, 2).reshape(e, gates * inter, cols)
    return Int4ExpertParams(pack_int4(*(rows(t) for t in up), group=group), pack_int4(*down, group=group),
                            activation)


def quantize_experts_int4(params, group: int = 128, zeros: bool = False):
    """``Int4ExpertParams`` of 16-bit expert parameters: ``MLPParams`` (for gated activations with gate and up columns interleaved),
    ``GLUParams`` or ``GLUInterleavedParams``."""
    from moe_explore.params import GLUInterleavedParams, GLUParams, MLPParams

    if isinstance(params, GLUParams):
        up, down = torch.stack((params.gate_weight, params.up_weight), 1), params.down_weight     # [E, 2, d, I]
    elif isinstance(params, (MLPParams, GLUInterleavedParams)):
        first, down = (params.weight1, params.weight2) if isinstance(params, MLPParams) else (params.interleaved_weight, params.down_weight)
        up = first.unflatten(-1, (-1, 2 if is_glu(params.activation) else 1)).permute(0, 3, 1, 2)
    else:
        raise ValueError(f"Unsupported expert parameters: {type(params)}")

    def all_of(w):   # matrix by matrix: the fp32 copies of a large layer would not fit
        parts = [_quantized(m, group, zeros, None) for m in w]
        return tuple(None if p[0] is None else torch.stack(p) for p in zip(*parts))
    return pack_experts_int4(all_of(up.transpose(-1, -2)), all_of(down.transpose(-1, -2)), params.activation, group=group)


def int4_matmul(x: torch.Tensor, weight: Int4Weight) -> torch.Tensor:
    """``x @ weight^T`` [..., N] for a few rows ``x`` [..., K] in the type of the weight's scales (any number of rows is right; the kernel is
    made for up to 64: beyond, the weights are read again for every 64)."""
    weight.checked(0, "weight")
    _native.require_cuda(x)
    if x.dim() < 1 or x.size(-1) != weight.k or x.device != weight.data.device:
        raise ValueError(f"rows of {tuple(x.shape)} on {x.device}, weights [{weight.n}, {weight.k}] on {weight.data.device}")
    if x.dtype is not weight.dtype:
        raise TypeError(f"rows are in the type of the scales, {weight.dtype}, got {x.dtype}")
    _native.refuse_tracing()
    if _native.needs_gradient(x):
        raise RuntimeError("products with 4-bit weights have no backward pass: call this under torch.no_grad()")
    with _native.on_device_of(x):
        rows = _dense(x if x.dim() == 2 else x.reshape(-1, weight.k))
        out = x.new_empty((rows.size(0), weight.n))
        if rows.size(0) <= _native.INT4_ROWS:
            _native.int4_matmul(rows, weight, out)
        else:
            for part, to in zip(rows.split(_native.INT4_ROWS), out.split(_native.INT4_ROWS)):
                _native.int4_matmul(part, weight, to)
    return out if x.dim() == 2 else out.view(*x.shape[:-1], weight.n)
