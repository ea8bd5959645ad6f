"""Matrices in 8 bits -- e4m3 values with one fp32 scale per block of 128 -- and their products, for serving.

Rows have a scale per row and 128 columns, weights one per 128 x 128 block and lie as [N, K] (K contiguous, as checkpoints store a
linear layer).  ``scale = max(max |v|, 2^-80) / 448`` and ``q = v / scale``, to nearest even; ``quantize_rows`` (and the experts'
dispatch) round the quotient once to fp32 before, results that are made in fp32 (the norm's, the activated products) by one unit
of fp32 more.  Nothing here has a backward pass: a product that is asked for a gradient, of rows, weights or scales, raises
``RuntimeError``.  No reference counterpart.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from moe_explore import _native
from moe_explore.functional.activation import Activation, is_glu

BLOCK = 128
TOP = 448.0            # largest e4m3 value
LEAST = 2.0 ** -80     # smallest block maximum a scale is made of
DTYPE = torch.float8_e4m3fn


def blocks(n: int) -> int:
    return -(-n // BLOCK)


@dataclass
class Fp8Rows:
    """Rows in 8 bits: row r, column c is ``data[r, c] * scales[r, c // 128]``."""
    data: torch.Tensor     # float8_e4m3fn [R, K]
    scales: torch.Tensor   # fp32 [R, ceil(K / 128)]
    dtype: torch.dtype = torch.bfloat16   # 16-bit type of the products

    def checked(self) -> "Fp8Rows":
        _native.require_cuda(self.data, self.scales)
        if self.data.dtype is not DTYPE or self.data.dim() != 2 or self.scales.dtype is not torch.float32 or \
                self.scales.shape != (self.data.size(0), blocks(self.data.size(1))) or self.scales.device != self.data.device:
            raise ValueError("8-bit rows are float8_e4m3fn [R, K] with fp32 scales [R, ceil(K / 128)] on one device, got "
                             f"{self.data.dtype} {tuple(self.data.shape)}, {self.scales.dtype} {tuple(self.scales.shape)}")
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"products of 8-bit rows are bf16 or fp16, got {self.dtype}")
        return self


@dataclass
class Fp8Weight:
    """Weights in 8 bits: element [..., n, k] is ``data[..., n, k] * scales[..., n // 128, k // 128]``."""
    data: torch.Tensor     # float8_e4m3fn [..., N, K]
    scales: torch.Tensor   # fp32 [..., ceil(N / 128), ceil(K / 128)]

    def checked(self, dims: int, what: str) -> "Fp8Weight":
        _native.require_cuda(self.data, self.scales)
        want = (*self.data.shape[:-2], blocks(self.data.size(-2)), blocks(self.data.size(-1))) if self.data.dim() == dims else None
        if self.data.dtype is not DTYPE or self.scales.dtype is not torch.float32 or tuple(self.scales.shape) != want or \
                self.scales.device != self.data.device:
            raise ValueError(f"{what} is float8_e4m3fn with {dims} axes [..., N, K] and fp32 scales [..., ceil(N / 128), ceil(K / 128)] "
                             f"on one device, got {self.data.dtype} {tuple(self.data.shape)}, {self.scales.dtype} "
                             f"{tuple(self.scales.shape)}")
        return self


def _dense(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """16-bit rows [R, K] in 8 bits; K a multiple of 16."""
    _native.require_cuda(x)
    if x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"quantize_rows takes bf16 or fp16 [R, K], got {x.dtype} {tuple(x.shape)}")
    _native.refuse_tracing()
    if _native.needs_gradient(x):
        raise RuntimeError("8-bit rows have no backward pass: call this under torch.no_grad()")
    with _native.on_device_of(x):
        x = _dense(x.detach())
        q = torch.empty(x.shape, dtype=DTYPE, device=x.device)
        scales = torch.empty(x.size(0), blocks(x.size(1)), dtype=torch.float32, device=x.device)
        _native.f8_quantize_rows(x, q, scales)
    return Fp8Rows(q, scales, x.dtype)


def quantize_weight(weight: torch.Tensor) -> Fp8Weight:
    """Weights [..., N, K] (16 or 32 bits) in 8 bits, detached.  Torch operations in fp32: done once, when a model is loaded."""
    w = weight.detach().float()
    n, k = w.shape[-2:]
    w = torch.nn.functional.pad(w, (0, blocks(k) * BLOCK - k, 0, blocks(n) * BLOCK - n))
    w = w.unflatten(-2, (blocks(n), BLOCK)).unflatten(-1, (blocks(k), BLOCK))   # [..., nb, 128, kb, 128]
    most = w.abs().amax((-3, -1), keepdim=True).clamp_min(LEAST)
    q = (w * (TOP / 512.0) / most * 512.0).clamp(-TOP, TOP).to(DTYPE)
    q = q.flatten(-2).flatten(-3, -2)[..., :n, :k].contiguous()
    return Fp8Weight(q, (most[..., :, 0, :, 0] / TOP).contiguous())


def quantize_experts(params):
    """``Fp8ExpertParams`` of 16-bit expert parameters: ``MLPParams`` (for gated activations with gate and up columns interleaved),
    ``GLUParams`` or ``GLUInterleavedParams``."""
    from moe_explore.params import Fp8ExpertParams, GLUInterleavedParams, GLUParams, MLPParams

    if isinstance(params, GLUParams):
        up, down = torch.stack((params.gate_weight, params.up_weight), 1), params.down_weight     # [E, 2, d, I]
    elif isinstance(params, (MLPParams, GLUInterleavedParams)):
        first, down = (params.weight1, params.weight2) if isinstance(params, MLPParams) else (params.interleaved_weight, params.down_weight)
        gates = 2 if is_glu(params.activation) else 1
        up = first.unflatten(-1, (-1, gates)).permute(0, 3, 1, 2)
    else:
        raise ValueError(f"Unsupported expert parameters: {type(params)}")
    # matrix by matrix: the fp32 copies of a large layer would not fit
    def all_of(w):
        parts = [quantize_weight(m) for m in w]
        return Fp8Weight(torch.stack([p.data.view(torch.uint8) for p in parts]).view(DTYPE), torch.stack([p.scales for p in parts]))
    return Fp8ExpertParams(all_of(up.transpose(-1, -2)), all_of(down.transpose(-1, -2)), Activation(params.activation))


def fp8_matmul(rows: Fp8Rows, weight: Fp8Weight) -> torch.Tensor:
    """``rows @ weight^T`` [R, N] in ``rows.dtype``; ``weight`` [N, K] or [1, N, K].  K a multiple of 16, N of 8."""
    if weight.data.dim() == 2:
        weight = Fp8Weight(weight.data[None], weight.scales[None])
    return fp8_rows_gemm(rows, weight, None, None, False, False, rows.data.size(0), 1, None)


@functools.lru_cache(maxsize=256)
def _maps_layout(num_rows: int, num_experts: int):
    """(byte offsets of pad_offsets, mtile_expert, tile_pairs, num_mtiles; int32 words)."""
    tiles = _native.padded_rows_bound(num_rows, num_experts) // _native.TILE_M
    offsets, words = [], 0
    for n in (num_experts + 1, tiles, tiles + num_experts + 1, 4):
        offsets.append(4 * words)
        words += (n + 3) // 4 * 4
    return tuple(offsets), words


def fp8_rows_gemm(rows: Fp8Rows, weight: Fp8Weight, group_indices, permute_indices, gather: bool, scatter: bool, num_rows: int, topk: int,
                  act) -> torch.Tensor:
    """What ``m_grouped_gemm`` does for 8-bit rows; without ``group_indices`` the rows are those of one expert."""
    from moe_explore.routing_plan import device_status

    rows.checked()
    weight.checked(3, "weight")
    E, n, k = weight.data.shape
    if rows.data.size(1) != k or rows.data.device != weight.data.device:
        raise ValueError(f"rows of {rows.data.size(1)} columns on {rows.data.device}, weights of {k} on {weight.data.device}")
    if group_indices is None and E != 1:
        raise ValueError(f"weight [N, K] or [1, N, K] is expected, got {E} matrices")
    if is_glu(act) or act not in _native.ACT_CODES:
        raise ValueError(f"products of 8-bit rows take no or an element-wise activation, got {act!r} "
                         "(gated experts: moe_explore.expert_compute.fp8_expert_compute)")
    _native.refuse_tracing()
    if _native.needs_gradient(rows.data, rows.scales, weight.data, weight.scales):
        raise RuntimeError("products in 8 bits have no backward pass, of rows, weights or scales: call this under torch.no_grad()")
    device = rows.data.device
    with _native.on_device_of(rows.data):
        out = torch.empty(num_rows, n, dtype=rows.dtype, device=device)
        if num_rows == 0:
            return out
        x, xs, w, ws = _dense(rows.data), rows.scales.contiguous(), _dense(weight.data), weight.scales.contiguous()
        p = _native.F8RowsPass(num_rows, x.size(0), E, k, n, topk if gather else 1, _native.ACT_CODES[act], _native.dtype_code(rows.dtype),
                               bool(gather), bool(scatter), x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), out.data_ptr())
        p.status = device_status(rows.data.get_device()).data_ptr()
        steps = [(_native.ROWS_GEMM, "f8_gemm:rows", 1)]
        if group_indices is not None:
            offsets, words = _maps_layout(num_rows, E)
            maps = torch.empty(words, dtype=torch.int32, device=device)
            p.group_indices = group_indices.data_ptr()
            p.pad_offsets, p.mtile_expert, p.tile_pairs, p.num_mtiles = (maps.data_ptr() + o for o in offsets)
            steps.insert(0, (_native.ROWS_LAYOUT, "routing", 1))
        if permute_indices is not None:
            p.perm = permute_indices.data_ptr()
        if gather:
            gathered = torch.empty(num_rows, k, dtype=DTYPE, device=device)
            gathered_scales = torch.empty(num_rows, blocks(k), dtype=torch.float32, device=device)
            p.gathered, p.gathered_scales = gathered.data_ptr(), gathered_scales.data_ptr()
            steps.insert(-1, (_native.ROWS_GATHER, "rows:f8", 1))
        _native.run_pass("moe_f8_rows_gemm", p, steps, num_rows)
    return out
