"""A whole layer for up to 16 tokens in two kernels, and experts in 4 bits.

The ordinary pass over the experts is made of seven or eight launches around tiles of 64 rows and more; a decoding step's few rows wait
for these launches as long as for the weights.  Here the first kernel adds the residual, norms and computes the router's logits, and the
second chooses the experts, reads their weights (once per eight slots of an expert) and folds the result.  No reference counterpart.
"""
from __future__ import annotations

import torch

from moe_explore import _native
from moe_explore.expert_compute import routed_expert_compute
from moe_explore.functional.activation import is_glu
from moe_explore.functional.fp8 import _dense
from moe_explore.params import ErnieRouterParams, GroupedTopkRouterParams, Int4ExpertParams, MLPParams, TopkRouterParams
from moe_explore.router import nothing_watches
from moe_explore.routing_plan import device_status

_PLAIN = (torch.Tensor, torch.nn.Parameter)
_HALF = (torch.bfloat16, torch.float16)


def _router_options(rp, dtype):
    """(score function, normalize, groups, open groups, best, scale, bias) of a router that the kernels know, else None."""
    weight = rp.router_weight
    if type(rp) is TopkRouterParams:
        if weight.dtype is not dtype:
            return None
        return 0 if rp.softmax_before_topk else 2, 1 if rp.normalize_routing and rp.softmax_before_topk else 0, 1, 1, 1, 1.0, None
    if type(rp) is ErnieRouterParams:
        return (0, 2, 1, 1, 1, 1.0, rp.bias) if weight.dtype is torch.float32 else None
    if type(rp) is GroupedTopkRouterParams:
        if weight.dtype not in (dtype, torch.float32) or rp.score_function not in ("sigmoid", "softmax"):
            return None
        best = rp.group_best if rp.num_groups > 1 else 1
        return (1 if rp.score_function == "sigmoid" else 0, 1 if rp.normalize_routing else 0, rp.num_groups, rp.topk_groups, best,
                float(rp.scale), rp.bias)
    return None


def few_token_layer(input: torch.Tensor, params, residual=None, addend=None, norm=None):
    """Norm (``norm``, with ``residual`` added before it), router and experts of ``params`` for up to 16 tokens: the layer's output, or, with
    ``residual``, (output, ``input + residual``).  ``addend`` [T, d] is added by the fold.  None where the kernels do not serve: more
    tokens, a gradient, another device than the current one, something that watches the single ops, routers or sizes that they do not know.

    The logits are not rounded to 16 bits; the choice among them is the routers' own (of exact arithmetic for ``GroupedTopkRouterParams``),
    equal values are taken in ascending index.  An expert's rows are not rounded before the fold."""
    if residual is not None and norm is None:
        raise ValueError("residual is added by the layer's norm: norm is None")
    ep, rp = params.expert_params, params.router_params
    int4 = type(ep) is Int4ExpertParams
    if not int4 and type(ep) is not MLPParams or type(input) not in _PLAIN or input.dim() != 2 or not 0 < input.size(0) <= _native.FEW_TOKENS or \
            input.dtype not in _HALF or not hasattr(rp, "router_weight"):
        return None
    T, d = input.shape
    E, topk = params.num_experts, params.topk
    weights = (ep.up.data, ep.down.data) if int4 else (ep.weight1, ep.weight2)
    bias = getattr(rp, "bias", None)
    tensors = [t for t in (input, rp.router_weight, bias, residual, addend, None if norm is None else norm.weight, *weights) if t is not None]
    if any(type(t) not in _PLAIN or not t.is_cuda for t in tensors) or not nothing_watches(*tensors) or _native.needs_gradient(*tensors):
        return None
    options = _router_options(rp, input.dtype)
    act = None if ep.activation is None else str(ep.activation)
    if options is None or act not in _native.ACT_CODES or type(topk) is not int or rp.topk != topk or T * topk > _native.FEW_SLOTS or \
            E > _native.FEW_EXPERTS or options[2] > _native.FEW_GROUPS or rp.router_weight.shape != (d, E) or d % 8 != 0 or d > _native.FEW_ROUTED_COLUMNS or \
            not 0 < topk <= E // max(options[2], 1) * options[3] or options[2] < 1 or E % options[2] != 0 or not 0 < options[3] <= options[2]:
        return None
    if bias is not None and (bias.dtype is not torch.float32 or bias.shape != (E,)):
        return None
    if any(t is not None and (t.shape != input.shape or t.dtype is not input.dtype) for t in (residual, addend)):
        return None
    if norm is not None and (norm.weight.shape != (d,) or norm.weight.dtype not in (input.dtype, torch.float32)):
        return None
    p = _experts(ep, input.dtype, E, d, act)
    if p is None:
        return None
    score_function, p.normalize, p.num_groups, p.topk_groups, p.group_best, p.scale, _ = options
    p.score_function = score_function
    held = [_dense(rp.router_weight.detach()), None if bias is None else bias.detach().contiguous()]
    p.router_w, p.router_bias = held[0].data_ptr(), _native._ptr(held[1])
    p.router_dtype = _native.float_code(held[0].dtype)
    stream = None
    if norm is not None:
        held.append(_dense(norm.weight.detach()))
        p.norm_w, p.norm_dtype, p.eps = held[-1].data_ptr(), _native.float_code(held[-1].dtype), float(norm.eps)
        if residual is not None:
            held.append(_dense(residual.detach()))
            stream = torch.empty(T, d, dtype=input.dtype, device=input.device)
            p.residual, p.stream_out = held[-1].data_ptr(), stream.data_ptr()
    out = _launch(p, input, topk, addend, held)
    return out if residual is None else (out, stream)


def _experts(ep, dtype, E: int, d: int, act):
    """The pass with its experts filled in, or None where they do not fit."""
    p = _native.FewPass()
    gates = 2 if is_glu(act) else 1
    if type(ep) is Int4ExpertParams:
        up, down = ep.up, ep.down
        inter = up.n // gates
        if up.dtype is not dtype or down.dtype is not dtype or up.zeros != down.zeros or up.group != down.group or \
                (up.n, up.k, down.n, down.k) != (gates * inter, d, d, inter) or up.data.size(0) != E or down.data.size(0) != E:
            return None
        up.checked(1, "up")
        down.checked(1, "down")
        p.bits, p.group, p.zeros, p.w1, p.w2 = 4, up.group, up.zeros, up.data.data_ptr(), down.data.data_ptr()
    else:
        w1, w2 = ep.weight1, ep.weight2
        if w1.dim() != 3 or w2.dim() != 3 or w1.dtype is not dtype or w2.dtype is not dtype:
            return None
        inter = w2.size(1)
        if w1.shape != (E, d, gates * inter) or w2.shape != (E, inter, d) or not all(w.is_contiguous() and w.data_ptr() % 16 == 0 for w in (w1, w2)):
            return None
        p.bits, p.w1, p.w2 = 16, w1.data_ptr(), w2.data_ptr()
    if inter % 8 != 0 or not 0 < inter <= _native.FEW_COLUMNS:
        return None
    p.d, p.inter, p.num_experts, p.act, p.dtype = d, inter, E, _native.ACT_CODES[act], _native.dtype_code(dtype)
    return p


def _launch(p, x, topk: int, addend, held):
    T, d = x.shape
    x = _dense(x.detach())
    out = torch.empty(T, d, dtype=x.dtype, device=x.device)
    workspace = torch.empty(_native.few_workspace_bytes(T, d, p.inter, p.num_experts, topk), dtype=torch.uint8, device=x.device)
    if addend is not None:
        addend = _dense(addend.detach())
        p.addend = addend.data_ptr()
    p.num_tokens, p.topk, p.x, p.out = T, topk, x.data_ptr(), out.data_ptr()
    p.status = device_status(x.get_device()).data_ptr()
    p.workspace, p.workspace_bytes = workspace.data_ptr(), workspace.numel()
    _native.few_tokens(p)
    return out


def weights_pay_in_16_bits(tokens: int, topk: int, experts: int, elements: int) -> bool:
    """Whether a call is shorter with the weights (``elements`` per expert) brought to 16 bits once, and the 16-bit pass over them, than by the
    kernel for a few tokens, 16 at a time.

    A slice of 16 tokens takes 21 us and reads every expert that it hits (``hit`` of them where choices are even) in 0.135 us per million
    elements; 16 bits take 0.75 us per million elements of all experts, hit or not: written, read again.  Their launches take 90 us; 130
    keeps small experts' weights unrounded for six slices.  Measured on both sides (us, slices / 16 bits): 64 experts of 7168 x 2048, 8 slots, 96
    tokens 1902 / 2320, 128 2579 / 2335; 256 of 2048 x 768, 8 slots, 160 tokens 865 / 1006, 208 1129 / 1006; 256 of 2048 x 1024, 1 slot,
    97 tokens 211 / 979, 512 995 / 1250, 1024 1980 / 1312; 1024 of 1024 x 256, 1 slot, 97 tokens 198 / 470, 1024 1488 / 633; 8 of 4096 x 14336, 2
    slots, 64 tokens 807 / 1157, 96 1217 / 1162; 6 of 128 x 64, 2 slots, 96 tokens 158 / 91, 160 247 / 89."""
    at_once = min(_native.FEW_TOKENS, _native.FEW_SLOTS // topk)
    slices = -(-tokens // at_once)
    hit = experts * (1 - (1 - 1 / experts) ** (at_once * topk))
    millions = elements * 1e-6
    return slices * (21 + 0.135 * millions * hit) > 130 + 0.75 * millions * experts


def int4_experts_in_16_bits(params: Int4ExpertParams) -> MLPParams:
    """The experts in 16 bits, each weight rounded once: what ``int4_expert_compute`` makes for itself when there are many tokens, for callers
    that want to keep it for a while (four times the memory)."""
    params.up.checked(1, "up")
    params.down.checked(1, "down")
    act = None if params.activation is None else str(params.activation)
    with _native.on_device_of(params.up.data):
        made = []
        for w, gated in ((params.up, is_glu(act)), (params.down, False)):
            out = torch.empty(w.data.size(0), w.k, w.n, dtype=w.dtype, device=w.data.device)
            _native.int4_expand(w, gated, out)
            made.append(out)
    return MLPParams(*made, params.activation)


def int4_expert_compute(x, scores, indices, params: Int4ExpertParams, addend=None) -> torch.Tensor:
    """out[t] = sum_s scores[t, s] * (act(x[t] @ up[e]^T) @ down[e]^T) with e = indices[t, s], the weights in 4 bits.  ``x`` [T, d] in the type
    of their scales, ``scores`` (rounded to that type) and ``indices`` (int64) [T, k]; slots with an expert id out of range add nothing (and
    are reported by the status word).  ``addend`` [T, d] is added by the fold.  For serving: no gradients.  Tokens go through the kernel
    for a few, 16 at a time, or, where that takes less time (``weights_pay_in_16_bits``: from some 100 tokens on where 16 tokens hit most
    experts, much later where they hit few), all through ``routed_expert_compute`` with the weights brought to 16 bits first: rounded
    there, and as much memory as 16-bit experts take for the time of the call.  ``params.expand`` = False keeps to the first, True to the
    second."""
    params.up.checked(1, "up")
    params.down.checked(1, "down")
    _native.require_cuda(x, scores, indices, addend)
    act = None if params.activation is None else str(params.activation)
    if act not in _native.ACT_CODES:
        raise ValueError(f"Unsupported activation: {act!r}")
    if x.dtype is not params.up.dtype:
        raise TypeError(f"rows are in the type of the scales, {params.up.dtype}, got {x.dtype}")
    if x.dim() != 2 or indices.dim() != 2 or indices.dtype is not torch.int64 or indices.size(0) != x.size(0) or scores.shape != indices.shape:
        raise ValueError("x is [tokens, d], indices (int64) and scores are [tokens, k]")
    if any(t.device != x.device for t in (scores, indices, params.up.data, params.down.data) + (() if addend is None else (addend,))):
        raise ValueError("all tensors lie on the device of the input")
    if addend is not None and (addend.shape != x.shape or addend.dtype is not x.dtype):
        raise ValueError("addend is like the result")
    _native.refuse_tracing()
    if _native.needs_gradient(x, scores, addend):
        raise RuntimeError("experts in 4 bits have no backward pass: call this under torch.no_grad(), or train 16-bit experts")
    T, topk = indices.shape
    E = params.up.data.size(0)
    if _experts(params, x.dtype, E, x.size(1), act) is None or not 0 < topk <= _native.FEW_SLOTS or not 0 < E <= _native.FEW_EXPERTS:
        raise ValueError(f"these experts do not fit together or are more than the kernel takes (1024 experts, 256 slots): input {tuple(x.shape)}, up "
                         f"[{params.up.n}, {params.up.k}], down [{params.down.n}, {params.down.k}] for {act!r}, {E} experts, {topk} slots")
    with _native.on_device_of(x):
        ids, scores = indices.contiguous(), scores.detach().to(x.dtype).contiguous()
        expand = params.expand
        if expand is None:
            expand = weights_pay_in_16_bits(T, topk, E, params.up.n * params.up.k + params.down.n * params.down.k)
        if expand and T > 0:
            experts = int4_experts_in_16_bits(params)
            with torch.no_grad():
                return routed_expert_compute(x, scores, experts.weight1, experts.weight2, ids, E, topk, act, addend=addend)
        outs = []
        at_once = min(_native.FEW_TOKENS, _native.FEW_SLOTS // topk)
        for t in range(0, T, at_once):
            part = slice(t, t + at_once)
            p = _experts(params, x.dtype, E, x.size(1), act)
            p.expert_idx, p.scores = ids[part].data_ptr(), scores[part].data_ptr()
            outs.append(_launch(p, x[part], topk, None if addend is None else addend[part], (ids, scores)))
        if not outs:
            return torch.empty(0, x.size(1), dtype=x.dtype, device=x.device)
        return outs[0] if len(outs) == 1 else torch.cat(outs)
