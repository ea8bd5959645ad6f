"""The top-k mixture-of-experts layer.

``topk_moe_forward`` keeps the reference signature (src/moe_explore/functional/topk_moe.py:10-64)
and is differentiable with respect to the input, the router weight and both expert weight
tensors.  ``topk_moe_torch`` restates the reference's per-expert torch loop
(functional/topk_moe.py:67-102) with out-of-place ops so that autograd works; it is a
torch-on-the-same-device cross-check, not a fallback of ``topk_moe_forward``.
"""
from __future__ import annotations

import torch

from moe_explore.expert_compute import (dense_expert, fp8_expert_compute, inference_pass, routed_expert_compute, routed_layer,
                                        router_and_experts_at_once, router_joins_the_pass)
from moe_explore.few_tokens import few_token_layer, int4_expert_compute
from moe_explore.functional.activation import activation
from moe_explore.functional.fp8 import Fp8Rows
from moe_explore.functional.rms_norm import rms_norm, rms_norm_fp8
from moe_explore.params import Fp8ExpertParams, Int4ExpertParams, MLPParams, MOEParams, TopkRouterParams
from moe_explore.router import fused_topk_router, router


def _shared_expert(input: torch.Tensor, shared) -> torch.Tensor:
    """The shared-expert branch (functional/topk_moe.py:56-62): ``h = act(input @ up_weight) @ down_weight`` followed
    by ``h.sum(0)``.  With 3-D weights -- ``up_weight`` [S, d, I or 2I], ``down_weight`` [S, I, d], S shared experts
    -- ``sum(0)`` adds the S experts' outputs per token; that case runs on the grouped-GEMM kernels as a top-S layer
    in which every token is routed to every shared expert with weight one (differentiable like the routed experts).
    With 2-D weights the reference's ``sum(0)`` runs over the TOKENS and the resulting [d] vector is broadcast onto
    every row; that literal behaviour is kept, in torch ops."""
    up, down = shared.up_weight, shared.down_weight
    if up.dim() == 3:
        num_shared = up.size(0)
        T = input.size(0)
        if num_shared == 1 and T > 0 and input.dim() == 2 and down.dim() == 3 and down.size(0) == 1:
            return dense_expert(input, up, down, shared.activation)
        indices = torch.arange(num_shared, device=input.device, dtype=torch.int64).repeat(T, 1)
        ones = torch.ones(T, num_shared, dtype=input.dtype, device=input.device)
        return routed_expert_compute(input, ones, up, down, indices, num_shared, num_shared, shared.activation)
    h = input @ up
    h = activation(h, shared.activation)
    h = h @ down
    return h.sum(0)


def topk_moe_forward(input: torch.Tensor, params: MOEParams, autotune_mode=None, *, fused_router: bool = False,
                     gather_in_gemm=None, fused_combine: bool = False, residual: torch.Tensor = None, save_fp8: bool = False,
                     few_tokens: bool = False):
    """The layer (functional/topk_moe.py:10-64).  ``autotune_mode`` is accepted and ignored.  Keyword-only additions:
    ``fused_router`` runs the router tail in one kernel with its own declared tie rule (see
    ``moe_explore.router.fused_topk_router``); ``gather_in_gemm`` / ``fused_combine`` as in ``expert_compute``; ``save_fp8`` as in
    ``routed_expert_compute``: a training pass keeps its experts' un-activated product in 8 bits and nothing else of their rows.

    With ``params.norm_params`` the layer begins with its norm: router, experts and shared expert see ``rms_norm(input)``, or, with
    ``residual``, ``rms_norm(input + residual)``, and the result is the pair (layer's output, ``input + residual``) that the next
    layer's norm takes.  Experts in 8 bits (``Fp8ExpertParams``) serve without gradients: the norm then gives their rows in 8 bits at
    once, and the router reads its 16-bit result.

    ``few_tokens``: where there are at most 16 tokens and no gradient is wanted, the layer runs in two kernels (see
    ``moe_explore.few_tokens.few_token_layer``, also for what it does not take and leaves to the ordinary pass; a shared expert is a pass
    of its own, as ever).  Its logits are fp32 sums that are not rounded to 16 bits, so that tokens whose logits nearly agree may go to
    other experts than in the ordinary pass.  Experts in 4 bits (``Int4ExpertParams``) serve without gradients, with or without it."""
    norm = getattr(params, "norm_params", None)
    if norm is None:
        if residual is not None:
            raise ValueError("residual is added by the layer's norm: params.norm_params is None")
        return _layer(input, None, params, fused_router, gather_in_gemm, fused_combine, save_fp8, few_tokens)
    if few_tokens and getattr(params, "shared_expert_params", None) is None:
        done = few_token_layer(input, params, residual, None, norm)
        if done is not None:
            return done
    rows = stream = None
    if isinstance(params.expert_params, Fp8ExpertParams):
        rows, normed, *rest = rms_norm_fp8(input, norm.weight, norm.eps, residual, with_rows=True)
        stream = rest[0] if rest else None
    elif residual is None:
        normed = rms_norm(input, norm.weight, norm.eps)
    else:
        normed, stream = rms_norm(input, norm.weight, norm.eps, residual)
    out = _layer(normed, rows, params, fused_router, gather_in_gemm, fused_combine, save_fp8, few_tokens)
    return out if residual is None else (out, stream)


def _layer(input: torch.Tensor, rows: Fp8Rows, params: MOEParams, fused_router: bool, gather_in_gemm, fused_combine: bool,
           save_fp8: bool, few_tokens: bool) -> torch.Tensor:
    """Router, experts and shared expert; ``rows``: the input in 8 bits where it is there already."""
    ep: MLPParams = params.expert_params
    shared = getattr(params, "shared_expert_params", None)
    shared_out = None if shared is None else _shared_expert(input, shared)
    # a [T, d] shared branch is added by the fold of the routed experts; the fused fold has no such place (experts in 8 or 4 bits
    # have no fused fold), and 2-D shared weights give a broadcast vector
    in_fold = not fused_combine or isinstance(ep, (Fp8ExpertParams, Int4ExpertParams))
    addend = shared_out if shared_out is not None and shared.up_weight.dim() == 3 and in_fold else None
    out = few_token_layer(input, params, None, addend) if few_tokens else None
    if out is not None:
        pass
    elif isinstance(ep, Int4ExpertParams):
        if fused_router and isinstance(params.router_params, TopkRouterParams):
            scores, indices = fused_topk_router(input, params.router_params)
        else:
            scores, indices = router(input, params.router_params)
        out = int4_expert_compute(input, scores, indices, ep, addend=addend)
    elif isinstance(ep, Fp8ExpertParams):
        if fused_router and isinstance(params.router_params, TopkRouterParams):
            scores, indices = fused_topk_router(input, params.router_params)
        else:
            scores, indices = router(input, params.router_params)
        out = fp8_expert_compute(input if rows is None else rows, scores, indices, ep, addend=addend)
    elif not save_fp8 and not fused_router and router_joins_the_pass(input, params.router_params, params.num_experts, params.topk):
        out = routed_layer(input, params.router_params, ep.weight1, ep.weight2, params.num_experts, ep.activation,
                           gather_in_gemm=gather_in_gemm, addend=addend)
    elif router_and_experts_at_once(input, params.router_params, ep.weight1, ep.weight2, params.num_experts, params.topk, addend):
        out = inference_pass(input, params.router_params, ep.weight1, ep.weight2, params.num_experts, params.topk, ep.activation,
                             gather_in_gemm=gather_in_gemm, fused_combine=fused_combine, addend=addend, fused_router=fused_router)
    else:
        if fused_router and isinstance(params.router_params, TopkRouterParams):
            scores, indices = fused_topk_router(input, params.router_params)
        else:
            scores, indices = router(input, params.router_params)
        out = routed_expert_compute(input, scores, ep.weight1, ep.weight2, indices, params.num_experts, params.topk,
                                    ep.activation, gather_in_gemm=gather_in_gemm, fused_combine=fused_combine, addend=addend,
                                    save_fp8=save_fp8)
    if shared_out is not None and addend is None:
        out = out + shared_out
    return out


def topk_moe_torch(input: torch.Tensor, params: MOEParams, autotune_mode=None) -> torch.Tensor:
    assert getattr(params, "norm_params", None) is None, "the torch form begins behind the norm"
    ep: MLPParams = params.expert_params
    scores, indices = router(input, params.router_params)
    flat_scores = scores.reshape(-1, 1)
    flat_experts = indices.reshape(-1)
    order = torch.sort(flat_experts, stable=True).indices
    counts = torch.bincount(flat_experts, minlength=params.num_experts)
    ends = counts.cumsum(0).tolist()
    out = torch.zeros_like(input)
    start = 0
    for expert_id, end in enumerate(ends):
        if end == start:
            continue
        rows = order[start:end]
        tok = rows // params.topk
        h = activation(input[tok] @ ep.weight1[expert_id], ep.activation)
        y = (h @ ep.weight2[expert_id]) * flat_scores[rows]
        out = out.index_add(0, tok, y)
        start = end
    return out
