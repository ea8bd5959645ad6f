"""Parameter bundles of the MoE layer.

Field names and order follow the reference dataclasses (src/moe_explore/params.py:6-59) so
that code constructing them positionally keeps working.  ``MOEParams`` additionally accepts
an optional ``shared_expert_params`` (the reference reads that attribute in
functional/topk_moe.py:56 although its dataclass does not declare it).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from moe_explore.functional.activation import Activation
from moe_explore.functional.fp8 import Fp8Weight
from moe_explore.functional.int4 import Int4Weight


@dataclass
class FFNParams:
    """Base of the expert feed-forward parameter bundles."""


@dataclass
class MLPParams(FFNParams):
    """Two-matrix expert: ``weight1`` [E, d, I] (or [E, d, 2I] interleaved gate/up for *glu),
    ``weight2`` [E, I, d]."""
    weight1: torch.Tensor
    weight2: torch.Tensor
    activation: Activation


@dataclass
class GLUParams(FFNParams):
    """Gated expert with separate gate / up matrices [E, d, I] and down [E, I, d]."""
    gate_weight: torch.Tensor
    up_weight: torch.Tensor
    down_weight: torch.Tensor
    activation: Activation


@dataclass
class GLUInterleavedParams(FFNParams):
    """Gated expert with gate (even columns) and up (odd columns) interleaved in one [E, d, 2I] matrix."""
    interleaved_weight: torch.Tensor
    down_weight: torch.Tensor
    activation: Activation


@dataclass
class SharedExpertParams(FFNParams):
    """Shared expert(s) applied to every token: ``up_weight`` [S, d, I] (or [S, d, 2I] interleaved for *glu),
    ``down_weight`` [S, I, d].  The reference reads exactly these three attributes
    (functional/topk_moe.py:56-62) without declaring a type for them."""
    up_weight: torch.Tensor
    down_weight: torch.Tensor
    activation: Activation


@dataclass
class Fp8ExpertParams(FFNParams):
    """Experts in 8 bits, for serving (``moe_explore.functional.fp8.quantize_experts`` makes them of 16-bit ones): ``up`` [E, 2, I, d]
    (gate, up) for swiglu / geglu, else [E, 1, I, d]; ``down`` [E, d, I].  No reference counterpart."""
    up: Fp8Weight
    down: Fp8Weight
    activation: Activation


@dataclass
class Int4ExpertParams(FFNParams):
    """Experts in 4 bits, for serving (``moe_explore.functional.int4.pack_experts_int4`` and ``quantize_experts_int4`` make them): ``up``
    [E, 2I, d] with eight rows of the gate and eight of the up matrix in turn for swiglu / geglu, else [E, I, d]; ``down`` [E, d, I].
    ``expand``: whether calls bring the weights to 16 bits first, which takes a 16-bit layer's memory for the time of the call: None where that
    is quicker (many tokens), False never, True always.  No reference counterpart."""
    up: Int4Weight
    down: Int4Weight
    activation: Activation
    expand: Optional[bool] = None


@dataclass
class RMSNormParams:
    """Root-mean-square norm in front of the layer (``moe_explore.functional.rms_norm``)."""
    weight: torch.Tensor   # [d], in the rows' dtype or fp32
    eps: float = 1e-6


@dataclass
class RouterParams:
    """Base of the router parameter bundles."""


@dataclass
class TopkRouterParams(RouterParams):
    router_weight: torch.Tensor  # [d, E]
    topk: int
    softmax_before_topk: bool = True
    normalize_routing: bool = False


@dataclass
class ErnieRouterParams(RouterParams):
    router_weight: torch.Tensor  # [d, E], fp32
    bias: torch.Tensor           # [E], fp32, added to the probabilities for selection only
    topk: int


@dataclass
class GroupedTopkRouterParams(RouterParams):
    """Sigmoid or softmax scores, a bias that balances the load (added for the selection only), experts in ``num_groups``
    equal groups of which the ``topk_groups`` best stay open (a group's score: the sum of its best ``group_best``
    biased scores, 1 or 2), top-k inside them, weights renormalised and scaled.  No reference counterpart."""
    router_weight: torch.Tensor           # [d, E]; fp32: the logits are computed in fp32
    topk: int
    bias: Optional[torch.Tensor] = None   # [E], fp32
    num_groups: int = 1
    topk_groups: int = 1
    group_best: int = 2
    score_function: str = "sigmoid"       # or "softmax"
    normalize_routing: bool = True
    scale: float = 1.0


@dataclass
class MOEParams:
    router_params: RouterParams
    expert_params: FFNParams
    num_experts: int
    topk: int
    shared_expert_params: Optional[FFNParams] = None
    norm_params: Optional["RMSNormParams"] = None   # the layer's own norm in front of router and experts


@dataclass
class ExpertMatmulParams:
    tokens: torch.Tensor
    weight: torch.Tensor
    group_indices: torch.Tensor
    token_to_group_indices: torch.Tensor
    scales: Optional[torch.Tensor]


def interleave_gate_up(gate_weight: torch.Tensor, up_weight: torch.Tensor) -> torch.Tensor:
    """[E, d, I] gate and up matrices -> one [E, d, 2I] matrix, gate in even columns, up in odd
    columns: the layout ``activation(x, "swiglu")`` expects (functional/activation.py:17-25)."""
    assert gate_weight.shape == up_weight.shape
    return torch.stack((gate_weight, up_weight), dim=-1).reshape(*gate_weight.shape[:-1], -1).contiguous()
