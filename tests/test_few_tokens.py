"""The layer for a few tokens in two kernels, and experts in 4 bits, against the formulas in 64 bits; refusals and what is left to the
ordinary pass."""
import math

import pytest
import torch

from moe_explore.expert_compute import routed_expert_compute
from moe_explore.few_tokens import few_token_layer, int4_expert_compute, int4_experts_in_16_bits
from moe_explore.functional.int4 import pack_experts_int4, quantize_experts_int4
from moe_explore.functional.topk_moe import topk_moe_forward
from moe_explore.params import (ErnieRouterParams, GroupedTopkRouterParams, Int4ExpertParams, MLPParams, MOEParams, RMSNormParams,
                                SharedExpertParams, TopkRouterParams)
from moe_explore.routing_plan import device_status
from test_activation_fp8 import act64, gated
from test_int4 import raw, weight64

gpu = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_router(g, kind, d, E, k, dtype):
    w = 1.5 * d ** -0.5 * torch.randn(d, E, generator=g, device="cuda")
    bias = 0.1 * torch.randn(E, generator=g, device="cuda")
    if kind == "ernie":
        return ErnieRouterParams(w, bias, k)
    if kind.startswith("groups"):
        return GroupedTopkRouterParams(w if "fp32" in kind else w.to(dtype), k, bias=None if "plain" in kind else bias, num_groups=4, topk_groups=3,
                                       group_best=1 if "one" in kind else 2, score_function="softmax" if "softmax" in kind else "sigmoid",
                                       normalize_routing="raw" not in kind, scale=2.5)
    return TopkRouterParams(w.to(dtype), k, "after" not in kind, "norm" in kind)


def route64(rp, logits):
    """(weights, experts), best first, equal values by ascending index."""
    def best(v, n):
        return torch.sort(v, dim=-1, descending=True, stable=True).indices[:, :n]
    E, k = logits.size(1), rp.topk
    if isinstance(rp, TopkRouterParams):
        i = best(logits, k)
        if not rp.softmax_before_topk:
            return torch.softmax(logits.gather(1, i), -1), i
        w = torch.softmax(logits, -1).gather(1, i)
        return w / w.sum(-1, keepdim=True) if rp.normalize_routing else w, i
    if isinstance(rp, ErnieRouterParams):
        p = torch.softmax(logits, -1)
        i = best(p + rp.bias, k)
        w = p.gather(1, i)
        return w / w.sum(-1, keepdim=True).clamp_min(1e-12), i
    p = torch.sigmoid(logits) if rp.score_function == "sigmoid" else torch.softmax(logits, -1)
    key = p if rp.bias is None else p + rp.bias
    value = key.view(-1, rp.num_groups, E // rp.num_groups).topk(min(rp.group_best, E // rp.num_groups)).values.sum(-1)
    open_ = torch.zeros_like(value, dtype=torch.bool).scatter_(1, best(value, rp.topk_groups), True).repeat_interleave(E // rp.num_groups, 1)
    i = best(torch.where(open_, key, -math.inf), k)
    w = p.gather(1, i)
    return (w / w.sum(-1, keepdim=True) if rp.normalize_routing else w) * rp.scale, i


def experts64(x, weights, indices, w1, w2, act):
    """x [T, d], matrices [E, d, N] and [E, I, d] in 64 bits, gate and up columns in turn."""
    out = torch.zeros_like(x)
    for e in indices.unique().tolist():
        token, slot = (indices == e).nonzero(as_tuple=True)
        out.index_add_(0, token, weights[token, slot, None] * (act64(x[token] @ w1[e], act) @ w2[e]))
    return out


def make_experts(g, bits, E, d, inter, act, dtype, group=128, zeros=False):
    """(parameters, w1 and w2 in 64 bits as ``experts64`` takes them)"""
    gates = 2 if gated(act) else 1
    if bits == 16:
        w1 = (torch.randn(E, d, gates * inter, generator=g, device="cuda") * d ** -0.5).to(dtype)
        w2 = (torch.randn(E, inter, d, generator=g, device="cuda") * inter ** -0.5).to(dtype)
        return MLPParams(w1, w2, act), w1.double(), w2.double()
    up, down = raw(g, E, gates, inter, d, group=group, zeros=zeros, dtype=dtype), raw(g, E, d, inter, group=group, zeros=zeros, dtype=dtype)
    w1 = weight64(*up, group).permute(0, 3, 2, 1).reshape(E, d, inter * gates)
    return pack_experts_int4(up, down, act, group=group), w1, weight64(*down, group).mT


def near(got, want, dtype, roundings):
    """At the root of the mean square each rounding to 16 bits is off by eps / 2 / sqrt(3) at most, of the activated product, the result, and
    of the normed rows, which the gate and the up matrix both read; the factor sqrt(3) is left for the activation's slope and fp32 sums."""
    assert got.dtype is dtype and got.shape == want.shape
    return float((got.double() - want).norm()) <= roundings * torch.finfo(dtype).eps / 2 * float(want.norm()) + 1e-30


CASES = [
    # T, d, E, k, I, act, dtype, bits, group, zeros, router, norm
    (1, 64, 4, 1, 8, "swiglu", torch.bfloat16, 16, 128, False, "topk", False),
    (1, 2048, 60, 4, 1408, "swiglu", torch.bfloat16, 16, 128, False, "topk", True),
    (16, 512, 64, 8, 264, "swiglu", torch.bfloat16, 16, 128, False, "topk norm", False),
    (7, 776, 12, 3, 1544, "geglu", torch.float16, 16, 128, False, "topk after", True),
    (16, 136, 2, 2, 200, "gelu", torch.bfloat16, 16, 128, False, "topk after", False),
    (5, 264, 7, 2, 40, "silu", torch.float16, 16, 128, False, "ernie", True),
    (3, 8, 8, 8, 8, "approx_gelu", torch.bfloat16, 16, 128, False, "topk", False),
    (11, 256, 32, 4, 96, None, torch.bfloat16, 16, 128, False, "groups fp32", False),
    (1, 1024, 8, 2, 4096, "swiglu", torch.bfloat16, 4, 128, False, "topk after", True),
    (7, 776, 12, 3, 1544, "geglu", torch.float16, 4, 32, True, "topk", False),
    (16, 520, 64, 8, 136, "swiglu", torch.bfloat16, 4, 64, False, "groups fp32", True),
    (13, 384, 16, 4, 264, "silu", torch.bfloat16, 4, 64, True, "groups softmax one", False),
    (2, 72, 3, 2, 24, "gelu", torch.float16, 4, 32, False, "ernie", False),
    (16, 256, 2, 1, 512, "swiglu", torch.float16, 4, 128, True, "topk", True),
    (9, 2048, 128, 8, 256, "swiglu", torch.bfloat16, 4, 128, False, "groups plain raw", True),
    (4, 128, 512, 16, 64, "swiglu", torch.bfloat16, 16, 128, False, "groups fp32 raw", True),
]


@gpu
@pytest.mark.parametrize("T,d,E,k,inter,act,dtype,bits,group,zeros,kind,normed", CASES)
def test_layer(T, d, E, k, inter, act, dtype, bits, group, zeros, kind, normed, native):
    g = gen(T * d + E)
    rp = make_router(g, kind, d, E, k, dtype)
    experts, w1, w2 = make_experts(g, bits, E, d, inter, act, dtype, group, zeros)
    norm = RMSNormParams((1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dtype if T % 2 else torch.float32), 1e-5) if normed else None
    p = MOEParams(rp, experts, E, k, None, norm)
    x = torch.randn(T, d, generator=g, device="cuda").to(dtype)
    for residual in (None, torch.randn(T, d, generator=g, device="cuda").to(dtype)) if normed else (None,):
        h = x if residual is None else x + residual
        y = h.double()
        if normed:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * norm.weight.double()
        want = experts64(y, *route64(rp, y @ rp.router_weight.double()), w1, w2, act)
        with torch.no_grad():
            assert few_token_layer(x, p, residual, None, norm) is not None, "the kernels serve this"
            out = topk_moe_forward(x, p, residual=residual, few_tokens=True)
        if residual is not None:
            out, stream = out
            assert torch.equal(stream, h)
        assert near(out, want, dtype, 4 if normed else 2)
    native.check_status(device_status(0))


@gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_whole_numbers_are_exact(bits, native):
    """Sums of small whole numbers without an activation: every step is exact in whatever order and share, so every index is right."""
    g = gen(4)
    for T, d, E, k, inter in ((1, 264, 4, 2, 200), (16, 136, 5, 5, 72), (6, 520, 3, 2, 1032)):
        ints = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda")
        sparse = lambda t, share: t * (torch.rand(t.shape, generator=g, device="cuda") < share)
        w1, w2 = sparse(ints(-1, 2, E, d, inter), 0.05), sparse(ints(-1, 2, E, inter, d), 0.05)
        if bits == 16:
            experts = MLPParams(w1.half(), w2.half(), None)
        else:
            def four(w):   # [E, K, N] -> values + 8 of [E, N, K]
                v = (w.mT + 8).to(torch.uint8)
                return v[..., 0::2] | (v[..., 1::2] << 4), torch.ones(E, w.size(2), -(-w.size(1) // 32), device="cuda").half(), None
            up = four(w1)
            experts = pack_experts_int4(tuple(None if t is None else t[:, None] for t in up), four(w2), None, group=32)
        x = ints(-2, 3, T, d).half()
        indices = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)]).cuda()
        scores = torch.ones(T, k, device="cuda").half()
        want = experts64(x.double(), scores.double(), indices, w1.double(), w2.double(), None)
        assert float(want.abs().max()) < 2048
        if bits == 4:
            assert bool((int4_expert_compute(x, scores, indices, experts).double() == want).all())
        # the same choice by the layer's own router: a logit of 1 + slot for the chosen experts (one more column of x), weights a half or one
        wide = torch.zeros(T, d + 8, device="cuda").half()
        wide[:, :d] = x
        if T == 1:   # one token can be given any logits
            wide[0, d] = 1
            rw = torch.zeros(d + 8, E, device="cuda").half()
            rw[d, indices[0]] = 20.0
            w1w = torch.zeros(E, d + 8, inter, device="cuda")
            w1w[:, :d] = w1
            w2w = torch.zeros(E, inter, d + 8, device="cuda")
            w2w[:, :, :d] = w2
            if bits == 16:
                p = MOEParams(TopkRouterParams(rw, k, False), MLPParams(w1w.half(), w2w.half(), None), E, k)
                with torch.no_grad():
                    got = topk_moe_forward(wide, p, few_tokens=True)
                assert bool((got[:, :d].double() * k == want).all())


@gpu
def test_same_bits_in_any_company(native):
    """A token's result does not depend on the other tokens of the call as long as the work is shared out alike, nor on the call."""
    g = gen(8)
    experts, _, _ = make_experts(g, 4, 8, 256, 128, "swiglu", torch.bfloat16)
    x = torch.randn(16, 256, generator=g, device="cuda").bfloat16()
    indices = torch.arange(2, device="cuda").repeat(16, 1)
    scores = torch.full((16, 2), 0.5, device="cuda").bfloat16()
    whole = int4_expert_compute(x, scores, indices, experts)
    assert all(torch.equal(whole, int4_expert_compute(x, scores, indices, experts)) for _ in range(20))
    assert torch.equal(int4_expert_compute(x[:5], scores[:5], indices[:5], experts), whole[:5])
    many = int4_expert_compute(x.repeat(3, 1)[:41], scores.repeat(3, 1)[:41], indices.repeat(3, 1)[:41], experts)
    assert torch.equal(many, whole.repeat(3, 1)[:41])
    assert int4_expert_compute(x[:0], scores[:0], indices[:0], experts).shape == (0, 256)


@gpu
def test_equal_logits_duplicates_and_bad_experts(native):
    g = gen(9)
    d, E, inter = 128, 8, 64
    w16, w1, w2 = make_experts(g, 16, E, d, inter, "swiglu", torch.bfloat16)
    x = torch.randn(3, d, generator=g, device="cuda").bfloat16()
    rw = torch.zeros(d, E, device="cuda").bfloat16()        # all logits are equal: the lowest experts
    with torch.no_grad():
        out = topk_moe_forward(x, MOEParams(TopkRouterParams(rw, 3, False), w16, E, 3), few_tokens=True)
    want = experts64(x.double(), torch.full((3, 3), 1 / 3, device="cuda", dtype=torch.float64), torch.arange(3, device="cuda").repeat(3, 1), w1, w2, "swiglu")
    assert near(out, want, torch.bfloat16, 2)
    q, w1, w2 = make_experts(g, 4, E, d, inter, "swiglu", torch.bfloat16)
    x = torch.randn(16, d, generator=g, device="cuda").bfloat16()
    scores = torch.rand(16, 4, generator=g, device="cuda").bfloat16()
    twice = torch.zeros(16, 4, dtype=torch.int64, device="cuda")    # one expert four times for each of 16 tokens
    twice[3] = 5
    want = torch.zeros(16, d, dtype=torch.float64, device="cuda")
    for s in range(4):
        want += experts64(x.double(), scores[:, s:s + 1].double(), twice[:, s:s + 1], w1, w2, "swiglu")
    assert near(int4_expert_compute(x, scores, twice, q), want, torch.bfloat16, 2)
    native.check_status(device_status(0))
    bad = torch.randint(0, E, (16, 4), generator=g, device="cuda")
    bad[2, 1], bad[7, 0], bad[9] = -1, E, 1 << 40
    want = torch.zeros(16, d, dtype=torch.float64, device="cuda")
    for s in range(4):
        ok = (bad[:, s] >= 0) & (bad[:, s] < E)
        want[ok] += experts64(x[ok].double(), scores[ok, s:s + 1].double(), bad[ok, s:s + 1], w1, w2, "swiglu")
    out = int4_expert_compute(x, scores, bad, q)
    assert near(out, want, torch.bfloat16, 2) and not out[9].any()
    assert native.read_status(device_status(0), reset=True) == native.STATUS_BAD_EXPERT_ID


@gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_all_slots_on_few_experts(bits, native):
    """Every token to every expert, 16 rows each (two blocks of eight), 16 slots per token, and the deepest and the shallowest rows."""
    g = gen(20)
    for T, d, E, inter in ((16, 136, 16, 8), (9, 8, 3, 1032), (16, 1032, 2, 264)):
        experts, w1, w2 = make_experts(g, bits, E, d, inter, "swiglu", torch.bfloat16, 32)
        rp = make_router(g, "topk norm", d, E, E, torch.bfloat16)
        x = torch.randn(T, d, generator=g, device="cuda").bfloat16()
        with torch.no_grad():
            out = few_token_layer(x, MOEParams(rp, experts, E, E))
        y = x.double()
        assert near(out, experts64(y, *route64(rp, y @ rp.router_weight.double()), w1, w2, "swiglu"), torch.bfloat16, 2)
    native.check_status(device_status(0))


@gpu
@pytest.mark.parametrize("d,E,inter,act,dtype,group,zeros", [(136, 4, 72, "swiglu", torch.bfloat16, 32, True), (512, 8, 264, "geglu", torch.float16, 128, False),
                                                             (72, 3, 136, "gelu", torch.bfloat16, 64, True), (256, 5, 40, "silu", torch.float16, 64, False)])
def test_prompts_through_experts_in_4_bits(d, E, inter, act, dtype, group, zeros, native):
    """The weights in 16 bits are their values rounded once, in the 16-bit experts' layout; many tokens are the 16-bit pass on them, few tokens
    are near it: six roundings (gate and up weights, down weights, the activated product, an expert's row, the result)."""
    g = gen(d + E)
    q, w1, w2 = make_experts(g, 4, E, d, inter, act, dtype, group, zeros)
    wide = int4_experts_in_16_bits(q)
    assert wide.weight1.shape == w1.shape and wide.weight2.shape == w2.shape
    assert torch.equal(wide.weight1, w1.to(dtype)) and torch.equal(wide.weight2, w2.to(dtype))
    T, k = 300, 2
    x, addend = (torch.randn(T, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    indices = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)]).cuda()
    scores = torch.rand(T, k, generator=g, device="cuda").to(dtype)
    many = int4_expert_compute(x, scores, indices, q, addend=addend)
    with torch.no_grad():
        assert torch.equal(many, routed_expert_compute(x, scores, wide.weight1, wide.weight2, indices, E, k, act, addend=addend))
    want = experts64(x.double(), scores.double(), indices, w1, w2, act) + addend.double()
    assert near(many, want, dtype, 6)
    few = torch.cat([int4_expert_compute(x[t:t + 90], scores[t:t + 90], indices[t:t + 90], q, addend=addend[t:t + 90]) for t in range(0, T, 90)])
    assert near(few, want, dtype, 2)


@gpu
@pytest.mark.parametrize("T", [96, 97, 130])
@pytest.mark.parametrize("E", [1, 6])
def test_prompts_with_bad_experts_in_a_graph(T, E, native):
    """On both sides of the line: slots of no expert add nothing and are reported, and a graph follows its inputs."""
    g = gen(100 * T + E)
    d, inter, k = 128, 64, 2
    q, w1, w2 = make_experts(g, 4, E, d, inter, "swiglu", torch.bfloat16, 64, True)
    x = torch.randn(T, d, generator=g, device="cuda").bfloat16()
    scores = torch.rand(T, k, generator=g, device="cuda").bfloat16()
    indices = torch.randint(0, E, (T, k), generator=g, device="cuda")   # the same expert twice, too
    int4_expert_compute(x, scores, indices, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = int4_expert_compute(x, scores, indices, q)
    for bad in (False, True):
        x.copy_(torch.randn(T, d, generator=g, device="cuda"))
        if bad:
            indices[0], indices[5, 1], indices[T - 1, 0] = E, -1, E + 7
        graph.replay()
        eager = int4_expert_compute(x, scores, indices, q)
        assert torch.equal(out, eager)
        real = (indices >= 0) & (indices < E)
        want = sum(experts64(x.double(), (scores.double() * real)[:, s:s + 1], indices.clamp(0, E - 1)[:, s:s + 1], w1, w2, "swiglu") for s in range(k))
        assert near(eager, want, torch.bfloat16, 6)
        assert not bad or not eager[0].any()
        assert native.read_status(device_status(0), reset=True) == (native.STATUS_BAD_EXPERT_ID if bad else 0)


@gpu
def test_values_that_are_not_finite(native):
    """A token that holds NaN or an infinity spoils its own row only."""
    g = gen(10)
    d, E, k = 256, 16, 4
    experts, _, _ = make_experts(g, 16, E, d, 64, "swiglu", torch.bfloat16)
    p = MOEParams(make_router(g, "topk", d, E, k, torch.bfloat16), experts, E, k)
    x = torch.randn(6, d, generator=g, device="cuda").bfloat16()
    with torch.no_grad():
        clean = topk_moe_forward(x, p, few_tokens=True)
        x[1, 3], x[4, 200] = math.nan, math.inf
        out = topk_moe_forward(x, p, few_tokens=True)
    assert torch.isnan(out[1]).all() and not torch.isfinite(out[4]).any()
    rest = [0, 2, 3, 5]
    assert float((out[rest].float() - clean[rest].float()).abs().max()) <= 2 * 2.0 ** -8 * float(clean.float().abs().max())


@gpu
def test_large_rows_get_their_norm(native):
    """bf16 rows whose squares leave fp32."""
    d = 512
    experts, w1, w2 = make_experts(gen(1), 16, 4, d, 64, "swiglu", torch.bfloat16)
    norm = RMSNormParams(torch.ones(d, device="cuda"), 1e-6)
    p = MOEParams(make_router(gen(2), "topk after", d, 4, 2, torch.bfloat16), experts, 4, 2, None, norm)
    x = torch.randn(2, d, generator=gen(3), device="cuda").bfloat16()
    with torch.no_grad():
        a, b = topk_moe_forward(x * 2.0 ** 100, p, few_tokens=True), topk_moe_forward(x * 2.0 ** 90, p, few_tokens=True)
    assert torch.isfinite(a).all() and torch.equal(a, b)


@gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_serving_with_a_shared_expert_in_a_graph_and_on_two_streams(bits, native):
    """Layers that hand the stream on, captured together and replayed with other inputs while an eager call runs on another stream."""
    g = gen(11)
    d, E, k, inter = 256, 16, 4, 96
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")
    layers = []
    for i in range(3):
        experts, _, _ = make_experts(g, bits, E, d, inter, "swiglu", torch.bfloat16)
        sp = SharedExpertParams((new(1, d, 2 * inter) * d ** -0.5).bfloat16(), (new(1, inter, d) * inter ** -0.5).bfloat16(), "swiglu") if i == 1 else None
        layers.append(MOEParams(make_router(g, "groups fp32", d, E, k, torch.bfloat16), experts, E, k, sp, RMSNormParams((1 + 0.1 * new(d)).bfloat16())))

    def model(x, residual):
        for p in layers:
            x, residual = topk_moe_forward(x, p, residual=residual, few_tokens=True)
        return x, residual
    with torch.no_grad():
        x, residual = new(8, d).bfloat16(), new(8, d).bfloat16()
        other = new(5, d).bfloat16(), new(5, d).bfloat16()
        want = model(*other)
        model(x, residual)
        torch.cuda.synchronize()
        graphs, outs = [], []
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(model(x, residual))
        x.copy_(new(8, d))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            with torch.cuda.stream(side):
                got = model(*other)
            graphs[0].replay()
            graphs[1].replay()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        eager = model(x, residual)
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # the shared expert's branch is in it
        one = MOEParams(layers[1].router_params, layers[1].expert_params, E, k, layers[1].shared_expert_params)
        bare = MOEParams(layers[1].router_params, layers[1].expert_params, E, k)
        from moe_explore.expert_compute import dense_expert
        both = topk_moe_forward(x, one, few_tokens=True).float()
        sp = layers[1].shared_expert_params
        apart = topk_moe_forward(x, bare, few_tokens=True).float() + dense_expert(x, sp.up_weight, sp.down_weight, "swiglu").float()
        # three results rounded once each
        assert bool(((both - apart).abs() <= 3 * 2.0 ** -8 * (both.abs() + dense_expert(x, sp.up_weight, sp.down_weight, "swiglu").float().abs()) + 1e-6).all())
    native.check_status(device_status(0))


@gpu
def test_what_is_left_to_the_ordinary_pass(native):
    g = gen(12)
    d, E, k = 128, 8, 2
    experts, _, _ = make_experts(g, 16, E, d, 64, "swiglu", torch.bfloat16)
    p = MOEParams(make_router(g, "topk", d, E, k, torch.bfloat16), experts, E, k)
    x = torch.randn(17, d, generator=g, device="cuda").bfloat16()
    with torch.no_grad():
        assert few_token_layer(x, p) is None
        assert torch.equal(topk_moe_forward(x, p, few_tokens=True), topk_moe_forward(x, p))
        assert few_token_layer(x[:16].float(), p) is None and few_token_layer(x[:0], p) is None
        # rows that are neither dense nor aligned, weights that are not either
        part = torch.randn(4, d + 5, generator=g, device="cuda").bfloat16()[:, 3:3 + d]
        assert torch.equal(topk_moe_forward(part, p, few_tokens=True), topk_moe_forward(part.contiguous(), p, few_tokens=True))
        turned = MOEParams(p.router_params, MLPParams(experts.weight1.mT.contiguous().mT, experts.weight2, "swiglu"), E, k)
        assert few_token_layer(x[:4], turned) is None
        assert torch.equal(topk_moe_forward(x[:4], turned, few_tokens=True), topk_moe_forward(x[:4], turned))
    leaf = x[:4].clone().requires_grad_(True)
    y = topk_moe_forward(leaf, p, few_tokens=True)
    assert y.requires_grad and torch.equal(y, topk_moe_forward(leaf, p))
    q = MOEParams(p.router_params, quantize_experts_int4(experts, 32), E, k)
    with pytest.raises(RuntimeError, match="no backward"):
        topk_moe_forward(leaf, q, few_tokens=True)
    with torch.no_grad():   # 4 bits behind the ordinary router, more tokens than a pass takes
        from moe_explore.router import router
        out = topk_moe_forward(x, q)
        scores, indices = router(x, p.router_params)
        assert torch.equal(out, int4_expert_compute(x, scores, indices, q.expert_params))
        assert float((out.float() - topk_moe_forward(x, p).float()).norm() / topk_moe_forward(x, p).float().norm()) < 0.3


@gpu
def test_a_wait_that_runs_out_is_reported(native):
    """With a limit of one cycle some CTA gives up before the last one comes: the status word says so, and the next call is right."""
    g = gen(13)
    experts, _, _ = make_experts(g, 16, 8, 256, 512, "swiglu", torch.bfloat16)
    p = MOEParams(make_router(g, "topk", 256, 8, 2, torch.bfloat16), experts, 8, 2)
    x = torch.randn(4, 256, generator=g, device="cuda").bfloat16()
    with torch.no_grad():
        want = topk_moe_forward(x, p, few_tokens=True)
        native.set_wait_limit_cycles(1)
        try:
            topk_moe_forward(x, p, few_tokens=True)
        finally:
            native.set_wait_limit_cycles(0)
        with pytest.raises(native.MoeNativeError, match="bounded wait"):
            native.check_status(device_status(0))
        assert native.read_status(device_status(0), reset=True) == 6
        assert torch.equal(topk_moe_forward(x, p, few_tokens=True), want)


def marked_experts(E, rows, dtype=torch.bfloat16):
    """Experts that say who they are: for a row with a single one in it, expert e adds a one in column e; so a layer's result [T, max(rows, E)]
    holds every expert's weight in its column."""
    d = (max(rows, E) + 7) // 8 * 8
    w1, w2 = torch.zeros(E, d, 8, device="cuda", dtype=dtype), torch.zeros(E, 8, d, device="cuda", dtype=dtype)
    w1[:, :, 0] = 1
    w2[torch.arange(E), 0, torch.arange(E)] = 1
    return MLPParams(w1, w2, None), d


def weights_of(logits, rp, E):
    """The layer's weights [T, E] for these fp32 logits: row t is all zeros but for a one in column t, so its logits are row t of the router."""
    T = logits.size(0)
    experts, d = marked_experts(E, T)
    rp.router_weight = torch.zeros(d, E, device="cuda", dtype=torch.float32)
    rp.router_weight[:T] = logits
    p = MOEParams(rp, experts, E, rp.topk)
    with torch.no_grad():
        out = few_token_layer(torch.eye(T, d, device="cuda", dtype=torch.bfloat16), p)
    return out[:, :E]


def grouped(E, k, bias, groups=1, open_=1, best=2, function="sigmoid", normalize=False):
    return GroupedTopkRouterParams(None, k, bias=bias, num_groups=groups, topk_groups=open_, group_best=best, score_function=function,
                                   normalize_routing=normalize, scale=1.0)


def chosen(logits, rp):
    """Indices of the router's own kernel, and the weights in its 32-bit scores."""
    from moe_explore.router import grouped_topk_of_logits
    scores, indices = grouped_topk_of_logits(logits, rp, torch.float32)
    return torch.zeros_like(logits).scatter_(1, indices, scores), indices


def same_choice(logits, rp):
    """The weights are those of the experts that the router's kernel chooses: they agree to a rounding of 16 bits, the last bits of two
    exponentials in 32 (each within 2 units of 2^-23, their sum and the division), and steps of the smallest numbers of 16 bits."""
    want, _ = chosen(logits, rp)
    got = weights_of(logits, rp, logits.size(1)).float()
    assert bool(((got - want).abs() <= (2.0 ** -8 + 2.0 ** -19) * want + 2.0 ** -132).all())


@gpu
def test_the_choice_is_that_of_exact_arithmetic(native):
    """Values whose difference fp32 does not hold: sigmoids near one, tiny ones beside a bias, groups of such values."""
    E = 64
    low = torch.full((1, E), -3.0, device="cuda")
    zero = torch.zeros(E, device="cuda")
    near_one = low.clone()
    near_one[0, 7], near_one[0, 50] = 20.0, 25.0           # both sigmoids are 1 in fp32
    same_choice(near_one, grouped(E, 1, zero))
    assert weights_of(near_one, grouped(E, 1, zero), E).nonzero().tolist() == [[0, 50]]
    tiny = torch.full((1, E), -60.0, device="cuda")
    tiny[0, 9], tiny[0, 40] = -22.0, -19.0                 # sigmoids of 3e-10 and 6e-9 beside a bias of a half
    rp = grouped(E, 1, torch.full((E,), 0.5, device="cuda"))
    want, indices = chosen(tiny, rp)
    assert indices.tolist() == [[40]]
    assert weights_of(tiny, rp, E).nonzero().tolist() == [[0, 40]]
    for best in (1, 2):                                    # groups whose best sum to the same number in fp32
        both = low.clone()
        both[0, 3], both[0, 5], both[0, 57], both[0, 60] = 21.0, 22.0, 23.0, 22.5
        for bias in (None, zero):
            rp = grouped(E, 2, bias, groups=8, open_=1, best=best)
            assert sorted(chosen(both, rp)[1][0].tolist()) == [57, 60]
            assert weights_of(both, rp, E).nonzero().tolist() == [[0, 57], [0, 60]]
    soft = torch.full((1, E), -40.0, device="cuda")        # all but one share are 0 beside the bias
    soft[0, 0], soft[0, 11], soft[0, 33] = 30.0, -1.0, 4.0
    rp = grouped(E, 2, torch.full((E,), 1.0, device="cuda"), function="softmax")
    assert sorted(chosen(soft, rp)[1][0].tolist()) == [0, 33]
    assert weights_of(soft, rp, E).nonzero().tolist() == [[0, 0], [0, 33]]


@gpu
@pytest.mark.parametrize("function", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,groups,open_,best", [(64, 1, 1, 1), (64, 8, 3, 2), (256, 8, 4, 2), (256, 32, 5, 1), (768, 6, 2, 2)])
def test_the_choice_is_the_routers(function, E, groups, open_, best, native):
    """Sixteen tokens at a time, logits of every scale: coarse ones (equal values), wide ones (shares of 0 and 1), ordinary ones."""
    g = gen(E + groups)
    k = 8 if E // groups * open_ >= 8 else 4
    for scale in (0.25, 2.0, 12.0, 30.0):
        for coarse in (False, True):
            logits = scale * torch.randn(16, E, generator=g, device="cuda")
            if coarse:
                logits = (logits / scale * 8).round() * (scale / 8)
            for bias in (None, torch.zeros(E, device="cuda"), 0.1 * torch.randn(E, generator=g, device="cuda")):
                same_choice(logits, grouped(E, k, bias, groups, open_, best, function))
    native.check_status(device_status(0))


@gpu
def test_logits_that_are_not_finite(native):
    """NaN comes after minus infinity where the router is one of groups; where the softmax runs over the selected logits, it comes first, as for
    the ordinary router, and the row is NaN."""
    E = 16
    logits = torch.full((1, E), -math.inf, device="cuda")
    logits[0, 0], logits[0, 1], logits[0, 12] = math.nan, math.nan, 1.0
    for rp in (grouped(E, 3, None), grouped(E, 3, torch.zeros(E, device="cuda")), grouped(E, 3, None, groups=4, open_=2, best=1)):
        assert chosen(logits, rp)[1][0, 0] == 12 and not any(i in (0, 1) for i in chosen(logits, rp)[1][0].tolist())
        got = weights_of(logits, rp, E)
        assert torch.isfinite(got).all() and got.nonzero().tolist() == [[0, 12]]
    experts, d = marked_experts(E, 1)
    w = torch.zeros(d, E, device="cuda").bfloat16()
    w[0] = torch.arange(E, device="cuda")
    w[0, 3] = math.nan
    p = MOEParams(TopkRouterParams(w, 2, False), experts, E, 2)
    x = torch.eye(1, d, device="cuda").bfloat16()
    with torch.no_grad():
        assert torch.isnan(topk_moe_forward(x, p)).all() and torch.isnan(topk_moe_forward(x, p, few_tokens=True)).all()


@gpu
@pytest.mark.parametrize("weight_type", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [512, 2056])
def test_rows_near_the_end_of_bf16_get_their_norm(d, weight_type, native):
    """Rows whose products with the norm's weight, and with the router's, leave fp32 before they are scaled; large values in all of a row, in
    one stretch of it only, and none.  The ordinary layer is finite and near, too."""
    g = gen(d)
    E, k, inter = 20, 3, 64
    experts, w1, w2 = make_experts(g, 16, E, d, inter, "swiglu", torch.bfloat16)
    norm = RMSNormParams((4 + 4 * torch.rand(d, generator=g, device="cuda")).to(weight_type), 1e-6)
    rp = make_router(g, "groups fp32", d, E, k, torch.bfloat16)
    p = MOEParams(rp, experts, E, k, None, norm)
    x = torch.randn(8, d, generator=g, device="cuda").clamp(-3.5, 3.5)
    x[0] *= 2.0 ** 125
    x[1, d // 2:d // 2 + 5] *= 2.0 ** 125
    x[2] *= 2.0 ** 70
    x[3, -1] = 2.0 ** 127
    x[4, :8] *= 2.0 ** 60
    x[5] *= 2.0 ** -50
    x = x.bfloat16()
    residual = (0.25 * torch.randn(8, d, generator=g, device="cuda") * x.abs().amax(1, keepdim=True).clamp_max(2.0 ** 124)).bfloat16()
    for r in (None, residual):
        h = x if r is None else x + r
        assert torch.isfinite(h).all()
        y = h.double()
        y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * norm.weight.double()
        want = experts64(y, *route64(rp, y @ rp.router_weight.double()), w1, w2, "swiglu")
        with torch.no_grad():
            few = topk_moe_forward(x, p, residual=r, few_tokens=True)
            ordinary = topk_moe_forward(x, p, residual=r)
        if r is not None:
            assert torch.equal(few[1], h)
            few, ordinary = few[0], ordinary[0]
        assert torch.isfinite(ordinary).all() and torch.isfinite(few).all()
        for t in range(8):
            assert near(few[t], want[t], torch.bfloat16, 4), t


def test_which_way_experts_in_4_bits_go():
    """By the experts that a slice of 16 tokens hits and the size of their weights, not by the number of tokens alone."""
    from moe_explore.few_tokens import weights_pay_in_16_bits as pays
    big = 3 * 7168 * 2048
    assert not pays(96, 8, 64, big) and pays(128, 8, 64, big)
    assert not pays(160, 8, 256, 3 * 2048 * 768) and pays(256, 8, 256, 3 * 2048 * 768)
    assert not pays(97, 1, 1024, 3 * 1024 * 256) and pays(1024, 1, 1024, 3 * 1024 * 256)
    assert not pays(512, 1, 256, 3 * 2048 * 1024) and pays(1024, 1, 256, 3 * 2048 * 1024)
    for topk, experts, elements in ((1, 1, 64), (2, 6, 3 * 128 * 64), (8, 64, big), (64, 64, 1 << 20), (256, 1024, 1 << 16)):
        ways = [pays(t, topk, experts, elements) for t in range(0, 2000)]
        assert not ways[0] and ways[-1] and ways == sorted(ways)   # one line, few tokens in front of it


@gpu
def test_the_way_that_the_parameters_name(native):
    """Never in 16 bits: the bits of the slices, and not the memory of the weights; always: the 16-bit pass, for few tokens too."""
    g = gen(40)
    d, E, k, inter, T = 512, 16, 2, 512, 400
    q, _, _ = make_experts(g, 4, E, d, inter, "swiglu", torch.bfloat16, 64)
    x = torch.randn(T, d, generator=g, device="cuda").bfloat16()
    indices = torch.rand(T, E, generator=g, device="cuda").topk(k, dim=1).indices
    scores = torch.rand(T, k, generator=g, device="cuda").bfloat16()
    wide = int4_experts_in_16_bits(q)
    in_16 = lambda t: routed_expert_compute(x[:t], scores[:t], wide.weight1, wide.weight2, indices[:t], E, k, "swiglu")
    slices = torch.cat([int4_expert_compute(x[t:t + 16], scores[t:t + 16], indices[t:t + 16], q) for t in range(0, T, 16)])
    with torch.no_grad():
        assert torch.equal(int4_expert_compute(x, scores, indices, q), in_16(T))
        q.expand = False
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        assert torch.equal(int4_expert_compute(x, scores, indices, q), slices)
        torch.cuda.synchronize()
        assert torch.cuda.max_memory_allocated() - before < (wide.weight1.numel() + wide.weight2.numel()) * 2
        q.expand = True
        assert torch.equal(int4_expert_compute(x[:5], scores[:5], indices[:5], q), in_16(5))
        assert int4_expert_compute(x[:0], scores[:0], indices[:0], q).shape == (0, d)
        # the layer asks them, too
        p = MOEParams(make_router(g, "topk", d, E, k, torch.bfloat16), q, E, k)
        from moe_explore.router import router
        for expand in (True, False, None):
            q.expand = expand
            assert torch.equal(topk_moe_forward(x, p), int4_expert_compute(x, *router(x, p.router_params), q))
    native.check_status(device_status(0))


@gpu
@pytest.mark.parametrize("groups,open_,E", [(33, 5, 99), (33, 33, 99), (64, 40, 256), (64, 1, 512), (64, 63, 1024)])
def test_many_groups(groups, open_, E, native):
    """More groups than lanes (the router's own kernel takes 32): against the choice in 64 bits."""
    g = gen(groups * open_)
    k = min(6, open_ * (E // groups))
    for best in (1, 2):
        rp = grouped(E, k, 0.1 * torch.randn(E, generator=g, device="cuda"), groups, open_, best, normalize=True)
        logits = torch.randn(16, E, generator=g, device="cuda")
        got = weights_of(logits, rp, E).double()
        w, i = route64(rp, logits.double())
        want = torch.zeros_like(got).scatter_(1, i, w)
        assert torch.equal(got != 0, want != 0)
        assert bool(((got - want).abs() <= (2.0 ** -8 + 2.0 ** -18) * want).all())   # (k sums of 32 bits beside the rounding)
    native.check_status(device_status(0))


@gpu
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 16), (torch.float16, 4)])
def test_the_widest_rows(dtype, bits, native):
    """16 tokens of 16384 columns: as much shared memory as the first kernel asks for."""
    g = gen(21)
    d, E, k, inter = 16384, 18, 2, 24
    experts, w1, w2 = make_experts(g, bits, E, d, inter, "swiglu", dtype)
    rp = make_router(g, "topk norm", d, E, k, dtype)
    norm = RMSNormParams((1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dtype), 1e-5)
    p = MOEParams(rp, experts, E, k, None, norm)
    x, residual = (torch.randn(16, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    h = (x + residual)
    y = h.double()
    y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * norm.weight.double()
    with torch.no_grad():
        out, stream = few_token_layer(x, p, residual, None, norm)
    assert torch.equal(stream, h)
    assert near(out, experts64(y, *route64(rp, y @ rp.router_weight.double()), w1, w2, "swiglu"), dtype, 4)
    native.check_status(device_status(0))


@gpu
@pytest.mark.parametrize("norm_type", [torch.bfloat16, torch.float32])
def test_the_library_with_a_norm_and_given_experts(norm_type, native):
    """The C entry without a router: one cluster norms the rows, experts and scores are the caller's."""
    g = gen(22)
    T, d, E, k, inter = 9, 264, 6, 2, 40
    experts, w1, w2 = make_experts(g, 16, E, d, inter, "swiglu", torch.bfloat16)
    weight = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(norm_type)
    x, residual = (torch.randn(T, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda")
    scores = torch.rand(T, k, generator=g, device="cuda").bfloat16()
    out, stream = torch.empty_like(x), torch.empty_like(x)
    workspace = torch.empty(native.few_workspace_bytes(T, d, inter, E, k), dtype=torch.uint8, device="cuda")
    p = native.FewPass(num_tokens=T, d=d, inter=inter, num_experts=E, topk=k, act=native.ACT_CODES["swiglu"], dtype=0, bits=16, eps=1e-5,
                       norm_dtype=native.float_code(norm_type))
    p.x, p.residual, p.norm_w, p.stream_out, p.out = (t.data_ptr() for t in (x, residual, weight, stream, out))
    p.w1, p.w2, p.expert_idx, p.scores = (t.data_ptr() for t in (experts.weight1, experts.weight2, ids, scores))
    p.status, p.workspace, p.workspace_bytes = device_status(0).data_ptr(), workspace.data_ptr(), workspace.numel()
    native.few_tokens(p)
    h = x + residual
    y = h.double()
    y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * weight.double()
    want = torch.zeros_like(y)
    for s in range(k):   # (a token may have an expert twice)
        want += experts64(y, scores[:, s:s + 1].double(), ids[:, s:s + 1], w1, w2, "swiglu")
    assert torch.equal(stream, h) and near(out, want, torch.bfloat16, 4)
    native.check_status(device_status(0))


# ------------------------------------------------------------------------------------------------------- refusals
def test_refusals_of_the_library(native):
    import ctypes
    lib = native.load()
    assert native.few_workspace_bytes(16, 256, 128, 8, 2) >= 16 * 2 * 256 * 4 and lib.moe_few_workspace_bytes(-1, 8, 8, 8, 1) == 0
    call = lambda p: (lib.moe_few_tokens(ctypes.byref(p), None), lib.moe_last_error())
    def base(**kw):
        p = native.FewPass(num_tokens=1, d=64, inter=64, num_experts=8, topk=2, act=3, dtype=0, bits=16, num_groups=1, topk_groups=1, group_best=1)
        p.expert_idx = p.scores = 16
        for name, v in kw.items():
            setattr(p, name, v)
        return p
    assert lib.moe_few_tokens(None, None) == -1
    for kw, rc, text in [(dict(num_tokens=17), -2, b"at most"), (dict(topk=0), -1, b"k=0"), (dict(num_experts=2000), -2, b"at most"), (dict(d=60), -2, b"multiples of 8"),
                         (dict(dtype=5), -1, b"dtype"), (dict(act=9), -1, b"activation"), (dict(bits=4, group=16), -1, b"groups"), (dict(bits=8), -1, b"16 bits"),
                         (dict(scores=None), -1, b"router, or"), (dict(router_w=16, num_groups=3), -1, b"groups"), (dict(router_w=16, router_dtype=7), -1, b"router options"),
                         (dict(router_w=16, score_function=2, router_bias=16), -1, b"without bias"), (dict(), -1, b"null"),
                         (dict(x=16, w1=16, w2=16, out=16, workspace=16), -1, b"workspace has"), (dict(x=8, w1=16, w2=16, out=16, workspace=16), -1, b"aligned"),
                         (dict(x=16, w1=16, w2=16, out=16, workspace=16, residual=16), -1, b"residual")]:
        got = call(base(**kw))
        assert got[0] == rc and text in got[1], (kw, got)
    assert call(base(num_tokens=0))[0] == 0


def test_the_library_refuses_norms_of_another_type(native):
    import ctypes
    lib = native.load()
    for dtype, norm_dtype in ((0, 1), (1, 0), (0, 3), (1, -1)):
        p = native.FewPass(num_tokens=1, d=64, inter=64, num_experts=8, topk=2, act=3, dtype=dtype, bits=16, norm_dtype=norm_dtype)
        p.expert_idx = p.scores = p.norm_w = 16
        assert lib.moe_few_tokens(ctypes.byref(p), None) == -1 and b"norm_w" in lib.moe_last_error()
        p.norm_w = None
        assert lib.moe_few_tokens(ctypes.byref(p), None) == -1 and b"null" in lib.moe_last_error()


@gpu
def test_refusals(native):
    g = gen(14)
    q, _, _ = make_experts(g, 4, 8, 64, 32, "swiglu", torch.bfloat16, 32)
    x = torch.randn(2, 64, device="cuda").bfloat16()
    s, i = torch.rand(2, 2, device="cuda").bfloat16(), torch.zeros(2, 2, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError, match="type of the scales"):
        int4_expert_compute(x.half(), s, i, q)
    with pytest.raises(ValueError, match="tokens, k"):
        int4_expert_compute(x, s, i.int(), q)
    with pytest.raises(ValueError, match="fit together"):
        int4_expert_compute(x[:, :56], s, i, q)
    with pytest.raises(ValueError, match="fit together"):
        int4_expert_compute(x, s, i, Int4ExpertParams(q.up, q.down, "silu"))
    with pytest.raises(ValueError, match="addend"):
        int4_expert_compute(x, s, i, q, addend=x[:1])
    with pytest.raises(RuntimeError, match="CUDA"):
        int4_expert_compute(x, s.cpu(), i, q)
    with pytest.raises(ValueError, match="norm is None"):
        few_token_layer(x, MOEParams(make_router(g, "topk", 64, 8, 2, torch.bfloat16), q, 8, 2), residual=x)
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda t: int4_expert_compute(t, s, i, q), (x,), check_trace=False)
