"""Activations and experts that keep the un-activated product in 8 bits, against the formulas in 64 bits; refusals."""
import math

import pytest
import torch

from moe_explore.expert_compute import routed_expert_compute
from moe_explore.functional.activation_fp8 import activation_fp8
from moe_explore.functional.fp8 import BLOCK, DTYPE, LEAST, quantize_rows
from moe_explore.functional.topk_moe import topk_moe_forward
from moe_explore.params import MLPParams, MOEParams, RMSNormParams, SharedExpertParams, TopkRouterParams
from moe_explore.router import router

gpu = pytest.mark.gpu
ACTS = ["silu", "gelu", "approx_gelu", "swiglu", "geglu", None]
DTYPES = [torch.bfloat16, torch.float16]


def gated(act):
    return act is not None and "glu" in act


def act64(z, act):
    g = z[..., 0::2] if gated(act) else z
    if act in ("silu", "swiglu"):
        y = g * torch.sigmoid(g)
    elif act in ("gelu", "geglu"):
        y = 0.5 * g * (1 + torch.erf(g / math.sqrt(2)))
    elif act == "approx_gelu":
        y = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    else:
        y = g
    return y * z[..., 1::2] if gated(act) else y


def kept64(x):
    """What 8 bits give back of 16-bit rows: the quotient x * 448 / max of short numbers has one rounding to fp32 and one to e4m3."""
    k = x.size(-1)
    pad = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    most = pad.abs().amax(-1, keepdim=True).clamp_min(LEAST)
    q = (pad * 0.875 / most * 512).to(DTYPE)
    return (q.double() * (most.double() / 448)).flatten(-2)[..., :k]


def gradient64(kept, dh, act):
    z = kept.detach().requires_grad_(True)
    return torch.autograd.grad(act64(z, act), z, dh)[0]


def close(got, want, size, dtype):
    """Half a step of the type, and behind it what fp32 evaluation is off by, relative to the size of the factors: the exponential of a
    rounded argument |x| < 32 (2^-24 * 32 * log2 e), hardware functions of 2^-21, cancellation in 1 + erf and 1 + x (1 - p), products
    and the scale (2^-23 each), together below 2^-17."""
    f = torch.finfo(dtype)
    return bool(((got.double() - want).abs() <= (f.eps / 2 * want.abs() + 2.0 ** -17 * size) * (1 + f.eps) + f.tiny * f.eps / 2).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,inter", [(1, 8), (3, 64), (1, 14336), (37, 776), (130, 1544), (700, 264), (6000, 136)])
def test_activation_and_gradient(rows, inter, act, dtype, native):
    g = torch.Generator(device="cuda").manual_seed(rows + inter)
    x = (3 * torch.randn(rows, inter * (2 if gated(act) else 1), generator=g, device="cuda")).to(dtype).requires_grad_(True)
    dy = torch.randn(rows, inter, generator=g, device="cuda").to(dtype)
    y = activation_fp8(x, act)
    dx, = torch.autograd.grad(y, x, dy)
    z = x.detach().double()
    assert y.dtype is dtype and dx.dtype is dtype and y.shape == dy.shape
    up = z[..., 1::2].abs() if gated(act) else torch.ones_like(dy, dtype=torch.float64)
    gate = z[..., 0::2].abs() if gated(act) else z.abs()
    assert close(y, act64(z, act), gate * up, dtype)
    kept = kept64(x.detach())
    g64 = kept[..., 0::2].abs() if gated(act) else kept.abs()
    size = dy.double().abs() * (1 + g64)
    if gated(act):
        size = torch.stack((size * kept[..., 1::2].abs(), size), -1).flatten(-2)
    assert close(dx, gradient64(kept, dy.double(), act), size, dtype)
    with torch.no_grad():
        assert torch.equal(activation_fp8(x, act), y)


@gpu
@pytest.mark.parametrize("act", ["swiglu", "gelu"])
def test_gradient_against_differences(act, native):
    """At values that 8 bits hold the gradient is the function's: central differences of the 64-bit formula (step h: off by h^2 / 6 times
    the third derivative, below 4 here, times the factors of at most 8)."""
    cols = 64
    x = torch.randint(-14, 15, (5, cols), device="cuda").div(4).bfloat16()
    x[:, 0] = 3.5                                       # the block's scale is 3.5 / 448 = 2^-7, and these are multiples of 32 of them
    assert torch.equal(kept64(x), x.double())
    x.requires_grad_(True)
    dy = torch.randint(-2, 3, (5, cols // 2 if gated(act) else cols), device="cuda").bfloat16()
    dx, = torch.autograd.grad(activation_fp8(x, act), x, dy)
    z, h = x.detach().double(), 1e-4
    for j in range(0, cols, 7):
        e = torch.zeros_like(z)
        e[:, j] = h
        slope = ((act64(z + e, act) - act64(z - e, act)) / (2 * h) * dy.double()).sum(-1)
        assert bool(((dx[:, j].double() - slope).abs() <= 2.0 ** -8 * slope.abs() + 1e-6 + h * h / 6 * 4 * 8).all())


@gpu
def test_shapes_strides_and_nothing(native):
    x = torch.randn(4, 6, 200, device="cuda").bfloat16()
    part = x[:, :, 5:5 + 192]                            # neither dense nor aligned
    assert torch.equal(activation_fp8(part, "swiglu"), activation_fp8(part.contiguous(), "swiglu"))
    leaf = x.clone().requires_grad_(True)
    dy = torch.randn(4, 6, 96, device="cuda").bfloat16()
    dx, = torch.autograd.grad(activation_fp8(leaf[:, :, 5:5 + 192], "swiglu"), leaf, dy.expand(4, 6, 96))
    dense = part.clone().requires_grad_(True)
    want, = torch.autograd.grad(activation_fp8(dense, "swiglu"), dense, dy)
    assert torch.equal(dx[:, :, 5:5 + 192], want) and not dx[:, :, :5].any() and not dx[:, :, 197:].any()
    one, = torch.autograd.grad(activation_fp8(leaf, "silu").sum(), leaf)        # the gradient of a sum: one value, expanded
    same, = torch.autograd.grad(activation_fp8(leaf, "silu"), leaf, torch.ones_like(leaf))
    assert torch.equal(one, same)
    empty = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = activation_fp8(empty, "swiglu")
    assert y.shape == (0, 32) and torch.autograd.grad(y, empty, torch.empty_like(y))[0].shape == (0, 64)
    assert activation_fp8(torch.randn(16, device="cuda").half(), "gelu").shape == (16,)


@gpu
def test_values_that_are_not_finite_stay_in_their_block(native):
    x = torch.randn(3, 512, device="cuda").bfloat16()
    x[0, 5], x[1, 300] = math.nan, math.inf
    x[2, :128] = 0
    leaf = x.clone().requires_grad_(True)
    dy = torch.ones(3, 512, device="cuda").bfloat16()
    dx, = torch.autograd.grad(activation_fp8(leaf, "silu"), leaf, dy)
    assert torch.isnan(dx[0, 5]) and torch.isfinite(dx[0, :5]).all() and torch.isfinite(dx[0, 6:]).all()
    assert torch.isfinite(dx[1, :256]).all() and torch.isfinite(dx[1, 384:]).all()
    assert bool((dx[2, :128] == 0.5).all())              # the slope of silu at zero


@gpu
def test_kept_bits_are_those_of_quantize_rows(native):
    x = torch.randn(40, 272, device="cuda").bfloat16()
    h, q = torch.empty(40, 136, dtype=x.dtype, device="cuda"), torch.empty(40, 272, dtype=DTYPE, device="cuda")
    scales = torch.empty(40, 3, device="cuda")
    native.act_f8_forward(x, h, q, scales, "swiglu")
    want = quantize_rows(x)
    assert torch.equal(q.view(torch.uint8), want.data.view(torch.uint8)) and torch.equal(scales, want.scales)


@gpu
def test_streams_graphs_and_an_eager_graph_that_lives(native):
    """Captured and replayed with other inputs, forward and backward, while an eager graph of the same leaf is alive; on a side stream."""
    leaf = torch.randn(300, 512, device="cuda").bfloat16().requires_grad_(True)
    dy = torch.randn(300, 256, device="cuda").bfloat16()
    alive = activation_fp8(leaf, "swiglu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        static = leaf.detach().clone().requires_grad_(True)
        for _ in range(2):
            torch.autograd.grad(activation_fp8(static, "swiglu"), static, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = activation_fp8(static, "swiglu")
        dx, = torch.autograd.grad(y, static, dy)
    with torch.no_grad():
        static.copy_(torch.randn(300, 512, device="cuda"))
        dy.copy_(torch.randn(300, 256, device="cuda"))
    graph.replay()
    now = static.detach().clone().requires_grad_(True)
    want = activation_fp8(now, "swiglu")
    assert torch.equal(y, want) and torch.equal(dx, torch.autograd.grad(want, now, dy)[0])
    assert torch.isfinite(torch.autograd.grad(alive, leaf, dy)[0]).all()


# --------------------------------------------------------------------------------------------------------- experts
def experts(T, d, E, k, inter, act, dtype, seed=0, skew=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")
    top = torch.topk(new(T, E) + skew * new(E), k, dim=-1)
    x, dy = new(T, d).to(dtype), new(T, d).to(dtype)
    w1 = (new(E, d, inter * (2 if gated(act) else 1)) * d ** -0.5).to(dtype)
    w2 = (new(E, inter, d) * inter ** -0.5).to(dtype)
    scores = torch.softmax(top.values, -1).to(dtype)
    return [t.requires_grad_(True) for t in (x, scores, w1, w2)], top.indices, dy


def reference(leaves, indices, dy, act):
    """The formulas in 64 bits on the product rounded to the 16 bits that are kept."""
    x, scores, w1, w2 = (t.detach().double() for t in leaves)
    dtype = leaves[0].dtype
    out = [torch.zeros_like(t) for t in (x, x, scores, w1, w2)]
    for e in range(w1.size(0)):
        token, slot = (indices == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        s = scores[token, slot, None]
        pre = (x[token] @ w1[e]).to(dtype)
        out[0].index_add_(0, token, s * (act64(pre.double(), act) @ w2[e]))
        kept = kept64(pre)
        h, du = act64(kept, act), dy.double()[token] @ w2[e].T
        d_pre = gradient64(kept, s * du, act)
        out[1].index_add_(0, token, d_pre @ w1[e].T)
        out[2][token, slot] = (du * h).sum(-1)
        out[3][e] = x[token].T @ d_pre
        out[4][e] = (s * h).T @ dy.double()[token]
    return out


@gpu
@pytest.mark.parametrize("T,d,E,k,inter,act,dtype,skew", [
    (1, 64, 4, 1, 32, "swiglu", torch.bfloat16, 0.0), (5, 64, 8, 8, 40, "silu", torch.float16, 0.0),
    (64, 256, 8, 2, 512, "swiglu", torch.bfloat16, 0.0), (301, 136, 12, 3, 264, "geglu", torch.float16, 2.0),
    (257, 264, 60, 4, 136, "gelu", torch.bfloat16, 3.0), (130, 128, 3, 2, 128, "approx_gelu", torch.bfloat16, 0.0),
    (90, 128, 6, 2, 72, None, torch.bfloat16, 1.0), (2000, 512, 16, 4, 256, "swiglu", torch.bfloat16, 1.0)])
def test_experts_and_gradients(T, d, E, k, inter, act, dtype, skew, native):
    """Relative to the root of the mean square of the whole tensor.  Each of the roundings in between (product, activated rows, an expert's
    row, u, its product with the slope, the weighted rows, the result) is off by at most half a step, eps / 2, of its value, eps / 2 /
    sqrt(3) at the root of the mean square; a rounded product that fp32 sums leave on the other side of a middle is rare.  No tensor has
    more than six of them: 6 * eps / 2 covers them whatever their correlation, twice over."""
    leaves, indices, dy = experts(T, d, E, k, inter, act, dtype, T, skew)
    y = routed_expert_compute(*leaves, indices, E, k, act, save_fp8=True)
    got = (y,) + torch.autograd.grad(y, leaves, dy)
    for name, a, b in zip(("y", "dx", "d_scores", "d_w1", "d_w2"), got, reference(leaves, indices, dy, act)):
        assert a.dtype is dtype and a.shape == b.shape
        assert float((a.detach().double() - b).norm()) <= 6 * torch.finfo(dtype).eps / 2 * float(b.norm()) + 1e-30, name
    native.check_status(__import__("moe_explore.routing_plan", fromlist=["device_status"]).device_status(0))


@gpu
def test_experts_keep_less_and_repeat(native):
    leaves, indices, dy = experts(1024, 256, 8, 4, 512, "swiglu", torch.bfloat16)
    def held(save):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = routed_expert_compute(*leaves, indices, 8, 4, "swiglu", save_fp8=save)
        return y, torch.cuda.memory_allocated() - before - y.numel() * 2
    y8, small = held(True)
    y16, large = held(False)
    # rows of 8 bits with their scales and the index arrays, against 16-bit rows of input, product, activated product and result
    assert small <= 4096 * (1024 + 4 * 8) * 1.4 + 2 ** 20 < large / 2
    first = torch.autograd.grad(y8, leaves, dy)
    second = torch.autograd.grad(routed_expert_compute(*leaves, indices, 8, 4, "swiglu", save_fp8=True), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with torch.no_grad():   # nothing to keep: the pass that has no gradient
        assert torch.equal(routed_expert_compute(*leaves, indices, 8, 4, "swiglu", save_fp8=True),
                           routed_expert_compute(*leaves, indices, 8, 4, "swiglu"))


@gpu
def test_experts_with_dropped_slots_empty_input_and_broadcast_gradients(native):
    from moe_explore.routing_plan import device_status

    leaves, indices, dy = experts(70, 64, 5, 2, 48, "swiglu", torch.bfloat16)
    bad = indices.clone()
    bad[3, 1], bad[60, 0] = 5, -1
    y = routed_expert_compute(*leaves, bad, 5, 2, "swiglu", save_fp8=True)
    got = (y,) + torch.autograd.grad(y, leaves, dy)
    assert native.read_status(device_status(0), reset=True) == native.STATUS_BAD_EXPERT_ID
    assert got[2][3, 1] == 0 and got[2][60, 0] == 0
    for a, b in zip(got, reference(leaves, bad, dy, "swiglu")):
        assert float((a.detach().double() - b).norm()) <= 6 * 2.0 ** -8 * float(b.norm())
    y = routed_expert_compute(*leaves, indices, 5, 2, "swiglu", save_fp8=True)
    a = torch.autograd.grad(y, leaves, torch.ones(1, device="cuda").bfloat16().expand(70, 64), retain_graph=True)
    b = torch.autograd.grad(y, leaves, torch.ones(70, 64, device="cuda").bfloat16())
    assert all(torch.equal(m, n) for m, n in zip(a, b))
    none = [leaves[0][:0].detach().requires_grad_(True), leaves[1][:0].detach().requires_grad_(True), *leaves[2:]]
    y = routed_expert_compute(*none, indices[:0], 5, 2, "swiglu", save_fp8=True)
    assert y.shape == (0, 64)
    grads = torch.autograd.grad(y, none, dy[:0])
    assert grads[0].shape == (0, 64) and not grads[2].any() and not grads[3].any()


@gpu
@pytest.mark.parametrize("normed", [False, True])
def test_layer_in_training(normed, native):
    """Norm, router, experts kept in 8 bits and shared expert together: the composed calls give the same bits; and the gradients are near
    those of the layer that keeps 16 bits (e4m3 is off by at most 2^-4 of a value, 2^-4 / sqrt(3) at the root of the mean square, in the
    two factors of the gated product and the slope)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")
    E, k, d, inter = 8, 2, 128, 96
    rp = TopkRouterParams((new(d, E) * d ** -0.5).bfloat16().requires_grad_(True), k, False)
    ep = MLPParams((new(E, d, 2 * inter) * d ** -0.5).bfloat16().requires_grad_(True), (new(E, inter, d) * inter ** -0.5).bfloat16().requires_grad_(True), "swiglu")
    sp = SharedExpertParams((new(1, d, 2 * inter) * d ** -0.5).bfloat16(), (new(1, inter, d) * inter ** -0.5).bfloat16(), "swiglu")
    norm = RMSNormParams((1 + 0.1 * new(d)).bfloat16()) if normed else None
    p = MOEParams(rp, ep, E, k, sp, norm)
    x = new(200, d).bfloat16().requires_grad_(True)
    dy = new(200, d).bfloat16()
    leaves = (x, rp.router_weight, ep.weight1, ep.weight2)
    y = topk_moe_forward(x, p, save_fp8=True)
    got = torch.autograd.grad(y, leaves, dy)
    if not normed:
        from moe_explore.expert_compute import dense_expert
        shared = dense_expert(x, sp.up_weight, sp.down_weight, "swiglu")   # (in the layer's order: the gradients of x add up in it)
        scores, indices = router(x, rp)
        composed = routed_expert_compute(x, scores, ep.weight1, ep.weight2, indices, E, k, "swiglu", save_fp8=True, addend=shared)
        assert torch.equal(y, composed)
        assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(composed, leaves, dy)))
    want = torch.autograd.grad(topk_moe_forward(x, p), leaves, dy)
    for a, b in zip(got, want):
        assert float((a.float() - b.float()).norm() / b.float().norm()) < 3 * 2.0 ** -4 / 3 ** 0.5


@gpu
def test_training_step_in_a_graph(native):
    leaves, indices, dy = experts(96, 128, 8, 2, 64, "swiglu", torch.bfloat16)
    step = lambda: torch.autograd.grad(routed_expert_compute(*leaves, indices, 8, 2, "swiglu", save_fp8=True), leaves, dy)
    # an eager graph of the same values (of the same leaves torch's engine would make the capture wait for the eager stream, and refuses)
    others = [t.detach().clone().requires_grad_(True) for t in leaves]
    alive = routed_expert_compute(*others, indices, 8, 2, "swiglu", save_fp8=True)
    want = torch.autograd.grad(alive, others, dy, retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(alive, others, dy), want))
    with torch.no_grad():
        leaves[0].copy_(torch.randn(96, 128, device="cuda"))
        indices.copy_(indices.flip(0))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(grads, step()))


def test_a_pass_that_keeps_8_bits_has_its_activation(native):
    """What the header rules out is refused before anything is launched: one expert for all rows, and products of rows that the activation's step
    would have written.  The masks of all steps hold that step."""
    import ctypes
    import os
    import re
    lib = native.load()
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(here, "include", "moe_sm100.h")) as f:
        masks = {name: int(value) for name, value in re.findall(r"#define (MOE_(?:FWD|BWD)_\w+) (\d+)", f.read())}
    assert masks["MOE_FWD_ALL"] & native.FWD_ACT and masks["MOE_BWD_ALL"] & native.BWD_ACT
    p = native.ExpertPass(num_tokens=0, padded_rows=0, d=64, inter=64, num_experts=1, topk=1, act=native.ACT_CODES["swiglu"], dtype=0)
    for f in ("pre_act", "hidden", "xs", "dh", "pre_q", "pre_scales"):
        setattr(p, f, 16)
    forward = lambda steps: (lib.moe_expert_forward(ctypes.byref(p), steps, None), lib.moe_last_error())
    backward = lambda steps: (lib.moe_expert_backward(ctypes.byref(p), steps, None), lib.moe_last_error())
    for call, steps in ((forward, native.FWD_UP | native.FWD_DOWN), (forward, 31), (backward, native.BWD_DOWN | native.BWD_UP),
                        (backward, native.BWD_DOWN | native.BWD_DW1), (backward, native.BWD_DOWN | native.BWD_DW2), (backward, 127)):
        got = call(steps)
        assert got[0] == -1 and b"_ACT" in got[1], (steps, got)
    p.identity = 1
    for call in (forward, backward):
        got = call(0)
        assert got[0] == -1 and b"identity" in got[1], got


# ------------------------------------------------------------------------------------------------------- refusals
def test_refusals_of_the_library(native):
    lib = native.load()
    assert lib.moe_act_f8_forward(None, None, None, None, 4, 64, 3, 0, None) == -1
    assert lib.moe_act_f8_forward(None, None, None, None, 4, 12, 3, 0, None) == -2 and b"multiple of 8" in lib.moe_last_error()
    assert lib.moe_act_f8_forward(None, None, None, None, -1, 64, 3, 0, None) == -1
    assert lib.moe_act_f8_backward(None, None, None, None, 4, 64, 9, 0, None) == -1 and b"activation" in lib.moe_last_error()
    assert lib.moe_act_f8_backward(None, None, None, None, 4, 64, 3, 7, None) == -1 and b"dtype" in lib.moe_last_error()
    assert lib.moe_act_f8_forward(16, 32, 48, None, 4, 64, 3, 0, None) == -1
    assert lib.moe_act_f8_forward(8, 32, None, None, 4, 64, 3, 0, None) == -1 and b"aligned" in lib.moe_last_error()


def test_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="CUDA"):
        activation_fp8(torch.zeros(2, 16).bfloat16(), "silu")


@gpu
def test_refusals(native):
    x = torch.randn(4, 48, device="cuda").bfloat16()
    with pytest.raises(TypeError, match="bf16 or fp16"):
        activation_fp8(x.float(), "silu")
    with pytest.raises(ValueError, match="multiples of 16"):
        activation_fp8(x[:, :24], "swiglu")
    with pytest.raises(ValueError, match="multiples of 8"):
        activation_fp8(x[:, :12], "silu")
    with pytest.raises(ValueError, match="Unsupported"):
        activation_fp8(x, "relu")
    leaves, indices, dy = experts(6, 64, 4, 2, 32, "swiglu", torch.bfloat16)
    call = lambda l, i=indices, **kw: routed_expert_compute(*l, i, 4, 2, "swiglu", save_fp8=True, **kw)
    with pytest.raises(ValueError, match="gather_in_gemm"):
        call(leaves, gather_in_gemm=True)
    with pytest.raises(ValueError, match="shapes"):
        call([leaves[0][:, :32], *leaves[1:]])
    with pytest.raises(ValueError, match="indices"):
        call(leaves, indices[:3])
    with pytest.raises(TypeError, match="one type"):
        call([leaves[0].half(), *leaves[1:]])
    with pytest.raises(ValueError, match="addend"):
        call(leaves, addend=leaves[0][:3])
    y = call(leaves)
    with torch.no_grad():
        leaves[0].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, leaves, dy)
