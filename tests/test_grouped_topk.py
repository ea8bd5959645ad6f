"""Routing to experts in groups: the choice, the weights and the logits' gradient against a plain form in 64 bits, and refusals."""
import math

import pytest
import torch

from moe_explore.params import GroupedTopkRouterParams
from moe_explore.router import grouped_topk_of_logits, grouped_topk_router, router


def plain(logits, p):
    """(weights, indices) in 64 bits; differentiable with respect to the logits."""
    x = logits.double()
    T, E = x.shape
    prob = torch.sigmoid(x) if p.score_function == "sigmoid" else torch.softmax(x, -1)
    key = prob.detach() if p.bias is None else prob.detach() + p.bias.double()
    groups = key.view(T, p.num_groups, -1)
    rank = groups.sort(-1, descending=True).values[..., :p.group_best].sum(-1)
    open_groups = rank.sort(dim=-1, descending=True, stable=True).indices[:, :p.topk_groups]
    open_ = torch.zeros(T, p.num_groups, dtype=torch.bool, device=x.device).scatter_(1, open_groups, True)
    open_ = open_.repeat_interleave(E // p.num_groups, 1)
    # closed experts come after every open one, whatever its value
    order = key.sort(dim=-1, descending=True, stable=True).indices
    first = open_.gather(1, order).int().sort(dim=-1, descending=True, stable=True).indices
    indices = order.gather(1, first)[:, :p.topk]
    w = prob.gather(1, indices)
    if p.normalize_routing:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return w * p.scale, indices


# experts, groups, open groups, best, k: one group; uneven lanes; every lane width; more groups than a power of two
SHAPES = [(8, 1, 1, 1, 2), (3, 1, 1, 1, 3), (60, 4, 2, 1, 4), (60, 4, 3, 2, 6), (256, 8, 4, 2, 8), (256, 8, 8, 2, 8), (256, 1, 1, 1, 32),
          (160, 8, 3, 1, 6), (30, 5, 2, 2, 5), (512, 2, 1, 2, 8), (1024, 32, 5, 2, 16), (1020, 17, 4, 2, 32), (32, 32, 7, 1, 7)]


def make(E, G, keep, best, k, score="sigmoid", bias=True, normalize=True, scale=2.5, device="cuda", seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    b = 0.1 * torch.randn(E, generator=g, device=device) if bias else None
    return GroupedTopkRouterParams(None, k, bias=b, num_groups=G, topk_groups=keep, group_best=best, score_function=score,
                                   normalize_routing=normalize, scale=scale)


def close(got, want, dtype):
    """One rounding to `dtype` on top of the evaluation in fp32: a few units each for exp, sums and quotients, one unit (2^-24) per
    addition of a softmax's sum (at most 64 per lane and 5 joins).  Below the type's normal range its steps are all
    tiny * eps wide (fp16: 2^-14 * 2^-10), and a rounding is off by half of one."""
    f = torch.finfo(dtype)
    return bool(((got.double() - want).abs() <= (f.eps / 2 + 80 * 2.0 ** -24) * want.abs() + f.tiny * f.eps / 2).all())


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("E,G,keep,best,k", SHAPES)
def test_choice_and_weights(E, G, keep, best, k, bias, score, native):
    for T, dtype, out, normalize in ((1, torch.float32, torch.bfloat16, True), (5, torch.bfloat16, torch.float16, False),
                                     (1000, torch.float32, torch.float32, True), (333, torch.float16, torch.float32, True)):
        p = make(E, G, keep, best, k, score, bias, normalize, seed=T)
        g = torch.Generator(device="cuda").manual_seed(T + E)
        logits = (1.5 * torch.randn(T, E, generator=g, device="cuda")).to(dtype)   # 16 bits: many equal logits
        scores, indices = grouped_topk_of_logits(logits, p, out)
        want, chosen = plain(logits, p)
        assert indices.dtype is torch.int64 and torch.equal(indices, chosen)
        assert scores.dtype is out and close(scores, want, out)


@pytest.mark.gpu
def test_values_too_close_for_32_bits_are_told_apart(native):
    """Biased scores that differ by 2^-40: the fp32 images are equal, the choice is still the exact one, in the group stage and in
    the expert stage.  (Biases are fp32: logit 0 gives p = 1/2, and p of other logits is matched by a bias in steps of 2^-26.)"""
    g = torch.Generator().manual_seed(0)
    T, E = 4096, 64
    logits = torch.randn(T, E, generator=g)
    p64 = torch.sigmoid(logits[0].double())
    bias = (0.75 - p64).float()          # c = 0.75 to within half a unit of the bias: 64 values that fp32 cannot order
    params = GroupedTopkRouterParams(None, 6, bias=bias.cuda(), num_groups=8, topk_groups=3, group_best=2)
    same = logits[:1].expand(T, E).contiguous()
    same[1:] += 1e-4 * torch.randn(T - 1, E, generator=g)
    _, indices = grouped_topk_of_logits(same.cuda(), params)
    _, want = plain(same.cuda(), params)
    assert torch.equal(indices, want)


@pytest.mark.gpu
@pytest.mark.parametrize("large", [64.0, 3.0e4, 3.0e38])
def test_members_that_cancel_rank_their_group_exactly(large, native):
    """A group's two members of +large and about -large leave a small sum with the large ones' roundings to fp32 (64 + p is rounded to
    2^-18 steps).  At 3e38 two members of one sign would leave the range of fp32, and p is below the bias's steps in 64 bits too."""
    g = torch.Generator().manual_seed(7)
    T, G = 4096, 16
    bias = torch.empty(G, 2)
    bias[:, 0], bias[:, 1] = large, -large + (0.5 if large < 1e5 else 0.0)
    if large > 1e5:
        bias[::2] = -large
    spread = 10.0 ** (-5.0 * torch.rand(T, 1, generator=g))      # 1e-5 to 1: around the steps of each of the sizes
    logits = spread * torch.randn(T, 2 * G, generator=g) + torch.randn(1, 2, generator=g).repeat(1, G)
    params = GroupedTopkRouterParams(None, 6, bias=bias.flatten().cuda(), num_groups=G, topk_groups=5, group_best=2)
    _, indices = grouped_topk_of_logits(logits.cuda(), params)
    _, want = plain(logits.cuda(), params)
    assert torch.equal(indices, want)


@pytest.mark.gpu
def test_ties_take_the_lowest_index(native):
    logits = torch.zeros(3, 24, device="cuda")
    logits[1, 20] = 1.0
    logits[2, 23] = 1.0
    logits[2, 6] = 1.0
    p = GroupedTopkRouterParams(None, 4, bias=torch.zeros(24, device="cuda"), num_groups=4, topk_groups=2)
    _, idx = grouped_topk_of_logits(logits, p)
    assert idx.tolist() == [[0, 1, 2, 3], [20, 0, 1, 2], [6, 23, 7, 8]]
    p.bias = None
    assert torch.equal(grouped_topk_of_logits(logits, p)[1], idx)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_equal_values_of_a_whole_prompt(score, native):
    """A bias of zeros, as training begins with it, and 16-bit logits: a third of the tokens have equal values among their best."""
    T, E = 16384, 256
    logits = (1.5 * torch.randn(T, E, generator=torch.Generator(device="cuda").manual_seed(11), device="cuda")).bfloat16()
    p = GroupedTopkRouterParams(None, 8, bias=torch.zeros(E, device="cuda"), num_groups=8, topk_groups=4, score_function=score)
    scores, indices = grouped_topk_of_logits(logits, p, torch.float32)
    best = logits.sort(-1, descending=True).values[:, :9]
    assert float((best[:, 1:] == best[:, :-1]).any(-1).float().mean()) > 0.25
    want, chosen = plain(logits, p)
    assert torch.equal(indices, chosen) and close(scores, want, torch.float32)
    p.bias = None
    assert torch.equal(grouped_topk_of_logits(logits, p)[1], chosen)


@pytest.mark.gpu
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
def test_masked_experts(low, native):
    """Logits or biases of minus infinity, or the type's lowest value, leave an expert for last; rows with nothing left still get k
    different experts."""
    logits = torch.randn(5, 16, device="cuda")
    logits[0, :13] = low
    logits[1] = low
    p = GroupedTopkRouterParams(None, 4, num_groups=2, topk_groups=2)
    scores, idx = grouped_topk_of_logits(logits, p)
    assert idx[0, :3].sort().values.tolist() == [13, 14, 15] and idx[0, 3] == 0
    assert idx[1].tolist() == [0, 1, 2, 3]
    assert torch.isfinite(scores).all() and scores[1].abs().max() == 0    # p = 0: 0 / (0 + 1e-20)
    bias = torch.zeros(16, device="cuda")
    bias[4:] = low
    q = GroupedTopkRouterParams(None, 4, bias=bias, num_groups=2, topk_groups=1)
    scores, idx = grouped_topk_of_logits(torch.randn(5, 16, device="cuda"), q)
    assert idx.sort(-1).values.tolist() == [[0, 1, 2, 3]] * 5 and torch.isfinite(scores).all()


@pytest.mark.gpu
def test_nan_comes_last_and_stays_in_its_row(native):
    logits = torch.randn(4, 16, device="cuda")
    clean = grouped_topk_of_logits(logits, GroupedTopkRouterParams(None, 3, num_groups=4, topk_groups=2))
    logits[1, 5] = math.nan
    logits[2] = math.nan
    scores, idx = grouped_topk_of_logits(logits, GroupedTopkRouterParams(None, 3, num_groups=4, topk_groups=2))
    for row in (0, 3):
        assert torch.equal(scores[row], clean[0][row]) and torch.equal(idx[row], clean[1][row])
    assert 5 not in idx[1].tolist() and torch.isfinite(scores[1]).all()
    assert len(set(idx[2].tolist())) == 3 and int(idx[2].max()) < 16 and torch.isnan(scores[2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T,E,G,keep,k,dtype,out", [(1, 8, 1, 1, 2, torch.float32, torch.float32), (257, 60, 4, 2, 4, torch.bfloat16, torch.bfloat16),
                                                    (100, 256, 8, 4, 8, torch.float32, torch.bfloat16), (33, 1024, 32, 9, 32, torch.float16, torch.float32)])
def test_gradient_of_the_logits(T, E, G, keep, k, dtype, out, normalize, score, native):
    p = make(E, G, keep, 2, k, score, True, normalize, seed=3)
    g = torch.Generator(device="cuda").manual_seed(E)
    logits = torch.randn(T, E, generator=g, device="cuda").to(dtype).requires_grad_(True)
    d = torch.randn(T, k, generator=g, device="cuda").to(out)
    scores, _ = grouped_topk_of_logits(logits, p, out)
    got, = torch.autograd.grad(scores, logits, d)
    leaf = logits.detach().double().requires_grad_(True)
    want, = torch.autograd.grad(plain(leaf, p)[0], leaf, d.double())
    assert got.dtype is dtype
    # fp32: the differences are taken in 64 bits, p and the softmax's inner product in 32 (see close()); relative to the row
    err = (got.double() - want).abs()
    assert bool((err <= torch.finfo(dtype).eps / 2 * want.abs() + 160 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True)
                 + (2.0 ** -25 if dtype is torch.float16 else 0)).all())


@pytest.mark.gpu
def test_gradient_against_differences(native):
    """Central differences of the weights in 64 bits, given the selection."""
    p = make(32, 4, 2, 2, 4, "softmax")
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(3, 32, generator=g, device="cuda").requires_grad_(True)
    d = torch.randn(3, 4, generator=g, device="cuda")
    scores, chosen = grouped_topk_of_logits(logits, p)
    got, = torch.autograd.grad(scores, logits, d)

    def loss(x):
        w = torch.softmax(x, -1).gather(1, chosen)
        return (p.scale * w / w.sum(-1, keepdim=True) * d.double()).sum()

    step = 1e-5
    for row, col in ((0, int(chosen[0, 0])), (1, int(chosen[1, 3])), (2, 0), (2, 31)):
        e = torch.zeros(3, 32, dtype=torch.float64, device="cuda")
        e[row, col] = step
        x = logits.detach().double()
        difference = float(loss(x + e) - loss(x - e)) / (2 * step)
        assert abs(float(got[row, col]) - difference) < 1e-6    # step^2 and fp32 rounding of values below 1


@pytest.mark.gpu
def test_router_dispatch_layer_and_its_gradient(native):
    """``router`` takes the parameters, and the layer trains through them: gradients reach input, router and experts."""
    from moe_explore.functional.topk_moe import topk_moe_forward, topk_moe_torch
    from moe_explore.params import MLPParams, MOEParams

    g = torch.Generator(device="cuda").manual_seed(0)
    new = lambda *s, scale=1.0: (scale * torch.randn(*s, generator=g, device="cuda")).bfloat16().requires_grad_(True)
    x, w1, w2 = new(77, 128), new(16, 128, 128, scale=0.1), new(16, 64, 128, scale=0.1)
    rw = (0.2 * torch.randn(128, 16, generator=g, device="cuda")).requires_grad_(True)
    rp = GroupedTopkRouterParams(rw, 3, bias=0.05 * torch.randn(16, generator=g, device="cuda"), num_groups=4, topk_groups=2)
    scores, indices = router(x, rp)
    assert scores.dtype is torch.bfloat16 and torch.equal(indices, plain(x.detach().float() @ rw.detach(), rp)[1])
    params = MOEParams(rp, MLPParams(w1, w2, "swiglu"), 16, 3)
    d = torch.randn(77, 128, generator=g, device="cuda").bfloat16()
    got = torch.autograd.grad(topk_moe_forward(x, params), (x, rw, w1, w2), d)
    want = torch.autograd.grad(topk_moe_torch(x, params), (x, rw, w1, w2), d)
    for a, b in zip(got, want):   # both sides round every product to bf16; the torch form each sum as well
        assert float((a.float() - b.float()).norm() / b.float().norm()) < 0.02
    with torch.no_grad():
        assert torch.equal(grouped_topk_router(x, rp)[1], indices)


@pytest.mark.gpu
def test_empty_strided_captured_and_on_another_stream(native):
    p = make(64, 8, 4, 2, 8)
    scores, indices = grouped_topk_of_logits(torch.empty(0, 64, device="cuda"), p)
    assert scores.shape == (0, 8) and indices.shape == (0, 8)
    wide = torch.randn(50, 128, device="cuda")
    a = grouped_topk_of_logits(wide[:, ::2], p)
    b = grouped_topk_of_logits(wide[:, ::2].contiguous(), p)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    odd = torch.empty(50 * 64 + 1, device="cuda")[1:].view(50, 64).copy_(wide[:, ::2])   # rows that begin between two 16-byte borders
    assert torch.equal(grouped_topk_of_logits(odd, p)[1], b[1])
    static = wide[:, ::2].contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grouped_topk_of_logits(static, p)
    static.copy_(torch.randn(50, 64, device="cuda"))
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = grouped_topk_of_logits(static, p)
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


def test_refusals(native):
    lib = native.load()
    call = lambda E=64, G=4, keep=2, best=2, k=4, dtype=2, T=4: lib.moe_grouped_topk(None, None, None, None, T, E, G, keep, best, k, 1, 1,
                                                                                   1.0, dtype, 2, None)
    assert call(E=63) == -1 and b"equal groups" in lib.moe_last_error()
    assert call(E=66, G=33) == -1 and b"groups" in lib.moe_last_error()
    assert call(keep=5) == -1 and call(keep=0) == -1
    assert call(E=8, G=4, keep=1, k=3) == -1 and b"hold no" in lib.moe_last_error()
    assert call(best=3) == -1 and call(E=4, G=4, k=2, best=2) == -1 and b"best one or two" in lib.moe_last_error()
    assert call(E=2048, G=1, keep=1) == -2 and call(E=512, G=1, keep=1, k=33) == -2
    assert call(dtype=9) == -1 and call(T=-1) == -1
    assert call() == -1 and b"null" in lib.moe_last_error()
    assert call(T=0) == 0
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        grouped_topk_of_logits(torch.zeros(2, 8), GroupedTopkRouterParams(None, 2))


@pytest.mark.gpu
def test_refusals_of_tensors(native):
    x = torch.zeros(2, 8, device="cuda")
    with pytest.raises(ValueError, match="score_function"):
        grouped_topk_of_logits(x, GroupedTopkRouterParams(None, 2, score_function="tanh"))
    with pytest.raises(ValueError, match="bias"):
        grouped_topk_of_logits(x, GroupedTopkRouterParams(None, 2, bias=torch.zeros(8, device="cuda", dtype=torch.bfloat16)))
    with pytest.raises(ValueError, match="tokens, experts"):
        grouped_topk_of_logits(x[0], GroupedTopkRouterParams(None, 2))
    with pytest.raises(TypeError):
        grouped_topk_of_logits(x.double(), GroupedTopkRouterParams(None, 2))
    with pytest.raises(native.MoeNativeError, match="equal groups"):
        grouped_topk_of_logits(x, GroupedTopkRouterParams(None, 2, num_groups=3))


@pytest.mark.gpu
def test_forward_mode_is_refused(native):
    from moe_explore.params import GroupedTopkRouterParams
    from moe_explore.router import grouped_topk_of_logits

    x = torch.randn(3, 16, device="cuda")
    p = GroupedTopkRouterParams(None, 2)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(Exception, match="forward"):
            grouped_topk_of_logits(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), p)
        scores, indices = grouped_topk_of_logits(x, p)
        assert scores.shape == indices.shape == (3, 2)
