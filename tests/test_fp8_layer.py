"""The operators of a serving layer run together, as a model runs them: residual and norm, routing in groups, experts in 8 bits, shared
expert; and the same layer in training, with 16-bit experts."""
import pytest
import torch

from moe_explore.expert_compute import fp8_expert_compute
from moe_explore.functional.fp8 import quantize_experts
from moe_explore.functional.rms_norm import rms_norm, rms_norm_fp8
from moe_explore.functional.topk_moe import topk_moe_forward, topk_moe_torch
from moe_explore.params import GroupedTopkRouterParams, MLPParams, MOEParams, RMSNormParams, SharedExpertParams, TopkRouterParams
from moe_explore.router import router

gpu = pytest.mark.gpu


def make(E=16, k=4, d=256, inter=192, dtype=torch.bfloat16, shared=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s, scale=1.0: (scale * torch.randn(*s, generator=g, device="cuda"))
    experts = MLPParams(new(E, d, 2 * inter, scale=d ** -0.5).to(dtype), new(E, inter, d, scale=inter ** -0.5).to(dtype), "swiglu")
    rp = GroupedTopkRouterParams(new(d, E, scale=d ** -0.5), k, bias=new(E, scale=0.05), num_groups=4, topk_groups=2, scale=1.5)
    sp = SharedExpertParams(new(1, d, 2 * inter, scale=d ** -0.5).to(dtype), new(1, inter, d, scale=inter ** -0.5).to(dtype), "swiglu") if shared else None
    norm = RMSNormParams((1.0 + new(d, scale=0.1)).to(dtype), 1e-5)
    return MOEParams(rp, experts, E, k, sp, norm), new


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("T", [1, 2, 37, 700])
def test_serving_layer_is_its_parts(T, shared, dtype, native):
    """The layer's result is, bit for bit, what its operators give one after the other; two layers in a row hand the stream on."""
    p, new = make(dtype=dtype, shared=shared)
    p8 = MOEParams(p.router_params, quantize_experts(p.expert_params), p.num_experts, p.topk, p.shared_expert_params, p.norm_params)
    x, residual = new(T, 256).to(dtype), new(T, 256).to(dtype)
    with torch.no_grad():
        for _ in range(2):
            out, stream = topk_moe_forward(x, p8, residual=residual)
            rows, normed, h = rms_norm_fp8(x, p.norm_params.weight, 1e-5, residual, with_rows=True)
            scores, indices = router(normed, p.router_params)
            addend = None
            if shared:
                from moe_explore.expert_compute import dense_expert
                addend = dense_expert(normed, p.shared_expert_params.up_weight, p.shared_expert_params.down_weight, "swiglu")
            assert torch.equal(stream, h) and torch.equal(h, x + residual)
            assert torch.equal(out, fp8_expert_compute(rows, scores, indices, p8.expert_params, addend=addend))
            assert torch.isfinite(out).all()
            x, residual = out, stream
        without = topk_moe_forward(x, p8)
        assert torch.equal(without, topk_moe_forward(x, p8))
    # and near the 16-bit layer: each of x, w1, hidden, w2 is off by at most 2^-4 of itself, by 2^-4 / sqrt(3) at the root of the mean
    # square; four such independent errors
    exact, _ = topk_moe_forward(x, p, residual=residual)
    eight, _ = topk_moe_forward(x, p8, residual=residual)
    assert float((eight.float() - exact.float()).norm() / exact.float().norm()) < 4 * 2.0 ** -4 / 3 ** 0.5


@gpu
def test_serving_layer_in_a_graph_and_behind_other_routers(native):
    p, new = make()
    p8 = MOEParams(p.router_params, quantize_experts(p.expert_params), p.num_experts, p.topk, None, p.norm_params)
    x, residual = new(5, 256).bfloat16(), new(5, 256).bfloat16()
    with torch.no_grad():
        topk_moe_forward(x, p8, residual=residual)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, stream = topk_moe_forward(x, p8, residual=residual)
        x.copy_(new(5, 256))
        graph.replay()
        again, stream2 = topk_moe_forward(x, p8, residual=residual)
        assert torch.equal(out, again) and torch.equal(stream, stream2)
        plain = TopkRouterParams(new(256, 16, scale=0.06).bfloat16(), 4)
        q8 = MOEParams(plain, p8.expert_params, 16, 4)
        scores, indices = router(x, plain)
        assert torch.equal(topk_moe_forward(x, q8), fp8_expert_compute(x, scores, indices, p8.expert_params))


@gpu
def test_training_layer_with_its_norm(native):
    """Gradients through norm, residual, router and 16-bit experts against the parts composed by hand in torch."""
    p, new = make()
    x, residual = (new(65, 256).bfloat16().requires_grad_(True) for _ in range(2))
    leaves = [x, residual, p.norm_params.weight.requires_grad_(True), p.router_params.router_weight.requires_grad_(True),
              p.expert_params.weight1.requires_grad_(True), p.expert_params.weight2.requires_grad_(True)]
    d_out, d_stream = new(65, 256).bfloat16(), new(65, 256).bfloat16()
    got = torch.autograd.grad(topk_moe_forward(x, p, residual=residual), leaves, (d_out, d_stream))
    h = x + residual
    hf = h.float()
    normed = (hf * torch.rsqrt(hf.square().mean(-1, keepdim=True) + 1e-5) * p.norm_params.weight.float()).bfloat16()
    bare = MOEParams(p.router_params, p.expert_params, p.num_experts, p.topk)
    want = torch.autograd.grad((topk_moe_torch(normed, bare), h), leaves, (d_out, d_stream))
    for a, b in zip(got, want):   # both round products to 16 bits, the torch form every step between them
        assert a.dtype is b.dtype and float((a.float() - b.float()).norm() / b.float().norm()) < 0.02
    y, s = topk_moe_forward(x, p, residual=residual)
    n, hh = rms_norm(x, p.norm_params.weight, 1e-5, residual)
    assert torch.equal(y, topk_moe_forward(n, bare)) and torch.equal(s, hh)


@gpu
def test_refusals(native):
    p, new = make()
    x = new(3, 256).bfloat16()
    with pytest.raises(ValueError, match="norm_params"):
        topk_moe_forward(x, MOEParams(p.router_params, p.expert_params, 16, 4), residual=x)
    p8 = MOEParams(p.router_params, quantize_experts(p.expert_params), 16, 4, None, p.norm_params)
    with pytest.raises(RuntimeError, match="no backward"):
        topk_moe_forward(x.requires_grad_(True), p8)


@gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning", "ignore::UserWarning")
def test_traces_are_refused(native):
    """A trace would hold the results of the traced input for constants; torch.compile runs the operators between its graphs."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from moe_explore.functional.fp8 import fp8_matmul, quantize_rows, quantize_weight
    from moe_explore.router import grouped_topk_of_logits

    p, new = make()
    experts = quantize_experts(p.expert_params)
    x, w = new(5, 256).bfloat16(), quantize_weight(new(64, 256))
    rows, scores = quantize_rows(x), torch.rand(5, 4, device="cuda").bfloat16()
    ids = torch.arange(4, device="cuda").expand(5, 4).contiguous()
    calls = [lambda x: rms_norm(x, p.norm_params.weight), lambda x: rms_norm_fp8(x, p.norm_params.weight).data.float(),
             lambda x: quantize_rows(x).data.float(), lambda x: fp8_matmul(rows, w) + x[:, :64],
             lambda x: fp8_expert_compute(x, scores, ids, experts),
             lambda x: grouped_topk_of_logits(x[:, :16], p.router_params)[0]]
    with torch.no_grad():
        for call in calls:
            want = call(x)
            with pytest.raises(RuntimeError, match="trace"):
                make_fx(call)(x)
            with pytest.raises(RuntimeError, match="trace"):
                torch.jit.trace(call, (x,), check_trace=False)
            assert torch.equal(call(x), want)
        torch._dynamo.reset()
        both = lambda x: rms_norm(x * 2, p.norm_params.weight) + 1
        assert torch.equal(torch.compile(both, backend="eager")(x), both(x))
        torch._dynamo.reset()


def test_parameters_keep_their_positions():
    """Positional construction as before, the new fields last."""
    p = MOEParams("router", "experts", 8, 2, "shared")
    assert (p.router_params, p.expert_params, p.num_experts, p.topk, p.shared_expert_params, p.norm_params) == ("router", "experts", 8, 2, "shared", None)


@gpu
def test_offsets_past_32_bits(native):
    """Rows, results and logits of more than 2^31 elements: the last rows are what they are by themselves."""
    from moe_explore.functional.fp8 import Fp8Rows, Fp8Weight, fp8_matmul, quantize_rows
    from moe_explore.router import grouped_topk_of_logits

    tail = 300
    rows, k = 270000, 8192
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[-tail:] = torch.randn(tail, k, device="cuda")
    w = torch.ones(k, device="cuda")
    q, y = rms_norm_fp8(x, w, with_rows=True)
    q_tail, y_tail = rms_norm_fp8(x[-tail:].clone(), w, with_rows=True)
    same = lambda a, b: torch.equal(a.data[-tail:].view(torch.uint8), b.data.view(torch.uint8)) and torch.equal(a.scales[-tail:], b.scales)
    assert same(q, q_tail) and torch.equal(y[-tail:], y_tail) and same(quantize_rows(x), quantize_rows(x[-tail:].clone()))
    del x, y
    up = Fp8Weight((torch.randn(264, k, device="cuda") * 20).to(torch.float8_e4m3fn), torch.ones(3, 64, device="cuda"))
    assert torch.equal(fp8_matmul(q, up)[-tail:], fp8_matmul(q_tail, up))                    # deep rows
    wide = Fp8Weight((torch.randn(k, 128, device="cuda") * 20).to(torch.float8_e4m3fn), torch.ones(64, 1, device="cuda"))
    narrow = Fp8Rows(q.data[:, :128].contiguous(), q.scales[:, :1].contiguous())
    few = Fp8Rows(narrow.data[-tail:].clone(), narrow.scales[-tail:].clone())
    assert torch.equal(fp8_matmul(narrow, wide)[-tail:], fp8_matmul(few, wide))              # wide results
    del q, narrow
    logits = torch.randn(2100000, 1024, device="cuda").bfloat16()
    p = GroupedTopkRouterParams(None, 8, num_groups=8, topk_groups=4)
    for a, b in zip(grouped_topk_of_logits(logits, p), grouped_topk_of_logits(logits[-tail:].clone(), p)):
        assert torch.equal(a[-tail:], b)
