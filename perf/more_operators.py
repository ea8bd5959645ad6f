"""A layer's decoding step, products with 4-bit weights and 8-bit activation checkpoints, and their plain forms: what their
performance and results are held against.

A case is a plain dict; ``prepare`` makes what a program has in hand before the call, ``run`` is one pass: in plain torch
operations, or, where ``own`` is true, through the package's public entry points.  Four kinds:

* ``layer``      -- ``topk_moe_forward(..., few_tokens=True)``: residual and norm (if any), router, experts in 16 or 4 bits, fold,
                    for up to 16 tokens;
* ``product``    -- ``int4_matmul``: a few 16-bit rows by 4-bit weights with a scale (and zero point) per group of 32, 64 or 128;
* ``activation`` -- ``activation_fp8`` and its gradient: the (gated) activation of a product that is kept in 8 bits for the
                    backward pass;
* ``experts``    -- ``routed_expert_compute(..., save_fp8=True)`` and its gradients: the experts of a training step that keep the
                    un-activated product in 8 bits and compute the rest again.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 128
TOP = 448.0            # largest e4m3 value
LEAST = 2.0 ** -80     # smallest block maximum a scale is made of
F8 = torch.float8_e4m3fn
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_WEIGHTS = 3 * 64 * 7168 * 2048          # of a layer in 4 bits; a quarter of it in 16 bits
MOST_FLOPS = 18.0 * 8192 * 4 * 2048 * 1408   # the largest listed case

# hidden size d, experts E, slots per token k, expert width I
SMALL = dict(d=2048, E=60, k=4, I=1408)
NARROW = dict(d=2048, E=64, k=8, I=1024)
WIDE = dict(d=4096, E=8, k=2, I=14336)
RANK = dict(d=7168, E=64, k=8, I=2048)


# ------------------------------------------------------------------------------------------------------------ cases
def _layer(T, shape, **more):
    case = dict(op="layer", T=T, act="swiglu", dtype="bf16", bits=16, group=128, zeros=False, router="softmax_first", normalize=False,
                norm=False, residual=False)
    case.update(shape)
    case.update(more)
    return case


def _product(rows, K, N, **more):
    case = dict(op="product", rows=rows, K=K, N=N, group=128, zeros=False, dtype="bf16")
    case.update(more)
    return case


def _activation(rows, I, **more):
    case = dict(op="activation", rows=rows, I=I, act="swiglu", dtype="bf16")
    case.update(more)
    return case


def _experts(T, shape, **more):
    case = dict(op="experts", T=T, act="swiglu", dtype="bf16", skew=0.0)
    case.update(shape)
    case.update(more)
    return case


def listed():
    return [
        # one sequence generating text with a fine-grained layer in 16 bits: the smallest call, latency and launches
        _layer(1, SMALL, name="layer_token"),
        # one sequence on few, wide experts in 4 bits, the layer with its norm and the residual stream
        _layer(1, WIDE, bits=4, router="softmax_after", norm=True, residual=True, name="layer_token_int4"),
        # a decoding batch: every expert is hit by about two tokens
        _layer(16, NARROW, normalize=True, name="layer_batch"),
        # a few drafted tokens through an odd half-precision layer, 4 bits with zero points and small groups
        _layer(7, dict(d=776, E=12, k=3, I=1544), bits=4, group=32, zeros=True, act="geglu", dtype="fp16", name="layer_odd_int4"),
        # a decoding batch on one rank's experts of a very large layer in 4 bits, router by sigmoids in groups with a bias
        _layer(16, RANK, bits=4, router="groups", normalize=True, norm=True, residual=True, name="layer_rank_int4"),
        # one row by a dense projection
        _product(1, 7168, 4096, name="product_token"),
        # an odd number of rows, sizes that are no multiple of any tile, zero points and small groups
        _product(13, 2000, 1416, group=32, zeros=True, dtype="fp16", name="product_odd"),
        # a serving batch by a wide projection
        _product(64, 4096, 28672, group=64, name="product_wide"),
        # the activation of a short sequence through ungated experts, odd sizes
        _activation(333, 1544, act="gelu", dtype="fp16", name="activation_odd"),
        # the activation of a training step of fine-grained experts
        _activation(65536, 1408, name="activation_wide"),
        # a training step with odd sizes and unevenly loaded experts
        _experts(1001, dict(d=776, E=12, k=3, I=1544), act="geglu", dtype="fp16", skew=0.5, name="experts_odd"),
        # a training step of a fine-grained layer: the largest pass
        _experts(8192, SMALL, name="experts_fine"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(("layer", "layer", "product", "activation", "experts"))
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        act = rng.choice(("swiglu", "swiglu", "geglu", "silu", "gelu"))
        if op == "layer":
            router = rng.choice(("softmax_first", "softmax_after", "groups"))
            E = 8 * _log_int(rng, 1, 32) if router == "groups" else _log_int(rng, 4, 256)
            shape = dict(d=8 * _log_int(rng, 32, 896), E=E, k=rng.randint(1, min(8, E // 2)), I=8 * _log_int(rng, 32, 1792))
            bits = rng.choice((16, 4))
            norm = rng.random() < 0.5
            case = _layer(_log_int(rng, 1, 16), shape, act=act, dtype=dtype, bits=bits, group=rng.choice((32, 64, 128)),
                          zeros=bits == 4 and rng.random() < 0.5, router=router, normalize=router != "softmax_after" and rng.random() < 0.5,
                          norm=norm, residual=norm and rng.random() < 0.7)
            if 3 * E * case["d"] * case["I"] > MOST_WEIGHTS * (1 if bits == 4 else 0.25):
                continue
        elif op == "product":
            case = _product(_log_int(rng, 1, 64), 8 * _log_int(rng, 16, 1024), 8 * _log_int(rng, 16, 3584), dtype=dtype,
                            group=rng.choice((32, 64, 128)), zeros=rng.random() < 0.5)
        elif op == "activation":
            case = _activation(_log_int(rng, 1, 65536), 8 * _log_int(rng, 16, 1792), act=act, dtype=dtype)
            if case["rows"] * case["I"] > 65536 * 1408:
                continue
        else:
            E = _log_int(rng, 4, 64)
            shape = dict(d=8 * _log_int(rng, 32, 512), E=E, k=rng.randint(1, min(8, E)), I=8 * _log_int(rng, 32, 512))
            case = _experts(_log_int(rng, 32, 8192), shape, act=act, dtype=dtype, skew=rng.choice((0.0, 0.5)))
            if 3 * E * case["d"] * case["I"] > MOST_WEIGHTS // 8:
                continue
        if work(case)["flops"] <= MOST_FLOPS:
            return case


# ----------------------------------------------------------------------------------------------------------- inputs
def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _weight(g, dtype, *shape):
    """Weights [E, K, N] of standard deviation K^-0.5, made matrix by matrix."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    for m in out:
        m.copy_(_rand(g, *shape[1:]).mul_(shape[1] ** -0.5))
    return out


def _int4(g, case, *shape):
    """4-bit weights [..., N, K]: two values per byte (the even column in the low half), scales per group of columns in the rows' type
    and zero points: element [n, k] is (value - zero) * scale, without zero points (value - 8) * scale."""
    *lead, n, k = shape
    groups = -(-k // case["group"])
    data = torch.randint(0, 256, (*lead, n, k // 2), dtype=torch.uint8, generator=g, device="cuda")
    scales = (0.5 + torch.rand(*lead, n, groups, generator=g, device="cuda")).mul_(k ** -0.5 / 4.6).to(DTYPES[case["dtype"]])
    zeros = None
    if case["zeros"]:
        zeros = torch.randint(4, 12, (*lead, n, groups), dtype=torch.uint8, generator=g, device="cuda")
    return data, scales, zeros


def _gates(case):
    return 2 if "glu" in case["act"] else 1


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=case)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "layer":
        T, d, E, I = case["T"], case["d"], case["E"], case["I"]
        s["x"] = _rand(g, T, d).to(dtype)
        s["residual"] = _rand(g, T, d).to(dtype) if case["residual"] else None
        s["norm"] = (1.0 + 0.1 * _rand(g, d)).to(dtype) if case["norm"] else None
        s["router"] = (1.5 * d ** -0.5 * _rand(g, d, E)).to(torch.float32 if case["router"] == "groups" else dtype)
        s["bias"] = 0.1 * _rand(g, E) if case["router"] == "groups" else None
        if case["bits"] == 4:
            s["up"] = _int4(g, case, E, _gates(case), I, d)
            s["down"] = _int4(g, case, E, d, I)
        else:
            s["up"] = _weight(g, dtype, E, d, _gates(case) * I)   # gate and up columns interleaved
            s["down"] = _weight(g, dtype, E, I, d)
        if own:
            s["params"] = _layer_params(s)
    elif case["op"] == "product":
        s["x"] = _rand(g, case["rows"], case["K"]).to(dtype)
        s["w"] = _int4(g, case, case["N"], case["K"])
        if own:
            _package()
            from moe_explore.functional.int4 import pack_int4
            s["packed"] = pack_int4(*s["w"], group=case["group"])
    elif case["op"] == "activation":
        s["x"] = _rand(g, case["rows"], _gates(case) * case["I"]).to(dtype).requires_grad_(True)
        s["dy"] = _rand(g, case["rows"], case["I"]).to(dtype)
    else:
        T, d, E, I, k = (case[n] for n in ("T", "d", "E", "I", "k"))
        logits = _rand(g, T, E) + case["skew"] * 2.0 * _rand(g, E)
        top = torch.topk(logits, k, dim=-1)
        s["x"] = _rand(g, T, d).to(dtype)
        s["scores"] = torch.softmax(top.values, -1).to(dtype)
        s["indices"] = top.indices
        s["up"] = _weight(g, dtype, E, d, _gates(case) * I)
        s["down"] = _weight(g, dtype, E, I, d)
        s["dy"] = _rand(g, T, d).to(dtype)
        s["most"] = int(torch.bincount(top.indices.reshape(-1), minlength=E).max())
        for name in ("x", "scores", "up", "down"):
            s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
def _best_first(values):
    """Indices in descending order of value, equal values in ascending index."""
    return torch.sort(values, dim=-1, descending=True, stable=True).indices


def _plain_route(c, logits, bias):
    """[T, E] weights, zero where a token does not go, of logits in 64 bits."""
    T, E = logits.shape
    if c["router"] == "groups":
        p = 1.0 / (1.0 + torch.exp(-logits))
        key = p + bias.double()
        groups = key.view(T, 8, E // 8)
        best = torch.sort(groups, dim=-1, descending=True).values[..., :min(2, E // 8)].sum(-1)
        kept = torch.zeros(T, 8, dtype=torch.bool, device=key.device).scatter_(1, _best_first(best)[:, :4], True)
        key = torch.where(kept.repeat_interleave(E // 8, 1), key, torch.full_like(key, -math.inf))
    else:
        p = torch.exp(logits - logits.max(-1, keepdim=True).values)
        key = p
    indices = _best_first(key)[:, :c["k"]]
    picked = p.gather(1, indices)
    if c["router"] == "softmax_first":
        picked = picked / p.sum(-1, keepdim=True)
    if c["router"] == "softmax_after" or c["normalize"]:
        picked = picked / picked.sum(-1, keepdim=True)
    return torch.zeros_like(p).scatter_(1, indices, picked)


def _unpacked(weight, group):
    """fp32 weights [..., N, K] of 4-bit ones."""
    data, scales, zeros = weight
    values = torch.stack((data & 15, data >> 4), -1).flatten(-2).float()
    k = values.size(-1)
    wide = lambda t: t.float().repeat_interleave(group, -1)[..., :k]
    return (values - (8.0 if zeros is None else wide(zeros))) * wide(scales)


def _activate(gate, up, act):
    if act in ("swiglu", "silu"):
        gate = gate / (1.0 + torch.exp(-gate))
    else:
        gate = 0.5 * gate * (1.0 + torch.erf(gate * math.sqrt(0.5)))
    return gate if up is None else gate * up


def _split(pre, act):
    """Gate and up columns of an interleaved product (up None without a gate)."""
    return (pre[..., 0::2], pre[..., 1::2]) if "glu" in act else (pre, None)


def _plain_layer(s):
    c = s["case"]
    x, out = s["x"].float(), {}
    if s["residual"] is not None:
        out["stream"] = (x + s["residual"].float()).to(s["x"].dtype)   # the stream as the next layer sees it
        x = out["stream"].float()
    if s["norm"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["norm"].float()
    weights = _plain_route(c, x.double() @ s["router"].double(), s["bias"]).float()
    y = torch.zeros_like(x)
    for e in range(c["E"]):   # every token through every expert; the weights say which count
        if c["bits"] == 4:
            part = lambda w: tuple(None if t is None else t[e] for t in w)
            pre = x @ _unpacked(part(s["up"]), c["group"]).transpose(-1, -2)   # [gates, T, I]
            gate, up = pre[0], pre[1] if pre.size(0) == 2 else None
            down = _unpacked(part(s["down"]), c["group"]).t()
        else:
            gate, up = _split(x @ s["up"][e].float(), c["act"])
            down = s["down"][e].float()
        y += weights[:, e:e + 1] * (_activate(gate, up, c["act"]) @ down)
    out["y"] = y.to(s["x"].dtype)
    return out


def _plain_product(s):
    return {"out": (s["x"].float() @ _unpacked(s["w"], s["case"]["group"]).t()).to(s["x"].dtype)}


def _kept(pre):
    """16-bit rows as 8 bits give them back, in fp32: e4m3 values and one scale per 128 columns."""
    k = pre.size(-1)
    blocks = -(-k // BLOCK)
    x = torch.nn.functional.pad(pre.float(), (0, blocks * BLOCK - k)).unflatten(-1, (blocks, BLOCK))
    most = x.abs().amax(-1, keepdim=True).clamp_min(LEAST)
    # x * 448 / most with one rounding: 16-bit values often lie in the middle between two 8-bit ones, and stay there
    q = (x * (TOP / 512.0) / most * 512.0).clamp(-TOP, TOP).to(F8)
    return (q.float() * (most / TOP)).flatten(-2)[..., :k]


def _slope(gate, act):
    """Derivative of the activation."""
    if act in ("swiglu", "silu"):
        p = 1.0 / (1.0 + torch.exp(-gate))
        return p * (1.0 + gate * (1.0 - p))
    return 0.5 * (1.0 + torch.erf(gate * math.sqrt(0.5))) + gate * torch.exp(-0.5 * gate * gate) * (2.0 * math.pi) ** -0.5


def _unactivate(kept, dh, act):
    """Gradient of the un-activated product, from what is kept of it."""
    gate, up = _split(kept, act)
    if up is None:
        return dh * _slope(gate, act)
    return torch.stack((dh * up * _slope(gate, act), dh * _activate(gate, None, act)), -1).flatten(-2)


def _plain_activation(s):
    act, x = s["case"]["act"], s["x"].detach()
    return {"y": _activate(*_split(x.float(), act), act).to(x.dtype),
            "dx": _unactivate(_kept(x), s["dy"].float(), act).to(x.dtype)}


def _plain_experts(s):
    c = s["case"]
    T, E, k, act, most = c["T"], c["E"], c["k"], c["act"], s["most"]
    dtype = s["x"].dtype
    owner, order = torch.sort(s["indices"].reshape(-1), stable=True)
    start = torch.searchsorted(owner, torch.arange(E + 1, device=owner.device))
    place = owner * most + torch.arange(T * k, device=owner.device) - start[owner]

    def batched(rows):   # rows in expert order -> [E, most, ...], zeros behind
        return rows.new_zeros(E * most, rows.size(1)).index_copy_(0, place, rows).view(E, most, -1)

    x = batched(s["x"].detach().float()[order // k])
    score = batched(s["scores"].detach().float().reshape(-1, 1)[order])
    up, down = s["up"].detach().float(), s["down"].detach().float()
    pre = torch.bmm(x, up).to(dtype)   # the product that is kept is a 16-bit tensor
    y = torch.bmm(_activate(*_split(pre.float(), act), act), down).flatten(0, 1)[place]
    slots = torch.empty_like(y).index_copy_(0, order, y).view(T, k, -1)
    out = {"y": (slots * s["scores"].detach().float()[..., None]).sum(1).to(dtype)}
    dy = batched(s["dy"].float()[order // k])
    kept = _kept(pre)
    h = _activate(*_split(kept, act), act)
    du = torch.bmm(dy, down.transpose(1, 2))
    d_pre = _unactivate(kept, score * du, act)
    d_score = (du * h).sum(-1).flatten()[place]
    out["d_scores"] = torch.empty_like(d_score).index_copy_(0, order, d_score).view(T, k).to(dtype)
    dx = torch.bmm(d_pre, up.transpose(1, 2)).flatten(0, 1)[place]
    out["dx"] = torch.empty_like(dx).index_copy_(0, order, dx).view(T, k, -1).sum(1).to(dtype)
    out["d_up"] = torch.bmm(x.transpose(1, 2), d_pre).to(dtype)
    out["d_down"] = torch.bmm((score * h).transpose(1, 2), dy).to(dtype)
    return out


# --------------------------------------------------------------------------------------------- the package's calls
def _package():
    path = os.path.join(os.getcwd(), "moe-explore_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


def _layer_params(s):
    _package()
    from moe_explore.functional.int4 import pack_experts_int4
    from moe_explore.params import GroupedTopkRouterParams, MLPParams, MOEParams, RMSNormParams, TopkRouterParams
    c = s["case"]
    if c["bits"] == 4:
        experts = pack_experts_int4(s["up"], s["down"], c["act"], group=c["group"])
    else:
        experts = MLPParams(s["up"], s["down"], c["act"])
    if c["router"] == "groups":
        router = GroupedTopkRouterParams(s["router"], c["k"], bias=s["bias"], num_groups=8, topk_groups=4,
                                         group_best=min(2, c["E"] // 8), normalize_routing=c["normalize"])
    else:
        router = TopkRouterParams(s["router"], c["k"], c["router"] == "softmax_first", c["normalize"])
    norm = None if s["norm"] is None else RMSNormParams(s["norm"], EPS)
    return MOEParams(router, experts, c["E"], c["k"], None, norm)


def _own_layer(s):
    from moe_explore.functional.topk_moe import topk_moe_forward
    with torch.no_grad():
        out = topk_moe_forward(s["x"], s["params"], residual=s["residual"], few_tokens=True)
    return {"y": out} if s["residual"] is None else {"y": out[0], "stream": out[1]}


def _own_product(s):
    from moe_explore.functional.int4 import int4_matmul
    return {"out": int4_matmul(s["x"], s["packed"])}


def _own_activation(s):
    from moe_explore.functional.activation_fp8 import activation_fp8
    y = activation_fp8(s["x"], s["case"]["act"])
    dx, = torch.autograd.grad(y, s["x"], s["dy"])
    return {"y": y, "dx": dx}


def _own_experts(s):
    from moe_explore.expert_compute import routed_expert_compute
    c = s["case"]
    leaves = (s["x"], s["scores"], s["up"], s["down"])
    y = routed_expert_compute(*leaves, s["indices"], c["E"], c["k"], c["act"], save_fp8=True)
    grads = torch.autograd.grad(y, leaves, s["dy"])
    return {"y": y, "dx": grads[0], "d_scores": grads[1], "d_up": grads[2], "d_down": grads[3]}


_PLAIN = {"layer": _plain_layer, "product": _plain_product, "activation": _plain_activation, "experts": _plain_experts}
_OWN = {"layer": _own_layer, "product": _own_product, "activation": _own_activation, "experts": _own_experts}


def run(state):
    if own:
        _package()
        return _OWN[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    if op == "product":
        rows, K, N = case["rows"], case["K"], case["N"]
        per_group = 3 if case["zeros"] else 2
        return {"bytes": 2 * rows * (K + N) + N * K / 2 + N * -(-K // case["group"]) * per_group, "flops": 2.0 * rows * K * N}
    if op == "activation":
        rows, I, n1 = case["rows"], case["I"], _gates(case) * case["I"]
        # forward: the product, its activation, what is kept; backward: that again, the incoming gradient, its own
        return {"bytes": rows * (2 * n1 + 2 * I + 2 * (n1 + 4 * -(-n1 // BLOCK)) + 2 * I + 2 * n1), "flops": 30.0 * rows * I}
    T, d, E, I, k, gates = (*(case[n] for n in ("T", "d", "E", "I", "k")), _gates(case))
    hit = E * (1.0 - (1.0 - k / E) ** T)
    weights = (gates + 1) * d * I
    if op == "layer":
        each = 2.0 if case["bits"] == 16 else 0.5 + (3 if case["zeros"] else 2) / case["group"]
        n = hit * weights * each + d * E * (4 if case["router"] == "groups" else 2) + 4 * T * d + (4 * T * d if case["residual"] else 0)
        return {"bytes": n, "flops": 2.0 * T * (k * weights + d * E)}
    # forward: x, weights, scores, indices, y; backward: dy, x, weights, gradients of all four; the kept product written and read
    n = 2 * T * d * 5 + 2 * hit * weights * 2 + 2 * E * weights + T * k * (2 + 8 + 2) + 2 * T * k * gates * I * (1 + 4 / BLOCK)
    return {"bytes": n, "flops": 6.0 * T * k * weights}


# ------------------------------------------------------------------------------------------------ 64-bit definitions
def _exact_route(c, logits, bias):
    """(weights [T, k], experts [T, k])"""
    T, E = logits.shape
    if c["router"] == "groups":
        prob = torch.special.expit(logits)
        key = prob + bias.double()
        width = E // 8
        value = torch.topk(key.reshape(-1, width), min(2, width)).values.sum(1).view(T, 8)
        dropped = torch.argsort(-value, dim=1, stable=True)[:, 4:]
        columns = (dropped[..., None] * width + torch.arange(width, device=key.device)).flatten(1)
        key = key.scatter(1, columns, -math.inf)
    else:
        prob = torch.softmax(logits, -1)
        key = logits
    chosen = torch.argsort(-key, dim=1, stable=True)[:, :c["k"]]
    if c["router"] == "softmax_after":
        return torch.softmax(torch.take_along_dim(logits, chosen, 1), -1), chosen
    w = torch.take_along_dim(prob, chosen, 1)
    return w / w.sum(1, keepdim=True) if c["normalize"] else w, chosen


def _exact_int4(weight, group):
    data, scales, zeros = weight
    n, k = data.size(-2), 2 * data.size(-1)
    w = torch.empty(*data.shape[:-1], k, dtype=torch.float64, device=data.device)
    w[..., 0::2] = data % 16
    w[..., 1::2] = torch.div(data, 16, rounding_mode="floor")
    at = torch.arange(k, device=data.device) // group
    return (w - (8 if zeros is None else zeros.double()[..., at])) * scales.double()[..., at]


def _exact_act(z, act):
    return z * (torch.special.expit(z) if act in ("swiglu", "silu") else torch.special.ndtr(z))


def _exact_hidden(pre, act):
    return _exact_act(pre[..., ::2], act) * pre[..., 1::2] if "glu" in act else _exact_act(pre, act)


def _exact_layer(s):
    c = s["case"]
    x, out = s["x"].double(), {}
    if c["residual"]:
        x = x + s["residual"].double()
        out["stream"] = x
        x = x.to(s["x"].dtype).double()
    if c["norm"]:
        x = x / (torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / c["d"] + EPS).sqrt() * s["norm"].double()
    w, chosen = _exact_route(c, x @ s["router"].double(), s["bias"])
    y = torch.zeros_like(x)
    for e in chosen.unique().tolist():
        token, slot = (chosen == e).nonzero(as_tuple=True)
        if c["bits"] == 4:
            pick = lambda t: tuple(None if v is None else v[e] for v in t)
            pre = torch.stack([x[token] @ m.T for m in _exact_int4(pick(s["up"]), c["group"])], -1).flatten(1)
            down = _exact_int4(pick(s["down"]), c["group"]).T
        else:
            pre, down = x[token] @ s["up"][e].double(), s["down"][e].double()
        y.index_add_(0, token, w[token, slot, None] * (_exact_hidden(pre, c["act"]) @ down))
    out["y"] = y
    return out


def _exact_product(s):
    return {"out": s["x"].double() @ _exact_int4(s["w"], s["case"]["group"]).T}


def _exact_kept(pre):
    """What 8 bits give back of 16-bit rows: each value replaced by the multiple of its block's scale that they hold."""
    x = pre.double()
    k = torch.arange(x.size(1), device=x.device) // BLOCK
    top = torch.zeros(x.size(0), int(k[-1]) + 1, dtype=torch.float64, device=x.device)
    top.scatter_reduce_(1, k.expand_as(x), x.abs(), "amax")
    top = top.clamp_min(LEAST)[:, k]
    return (x * TOP / top).clamp(-TOP, TOP).to(F8).double() * (top / TOP)


def _exact_gradient(kept, dh, act):
    with torch.enable_grad():
        z = kept.detach().requires_grad_(True)
        return torch.autograd.grad(_exact_hidden(z, act), z, dh)[0]


def _exact_activation(s):
    act, x = s["case"]["act"], s["x"].detach()
    y = torch.empty(s["dy"].shape, dtype=torch.float64, device=x.device)
    dx = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for a in range(0, x.size(0), 8192):
        rows = slice(a, a + 8192)
        y[rows] = _exact_hidden(x[rows].double(), act)
        dx[rows] = _exact_gradient(_exact_kept(x[rows]), s["dy"][rows].double(), act)
    return {"y": y, "dx": dx}


def _exact_experts(s):
    c = s["case"]
    act, dtype = c["act"], s["x"].dtype
    x, scores, dy = s["x"].detach().double(), s["scores"].detach().double(), s["dy"].double()
    out = {"y": torch.zeros_like(x), "dx": torch.zeros_like(x), "d_scores": torch.zeros_like(scores),
           "d_up": torch.zeros(s["up"].shape, dtype=torch.float64, device="cuda"),
           "d_down": torch.zeros(s["down"].shape, dtype=torch.float64, device="cuda")}
    for e in range(c["E"]):
        token, slot = (s["indices"] == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        up, down = s["up"][e].detach().double(), s["down"][e].detach().double()
        w = scores[token, slot, None]
        pre = (x[token] @ up).to(dtype)
        out["y"].index_add_(0, token, w * (_exact_hidden(pre.double(), act) @ down))
        kept = _exact_kept(pre)
        h = _exact_hidden(kept, act)
        du = dy[token] @ down.T
        d_pre = _exact_gradient(kept, w * du, act)
        out["d_scores"][token, slot] = torch.einsum("ri,ri->r", du, h)
        out["dx"].index_add_(0, token, d_pre @ up.T)
        out["d_up"][e] = x[token].T @ d_pre
        out["d_down"][e] = (w * h).T @ dy[token]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"layer": _exact_layer, "product": _exact_product, "activation": _exact_activation, "experts": _exact_experts}[case["op"]](s)
