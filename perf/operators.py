"""The serving operators around the experts, and their plain forms: what their performance and results are held against.

A case is a plain dict; ``prepare`` makes what a program has in hand before the call, ``run`` is one pass: in plain torch
operations, or, where ``own`` is true, through the package's public entry points.  Four kinds:

* ``route``   -- ``grouped_topk_of_logits``: scores, bias for balance, groups, top-k, renormalised weights; with ``train`` also
                 the gradient of the logits;
* ``norm``    -- ``rms_norm`` / ``rms_norm_fp8``: the residual's addition, root-mean-square norm, and for serving its result in 8
                 bits with a scale for each block of 128; with ``train`` the gradients of input, residual and weight;
* ``product`` -- ``fp8_matmul`` / ``m_grouped_gemm`` of 8-bit rows (a scale per row and 128 columns) and 8-bit weights (a scale per
                 128 x 128 block), dense or grouped by expert;
* ``experts`` -- ``fp8_expert_compute``: rows to 8 bits, gate/up product, activation, 8 bits again, down product, weighted fold.
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
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_FLOPS = 6.0 * 8192 * 4096 * 14336   # the largest listed case
MOST_WEIGHTS = 3 * 8 * 4096 * 14336


# ------------------------------------------------------------------------------------------------------------ cases
def _route(T, E, G, keep, k, **more):
    case = dict(op="route", T=T, E=E, G=G, keep=keep, k=k, score="sigmoid", bias=True, best=2, normalize=True, scale=1.0,
                logits="fp32", out="bf16", train=False)
    case.update(more)
    return case


def _norm(T, d, **more):
    case = dict(op="norm", T=T, d=d, dtype="bf16", weight="bf16", residual=True, train=False)
    case.update(more)
    return case


def _product(rows, E, K, N, **more):
    case = dict(op="product", rows=rows, E=E, K=K, N=N, out="bf16", skew=0.0)
    case.update(more)
    return case


def _experts(T, E, k, d, I, **more):
    case = dict(op="experts", T=T, E=E, k=k, d=d, I=I, act="swiglu", dtype="bf16", skew=0.0)
    case.update(more)
    return case


def listed():
    return [
        # one sequence generating text: latency and launches
        _route(1, 256, 8, 4, 8, scale=2.5, name="route_token"),
        # a long prompt through the same router
        _route(16384, 256, 8, 4, 8, scale=2.5, name="route_prompt"),
        # training of a softmax router without a bias on an odd number of tokens and experts
        _route(4099, 60, 4, 2, 4, score="softmax", bias=False, best=1, logits="bf16", train=True, name="route_train"),
        # the norm before the experts, one sequence
        _norm(1, 4096, name="norm_token"),
        # the same for a prompt of a very wide model
        _norm(8192, 7168, name="norm_prompt"),
        # the norm of a training step, odd token count, fp32 weight
        _norm(8191, 2048, train=True, weight="fp32", name="norm_train"),
        # a dense projection for a serving batch: the weight is read for 64 rows
        _product(64, 1, 7168, 4096, name="product_batch"),
        # a grouped product in the middle of a prompt, sizes that are no multiple of any tile, unevenly loaded experts
        _product(16391, 60, 2000, 1416, skew=0.5, out="fp16", name="product_grouped"),
        # one token through few, wide experts
        _experts(1, 8, 2, 4096, 14336, name="experts_token"),
        # a decoding batch on one rank's fine-grained experts: every weight is read for about 16 rows
        _experts(128, 64, 8, 7168, 2048, name="experts_batch"),
        # a prompt of odd length, uneven load, a half-precision model with the other gate
        _experts(3001, 64, 8, 2048, 1024, act="geglu", dtype="fp16", skew=0.5, name="experts_prompt"),
        # a large prefill batch on few, wide experts: the largest pass
        _experts(4096, 8, 2, 4096, 14336, name="experts_prefill"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(("route", "norm", "product", "experts"))
        if op == "route":
            G = rng.choice((1, 1, 2, 4, 5, 8))
            E = G * _log_int(rng, 2, 512 // G)
            keep = rng.randint(1, G)
            train = rng.random() < 0.5
            case = _route(_log_int(rng, 1, 16384), E, G, keep, rng.randint(1, min(16, keep * (E // G))),
                          score=rng.choice(("sigmoid", "softmax")), bias=rng.random() < 0.6, best=rng.choice((1, 2)),
                          normalize=rng.random() < 0.7, scale=rng.choice((1.0, 2.5)), logits=rng.choice(("fp32", "bf16")),
                          out=rng.choice(("bf16", "fp16", "fp32")), train=train)
            if train and case["k"] == 1:
                case["normalize"] = False   # a single renormalised weight is a constant: nothing to train
        elif op == "norm":
            train = rng.random() < 0.5
            case = _norm(_log_int(rng, 1, 16384), 16 * _log_int(rng, 8, 512), dtype=rng.choice(("bf16", "bf16", "fp16")),
                         weight=rng.choice(("same", "fp32")), residual=rng.random() < 0.7, train=train)
            if case["weight"] == "same":
                case["weight"] = case["dtype"]
            if case["T"] * case["d"] > 8192 * 7168:
                continue
        elif op == "product":
            E = rng.choice((1, 1, _log_int(rng, 2, 64)))
            case = _product(_log_int(rng, 1, 32768), E, 16 * _log_int(rng, 16, 512), 8 * _log_int(rng, 32, 1024),
                            out=rng.choice(("bf16", "fp16")), skew=rng.choice((0.0, 0.5)) if E > 1 else 0.0)
        else:
            E = _log_int(rng, 2, 64)
            case = _experts(_log_int(rng, 1, 8192), E, rng.randint(1, min(8, E)), 16 * _log_int(rng, 16, 512),
                            16 * _log_int(rng, 16, 256), act=rng.choice(("swiglu", "swiglu", "geglu", "silu", "gelu")),
                            dtype=rng.choice(("bf16", "bf16", "fp16")), skew=rng.choice((0.0, 0.5)))
        weights = (case["E"] * case["K"] * case["N"] if op == "product" else
                   3 * case["E"] * case["d"] * case["I"] if op == "experts" else 0)
        if work(case)["flops"] <= MOST_FLOPS and weights <= MOST_WEIGHTS:
            return case


# ----------------------------------------------------------------------------------------------------------- inputs
def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _fp8_weight(g, *shape):
    """Weights of standard deviation K^-0.5 as 8-bit values and one fp32 scale per 128 x 128 block of the last two axes."""
    n, k = shape[-2:]
    data = _rand(g, *shape).mul_(96.0).clamp_(-TOP, TOP).to(F8)
    scales = 0.5 + torch.rand(*shape[:-2], -(-n // BLOCK), -(-k // BLOCK), generator=g, device="cuda")
    return data, scales.mul_(k ** -0.5 / 96.0)


def _fp8_rows(g, rows, k):
    data = _rand(g, rows, k).mul_(128.0).clamp_(-TOP, TOP).to(F8)
    return data, (0.5 + torch.rand(rows, -(-k // BLOCK), generator=g, device="cuda")).div_(128.0)


def _popularity(case, g):
    return case["skew"] * 2.0 * _rand(g, case["E"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=case)
    if case["op"] == "route":
        T, E = case["T"], case["E"]
        s["logits"] = (1.5 * _rand(g, T, E)).to(DTYPES[case["logits"]])
        s["bias"] = 0.1 * _rand(g, E) if case["bias"] else None
        if case["train"]:
            s["logits"].requires_grad_(True)
            s["d_scores"] = _rand(g, T, case["k"]).to(DTYPES[case["out"]])
    elif case["op"] == "norm":
        T, d, dtype = case["T"], case["d"], DTYPES[case["dtype"]]
        s["x"] = _rand(g, T, d).to(dtype)
        s["residual"] = (2.0 * _rand(g, T, d)).to(dtype) if case["residual"] else None
        s["weight"] = (1.0 + 0.1 * _rand(g, d)).to(DTYPES[case["weight"]])
        if case["train"]:
            s["dy"] = _rand(g, T, d).to(dtype)
            s["dh"] = _rand(g, T, d).to(dtype) if case["residual"] else None
            for name in ("x", "residual", "weight"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    elif case["op"] == "product":
        rows, E = case["rows"], case["E"]
        s["x"], s["x_scales"] = _fp8_rows(g, rows, case["K"])
        s["w"], s["w_scales"] = _fp8_weight(g, E, case["N"], case["K"])
        owner = torch.multinomial(torch.softmax(_popularity(case, g), 0), rows, True, generator=g)
        counts = torch.bincount(owner, minlength=E)
        s["groups"] = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
        s["most"] = int(counts.max())
    else:
        T, E, k = case["T"], case["E"], case["k"]
        s["x"] = _rand(g, T, case["d"]).to(DTYPES[case["dtype"]])
        gates = 2 if "glu" in case["act"] else 1
        s["up"], s["up_scales"] = _fp8_weight(g, E, gates, case["I"], case["d"])
        s["down"], s["down_scales"] = _fp8_weight(g, E, case["d"], case["I"])
        logits = _rand(g, T, E) + _popularity(case, g)
        top = torch.topk(logits, k, dim=-1)
        s["scores"] = torch.softmax(top.values, -1).to(DTYPES[case["dtype"]])
        s["indices"] = top.indices
        s["most"] = int(torch.bincount(top.indices.reshape(-1), minlength=E).max())
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
def _best_first(values):
    """Indices in descending order of value, equal values in ascending index."""
    return torch.sort(values, dim=-1, descending=True, stable=True).indices


def _plain_route(s):
    c = s["case"]
    T, E, G, k = c["T"], c["E"], c["G"], c["k"]
    logits = s["logits"].detach().double()   # values next to the border of the selection
    if c["score"] == "sigmoid":
        p = 1.0 / (1.0 + torch.exp(-logits))
    else:
        p = torch.exp(logits - logits.max(-1, keepdim=True).values)
        p = p / p.sum(-1, keepdim=True)
    key = p if s["bias"] is None else p + s["bias"].double()
    groups = key.view(T, G, E // G)
    group_score = torch.sort(groups, dim=-1, descending=True).values[..., :c["best"]].sum(-1)
    kept = torch.zeros(T, G, dtype=torch.bool, device=key.device).scatter_(1, _best_first(group_score)[:, :c["keep"]], True)
    open_ = kept.repeat_interleave(E // G, 1)
    indices = _best_first(torch.where(open_, key, torch.full_like(key, -math.inf)))[:, :k]
    picked = p.gather(1, indices)
    total = picked.sum(-1, keepdim=True) + 1e-20
    weights = picked / total if c["normalize"] else picked
    out = {"scores": (weights * c["scale"]).to(DTYPES[c["out"]]), "indices": indices}
    if c["train"]:
        d = s["d_scores"].double() * c["scale"]
        if c["normalize"]:
            d = (d - (d * weights).sum(-1, keepdim=True)) / total
        d_all = torch.zeros_like(p).scatter_(1, indices, d)
        if c["score"] == "sigmoid":
            d_logits = d_all * p * (1.0 - p)
        else:
            d_logits = p * (d_all - (d_all * p).sum(-1, keepdim=True))
        out["d_logits"] = d_logits.to(s["logits"].dtype)
    return out


def _blocks(x):
    """[..., K] -> [..., blocks, 128], zeros behind the last column."""
    k = x.size(-1)
    blocks = -(-k // BLOCK)
    return torch.nn.functional.pad(x, (0, blocks * BLOCK - k)).unflatten(-1, (blocks, BLOCK))


def _to_fp8(x):
    """8-bit values and one scale per 128 columns of x [..., K] in fp32."""
    blocks = _blocks(x)
    most = blocks.abs().amax(-1, keepdim=True).clamp_min(LEAST)
    # x * 448 / most with one rounding: 16-bit values often lie in the middle between two 8-bit ones, and stay there
    q = (blocks * (TOP / 512.0) / most * 512.0).clamp(-TOP, TOP).to(F8)
    return q.flatten(-2)[..., :x.size(-1)], most[..., 0] / TOP


def _plain_norm(s):
    c = s["case"]
    x, dtype = s["x"].detach().float(), s["x"].dtype
    w = s["weight"].detach().float()
    out = {}
    if s["residual"] is not None:
        out["h"] = (x + s["residual"].detach().float()).to(dtype)   # the stream as the next layer sees it
        x = out["h"].float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    y = x * r * w
    out["y"] = y.to(dtype)
    if not c["train"]:
        q, out["scales"] = _to_fp8(y)
        out["q"] = q.contiguous()
        return out
    n, dy = x * r, s["dy"].float()
    g = dy * w
    dx = r * (g - n * (g * n).mean(-1, keepdim=True))
    if s["residual"] is not None:
        dx = dx + s["dh"].float()
    out["dx"] = dx.to(dtype)
    out["dw"] = (dy * n).sum(0, dtype=torch.float64).to(s["weight"].dtype)
    return out


def _rows_of(data, scales):
    """fp32 rows of 8-bit data [R, K] with scales [R, blocks]."""
    return (_blocks(data.float()) * scales[..., None]).flatten(-2)[..., :data.size(-1)]


def _weight_of(data, scales):
    """fp32 weights of 8-bit data [..., N, K] with scales per 128 x 128 block."""
    n, k = data.shape[-2:]
    grid = scales.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]
    return data.float() * grid


def _batched(rows, start, owner, most):
    """Rows in expert order -> [E, most, K], and where each went."""
    E = start.numel() - 1
    place = owner * most + torch.arange(rows.size(0), device=rows.device) - start[owner]
    wide = rows.new_zeros(E * most, rows.size(1)).index_copy_(0, place, rows)
    return wide.view(E, most, -1), place


def _plain_product(s):
    c = s["case"]
    rows, w = _rows_of(s["x"], s["x_scales"]), _weight_of(s["w"], s["w_scales"])
    start = s["groups"].long()
    owner = torch.searchsorted(start[1:].contiguous(), torch.arange(c["rows"], device=rows.device), right=True)
    wide, place = _batched(rows, start, owner, s["most"])
    out = torch.bmm(wide, w.transpose(1, 2)).flatten(0, 1)[place]
    return {"out": out.to(DTYPES[c["out"]])}


def _activate(up, act):
    """[E, gates, rows, I] -> [E, rows, I]."""
    gate = up[:, 0]
    if act in ("swiglu", "silu"):
        gate = gate / (1.0 + torch.exp(-gate))
    else:
        gate = 0.5 * gate * (1.0 + torch.erf(gate * math.sqrt(0.5)))
    return gate * up[:, 1] if "glu" in act else gate


def _plain_experts(s):
    c = s["case"]
    T, E, k = c["T"], c["E"], c["k"]
    owner, order = torch.sort(s["indices"].reshape(-1), stable=True)
    start = torch.searchsorted(owner, torch.arange(E + 1, device=owner.device))
    rows = _rows_of(*_to_fp8(s["x"].float()))[order // k]
    wide, place = _batched(rows, start, owner, s["most"])
    up = torch.matmul(wide[:, None], _weight_of(s["up"], s["up_scales"]).transpose(-1, -2))
    q, scales = _to_fp8(_activate(up, c["act"]))
    hidden = _rows_of(q, scales)
    down = torch.bmm(hidden, _weight_of(s["down"], s["down_scales"]).transpose(1, 2)).flatten(0, 1)[place]
    slots = torch.empty_like(down).index_copy_(0, order, down).view(T, k, -1)
    return {"out": (slots * s["scores"].float()[..., None]).sum(1).to(s["x"].dtype)}


# --------------------------------------------------------------------------------------------- the package's calls
def _package():
    path = os.path.join(os.getcwd(), "moe-explore_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


def _own_route(s):
    from moe_explore.params import GroupedTopkRouterParams
    from moe_explore.router import grouped_topk_of_logits
    c = s["case"]
    params = GroupedTopkRouterParams(None, c["k"], bias=s["bias"], num_groups=c["G"], topk_groups=c["keep"],
                                     group_best=c["best"], score_function=c["score"], normalize_routing=c["normalize"],
                                     scale=c["scale"])
    scores, indices = grouped_topk_of_logits(s["logits"], params, DTYPES[c["out"]])
    out = {"scores": scores, "indices": indices}
    if c["train"]:
        out["d_logits"], = torch.autograd.grad(scores, s["logits"], s["d_scores"])
    return out


def _own_norm(s):
    from moe_explore.functional.rms_norm import rms_norm, rms_norm_fp8
    if not s["case"]["train"]:
        if s["residual"] is None:
            rows, y = rms_norm_fp8(s["x"], s["weight"], with_rows=True)
            return {"y": y, "q": rows.data, "scales": rows.scales}
        rows, y, h = rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], with_rows=True)
        return {"h": h, "y": y, "q": rows.data, "scales": rows.scales}
    if s["residual"] is None:
        y = rms_norm(s["x"], s["weight"])
        dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    y, h = rms_norm(s["x"], s["weight"], residual=s["residual"])
    dx, dr, dw = torch.autograd.grad((y, h), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dh"]))
    return {"h": h, "y": y, "dx": dx, "dw": dw}


def _own_product(s):
    from moe_explore.functional.fp8 import Fp8Rows, Fp8Weight, fp8_matmul
    from moe_explore.triton_kernels.m_grouped_gemm import MGroupedGEMMParams, m_grouped_gemm
    c = s["case"]
    rows, weight = Fp8Rows(s["x"], s["x_scales"], DTYPES[c["out"]]), Fp8Weight(s["w"], s["w_scales"])
    if c["E"] == 1:
        return {"out": fp8_matmul(rows, weight)}
    return {"out": m_grouped_gemm(rows, MGroupedGEMMParams(weight, s["groups"], None, False, False, c["rows"], 1))}


def _own_experts(s):
    from moe_explore.expert_compute import fp8_expert_compute
    from moe_explore.functional.fp8 import Fp8Weight
    from moe_explore.params import Fp8ExpertParams
    params = Fp8ExpertParams(Fp8Weight(s["up"], s["up_scales"]), Fp8Weight(s["down"], s["down_scales"]), s["case"]["act"])
    return {"out": fp8_expert_compute(s["x"], s["scores"], s["indices"], params)}


_PLAIN = {"route": _plain_route, "norm": _plain_norm, "product": _plain_product, "experts": _plain_experts}
_OWN = {"route": _own_route, "norm": _own_norm, "product": _own_product, "experts": _own_experts}


def run(state):
    if own:
        _package()
        return _OWN[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        n = T * E * size[case["logits"]] + T * k * (8 + size[case["out"]]) + (4 * E if case["bias"] else 0)
        if case["train"]:
            n += T * k * size[case["out"]] + T * E * size[case["logits"]]
        return {"bytes": n, "flops": 8 * T * E}
    if case["op"] == "norm":
        T, d = case["T"], case["d"]
        n = 2 * T * d * (4 if case["residual"] else 2) + d * size[case["weight"]]     # x, residual, h, y
        if case["train"]:
            n += 2 * T * d * (3 if case["residual"] else 2) + d * size[case["weight"]]  # dy, dh, dx
        else:
            n += T * d + 4 * T * -(-d // BLOCK)
        return {"bytes": n, "flops": T * d * (14 if case["train"] else 6)}
    if case["op"] == "product":
        rows, E, K, N = case["rows"], case["E"], case["K"], case["N"]
        hit = E * (1.0 - (1.0 - 1.0 / E) ** rows)
        n = rows * (K + 4 * -(-K // BLOCK) + 2 * N) + hit * N * K * (1 + 4 / BLOCK ** 2)
        return {"bytes": n, "flops": 2.0 * rows * K * N}
    T, E, k, d, I = (case[n] for n in ("T", "E", "k", "d", "I"))
    gates = 2 if "glu" in case["act"] else 1
    hit = E * (1.0 - (1.0 - k / E) ** T)
    n = 4 * T * d + T * k * 10 + hit * (gates + 1) * d * I * (1 + 4 / BLOCK ** 2)
    return {"bytes": n, "flops": 2.0 * T * k * d * I * (gates + 1)}


# ------------------------------------------------------------------------------------------------ 64-bit definitions
def _exact_route(s):
    c = s["case"]
    x = s["logits"].detach().to(torch.float64)
    prob = torch.special.expit(x) if c["score"] == "sigmoid" else torch.softmax(x, -1)
    key = prob.clone() if s["bias"] is None else prob + s["bias"]
    width = c["E"] // c["G"]
    value = torch.topk(key.reshape(-1, width), c["best"]).values.sum(1).view(c["T"], c["G"])
    dropped = torch.argsort(-value, dim=1, stable=True)[:, c["keep"]:]
    columns = (dropped[..., None] * width + torch.arange(width, device=x.device)).flatten(1)
    chosen = torch.argsort(-key.scatter(1, columns, -math.inf), dim=1, stable=True)[:, :c["k"]]
    w = torch.take_along_dim(prob, chosen, 1)
    total = w.sum(1, keepdim=True)
    share = w / total if c["normalize"] else w
    out = {"scores": c["scale"] * share, "indices": None}
    if c["train"]:
        up = c["scale"] * s["d_scores"].to(torch.float64)
        if c["normalize"]:
            up = up / total - (up * w).sum(1, keepdim=True) / total ** 2
        dense = torch.zeros_like(prob)
        dense.scatter_add_(1, chosen, up)
        out["d_logits"] = (dense * prob * (1 - prob) if c["score"] == "sigmoid"
                           else dense * prob - prob * torch.einsum("te,te->t", dense, prob)[:, None])
    return out


def _exact_norm(s):
    c = s["case"]
    h = s["x"].detach().to(torch.float64)
    w = s["weight"].detach().to(torch.float64)
    out = {}
    if s["residual"] is not None:
        h = h + s["residual"].detach().to(torch.float64)
        out["h"] = h
        h = h.to(s["x"].dtype).to(torch.float64)
    rms = (torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / c["d"] + 1e-6).sqrt()
    y = h / rms * w
    out["y"] = y
    if not c["train"]:
        columns = torch.arange(c["d"], device=h.device) // BLOCK
        top = torch.zeros(c["T"], int(columns[-1]) + 1, dtype=torch.float64, device=h.device)
        top.scatter_reduce_(1, columns.expand_as(y), y.abs(), "amax")
        out["scales"] = top / TOP
        out["q"] = y / out["scales"][:, columns]
        return out
    dy = s["dy"].to(torch.float64)
    inner = torch.einsum("td,d,td->t", dy, w, h)[:, None]
    out["dx"] = dy * w / rms - h * inner / (c["d"] * rms ** 3) + (0 if s["residual"] is None else s["dh"].to(torch.float64))
    out["dw"] = torch.einsum("td,td->d", dy, h / rms)
    return out


def _expand(data, scales):
    k = torch.arange(data.size(-1), device=data.device) // BLOCK
    return data.to(torch.float64) * scales.to(torch.float64)[..., k]


def _expand_weight(data, scales):
    n = torch.arange(data.size(-2), device=data.device) // BLOCK
    return _expand(data, scales[..., n, :])


def _eight_bits(x):
    """Each value replaced by the multiple of its block's scale that 8 bits hold."""
    k = torch.arange(x.size(1), device=x.device) // BLOCK
    top = torch.zeros(x.size(0), int(k[-1]) + 1, dtype=torch.float64, device=x.device)
    top.scatter_reduce_(1, k.expand_as(x), x.abs(), "amax")
    top = top.clamp_min(LEAST)[:, k]
    return (x * TOP / top).clamp(-TOP, TOP).to(F8).to(torch.float64) * (top / TOP)


def _exact_product(s):
    c = s["case"]
    ends = s["groups"].tolist()
    out = torch.empty(c["rows"], c["N"], dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        a, b = ends[e], ends[e + 1]
        out[a:b] = _expand(s["x"][a:b], s["x_scales"][a:b]) @ _expand_weight(s["w"][e], s["w_scales"][e]).T
    return {"out": out}


def _exact_experts(s):
    c = s["case"]
    out = torch.zeros(c["T"], c["d"], dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        token, slot = (s["indices"] == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        x = _eight_bits(s["x"][token].to(torch.float64))
        first = x @ _expand_weight(s["up"][e, 0], s["up_scales"][e, 0]).T
        hidden = first * (torch.special.expit(first) if c["act"] in ("swiglu", "silu") else torch.special.ndtr(first))
        if "glu" in c["act"]:
            hidden = hidden * (x @ _expand_weight(s["up"][e, 1], s["up_scales"][e, 1]).T)
        y = _eight_bits(hidden) @ _expand_weight(s["down"][e], s["down_scales"][e]).T
        out.index_add_(0, token, y * s["scores"][token, slot].to(torch.float64)[:, None])
    return {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "norm": _exact_norm, "product": _exact_product, "experts": _exact_experts}[case["op"]](s)
