"""Rows, weights, products and experts in 8 bits against plain forms in 64 bits; refusals."""
import glob
import math
import os
import re

import pytest
import torch

from conftest import ROOT
from moe_explore.functional.fp8 import BLOCK, DTYPE, LEAST, Fp8Rows, Fp8Weight, fp8_matmul, quantize_experts, quantize_rows, quantize_weight
from moe_explore.params import Fp8ExpertParams, GLUParams, MLPParams
from moe_explore.triton_kernels.m_grouped_gemm import MGroupedGEMMParams, m_grouped_gemm

gpu = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def random_rows(g, rows, k, dtype=torch.bfloat16):
    data = (torch.randn(rows, k, generator=g, device="cuda") * 100).clamp(-448, 448).to(DTYPE)
    return Fp8Rows(data, 0.01 * (0.5 + torch.rand(rows, -(-k // BLOCK), generator=g, device="cuda")), dtype)


def random_weight(g, *shape):
    n, k = shape[-2:]
    data = (torch.randn(*shape, generator=g, device="cuda") * 100).clamp(-448, 448).to(DTYPE)
    scales = 0.5 + torch.rand(*shape[:-2], -(-n // BLOCK), -(-k // BLOCK), generator=g, device="cuda")
    return Fp8Weight(data, scales * k ** -0.5 / 100)


def rows64(rows):
    return rows.data.double() * rows.scales.double().repeat_interleave(BLOCK, -1)[:, :rows.data.size(1)]


def weight64(w):
    n, k = w.data.shape[-2:]
    return w.data.double() * w.scales.double().repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def sum_error(k):
    """Of a product of depth k in fp32, relative to the sum of the terms' magnitudes: 128 additions per block inside the tensor core,
    at a unit (2^-23) of the running sum each, then one scaled addition per block (two roundings of 2^-24 for the factor, one for
    the sum)."""
    return 128 * 2.0 ** -23 + (2 + k / BLOCK) * 2.0 ** -24


def check_product(out, x, w, dtype):
    want, terms = x @ w.mT, x.abs() @ w.abs().mT
    f = torch.finfo(dtype)
    assert out.dtype is dtype and out.shape == want.shape
    assert bool(((out.double() - want).abs() <= f.eps / 2 * want.abs() + (1 + f.eps) * sum_error(x.size(1)) * terms + f.tiny * f.eps / 2).all())


# ------------------------------------------------------------------------------------------------------------ rows
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 4096), (7, 144), (300, 1040), (1000, 7168), (5, 128)])
def test_rows_to_8_bits(rows, k, dtype, native):
    """The bits of the definition: x * 448 / (largest magnitude of the block) is a quotient of short numbers, rounded once to fp32 and
    once to e4m3 (which the fp32 rounding cannot carry over the middle between two values)."""
    x = torch.randn(rows, k, generator=gen(k), device="cuda").mul_(3).to(dtype)
    x[0, : min(k, 128)] = 0
    if rows > 2:
        x[2] = x[2].round()                      # many exact halves
        x[1, 0] = 65504.0 if dtype is torch.float16 else 3e38
    got = quantize_rows(x)
    pad = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    most = pad.abs().amax(-1, keepdim=True).clamp_min(LEAST)
    want = (pad * 0.875 / most * 512).to(DTYPE).flatten(1)[:, :k]
    assert got.dtype is dtype and torch.equal(got.data.view(torch.uint8), want.contiguous().view(torch.uint8))
    assert bool(((got.scales - most[..., 0] / 448).abs() <= 2.0 ** -23 * got.scales).all())


@gpu
def test_rows_that_are_not_finite_strided_and_empty(native):
    x = torch.randn(6, 300, device="cuda").bfloat16()
    with pytest.raises(native.MoeNativeError, match="multiple of 16"):
        quantize_rows(x)
    y = x[:, 2:290]                              # strided, not aligned
    a, b = quantize_rows(y), quantize_rows(y.contiguous())
    assert torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8)) and torch.equal(a.scales, b.scales)
    z = y.contiguous()
    z[1, 5] = math.nan
    z[2, 200] = -math.inf
    c = quantize_rows(z)
    back = rows64(c)
    assert torch.isnan(back[1, 5]) and torch.isfinite(back[1, 6:]).all() and torch.isnan(back[2, 200]) and torch.isfinite(back[2, :128]).all()
    assert torch.equal(back[3:], rows64(b)[3:])
    assert quantize_rows(z[:0]).data.shape == (0, 288)


def test_weights_to_8_bits(native):
    w = torch.randn(3, 200, 300, generator=gen(0, "cpu"))
    w[1, 128:] = 0
    q = quantize_weight(w)
    assert q.scales.shape == (3, 2, 3) and bool((q.scales > 0).all())
    scale = q.scales.double().repeat_interleave(BLOCK, 1)[:, :200].repeat_interleave(BLOCK, 2)[:, :, :300]
    back = q.data.double() * scale
    assert bool(((back - w).abs() <= 2.0 ** -4 * w.abs() + 2.0 ** -10 * scale + 2.0 ** -22 * w.abs()).all())   # half a step of e4m3
    glu = MLPParams(torch.randn(2, 64, 96), torch.randn(2, 48, 64), "swiglu")
    p = quantize_experts(glu)
    assert p.up.data.shape == (2, 2, 48, 64) and p.down.data.shape == (2, 64, 48)
    gate, up = glu.weight1[..., 0::2].mT, glu.weight1[..., 1::2].mT
    same = quantize_experts(GLUParams(gate.mT, up.mT, glu.weight2, "swiglu"))
    assert torch.equal(p.up.data.view(torch.uint8), same.up.data.view(torch.uint8)) and torch.equal(p.up.scales, same.up.scales)
    assert float((p.up.data[:, 0].float() * p.up.scales[:, 0] - gate).norm() / gate.norm()) < 2.0 ** -4


# -------------------------------------------------------------------------------------------------------- products
SIZES = [(1, 128, 128), (1, 8, 16), (3, 40, 144), (16, 256, 2000), (17, 264, 128), (64, 4096, 1024), (65, 136, 272), (100, 1000, 512),
         (128, 128, 4096), (129, 512, 384), (200, 264, 2000), (256, 256, 128), (257, 1416, 656), (1000, 2040, 2000), (2049, 520, 1024)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_dense_product(m, n, k, dtype, native):
    g = gen(m + n + k)
    rows, w = random_rows(g, m, k, dtype), random_weight(g, n, k)
    out = fp8_matmul(rows, w)
    check_product(out, rows64(rows), weight64(w), dtype)
    assert torch.equal(out, fp8_matmul(rows, Fp8Weight(w.data[None], w.scales[None])))


@gpu
def test_whole_numbers_are_exact(native):
    """Small integers with scale 1: every sum is exact, so is the result."""
    g = gen(1)
    for m, n, k in ((1, 128, 256), (40, 200, 272), (300, 600, 512)):
        x = torch.randint(-4, 5, (m, k), generator=g, device="cuda").float()
        w = torch.randint(-1, 2, (n, k), generator=g, device="cuda").float()
        x[:, 32:] *= torch.rand(m, k - 32, generator=g, device="cuda") < 0.1
        out = fp8_matmul(Fp8Rows(x.to(DTYPE), torch.ones(m, -(-k // 128), device="cuda"), torch.float16),
                         Fp8Weight(w.to(DTYPE), torch.ones(-(-n // 128), -(-k // 128), device="cuda")))
        want = x.double() @ w.double().T
        assert want.abs().max() < 2048 and torch.equal(out.double(), want)


def grouped_case(g, counts, k, n, topk=1):
    E, rows = len(counts), sum(counts)
    groups = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    owner = torch.repeat_interleave(torch.arange(E, device="cuda"), torch.tensor(counts, device="cuda"))
    return groups, owner, random_weight(g, E, n, k), rows


COUNTS = [[5], [0, 1, 0, 130, 0], [64, 64, 1, 200], [300, 0, 700, 129, 128], [3] * 40, [0, 0, 513], [1000, 17, 255]]


@gpu
@pytest.mark.parametrize("counts", COUNTS, ids=str)
def test_grouped_product(counts, native):
    g = gen(len(counts))
    for k, n, dtype, act in ((144, 264, torch.float16, None), (1024, 128, torch.bfloat16, None), (272, 40, torch.bfloat16, "silu")):
        groups, owner, w, rows = grouped_case(g, counts, k, n)
        x = random_rows(g, rows, k, dtype)
        out = m_grouped_gemm(x, MGroupedGEMMParams(w, groups, None, False, False, rows, 1, activation=act))
        for e in range(len(counts)):
            if counts[e]:
                r64, w64 = rows64(x)[owner == e], weight64(Fp8Weight(w.data[e], w.scales[e]))
                if act is None:
                    check_product(out[owner == e], r64, w64, dtype)
                else:
                    z, terms = r64 @ w64.T, r64.abs() @ w64.abs().T
                    want = z * torch.sigmoid(z)    # slope at most 1.1; evaluation in fp32 2^-20
                    assert bool(((out[owner == e].double() - want).abs() <= (half_step(dtype) + 2.0 ** -20) * want.abs()
                                 + 1.2 * sum_error(k) * terms).all())


@gpu
@pytest.mark.parametrize("gather,scatter", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("T,E,topk", [(1, 4, 2), (50, 8, 2), (700, 3, 2)])
def test_gather_and_scatter(T, E, topk, gather, scatter, native):
    g = gen(T)
    k, n = 272, 136
    ids = torch.stack([torch.randperm(E, generator=g, device="cuda")[:topk] for _ in range(T)]).reshape(-1)
    order = torch.sort(ids, stable=True).indices
    groups = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), torch.bincount(ids, minlength=E).cumsum(0))).to(torch.int32)
    w = random_weight(g, E, n, k)
    x = random_rows(g, T if gather else T * topk, k)
    out = m_grouped_gemm(x, MGroupedGEMMParams(w, groups, order, gather, scatter, T, topk))
    plain = random_rows(g, 1, k)  # (rows by hand)
    data = x.data.view(torch.uint8)[order // topk if gather else slice(None)].view(DTYPE)
    plain = Fp8Rows(data, x.scales[order // topk] if gather else x.scales, x.dtype)
    want = m_grouped_gemm(plain, MGroupedGEMMParams(w, groups, None, False, False, T * topk, 1))
    if scatter:
        want = torch.empty_like(want).index_copy_(0, order, want)
    assert torch.equal(out, want)
    if T == 50:   # positions that were dropped: a zero row, not stored
        order[3] = -1
        out2 = m_grouped_gemm(x, MGroupedGEMMParams(w, groups, order, gather, scatter, T, topk))
        torch.cuda.synchronize()
        if gather and not scatter:
            assert out2[3].abs().max() == 0
            assert torch.equal(out2[4:], out[4:]) and torch.equal(out2[:3], out[:3])


@gpu
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("T,E,k", [(25, 4, 272), (500, 4, 256), (1000, 3, 272), (4096, 16, 1024)], ids=["few", "single", "pairs", "prompt"])
def test_scattered_rows_go_nowhere_else(T, E, k, gather, native):
    """Rows behind a scatter: each lies at its place, a dropped position (-1) is stored nowhere, and what lay there is left as it was.
    The sizes reach the kernel of few rows, single CTAs, pairs, and a prompt's gather and scatter."""
    import ctypes

    from moe_explore.functional.fp8 import _maps_layout
    from moe_explore.routing_plan import device_status

    g, n, topk = gen(T), 136, 2
    ids = torch.stack([torch.randperm(E, generator=g, device="cuda")[:topk] for _ in range(min(T, 64))]).repeat(-(-T // 64), 1)[:T].reshape(-1)
    rows = T * topk
    order = torch.sort(ids, stable=True).indices
    groups = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), torch.bincount(ids, minlength=E).cumsum(0))).to(torch.int32)
    w, x = random_weight(g, E, n, k), random_rows(g, T if gather else rows, k)
    data = x.data.view(torch.uint8)[order // topk if gather else slice(None)].view(DTYPE)
    sorted_rows = Fp8Rows(data, x.scales[order // topk] if gather else x.scales, x.dtype)
    want = m_grouped_gemm(sorted_rows, MGroupedGEMMParams(w, groups, None, False, False, rows, 1))
    for e in range(E):
        at = slice(int(groups[e]), int(groups[e + 1]))
        check_product(want[at], rows64(sorted_rows)[at], weight64(Fp8Weight(w.data[e], w.scales[e])), torch.bfloat16)
    drop = torch.tensor([0, 3, rows // 2, rows - 1], device="cuda")
    perm = order.clone()
    perm[drop] = -1
    keep = perm >= 0
    there = torch.full_like(want, 7.0)
    there[order[keep]] = want[keep]
    out = torch.full_like(want, 7.0)
    offsets, words = _maps_layout(rows, E)
    maps = torch.empty(words, dtype=torch.int32, device="cuda")
    gathered, gathered_scales = torch.empty(rows, k, dtype=DTYPE, device="cuda"), torch.empty(rows, -(-k // BLOCK), device="cuda")
    p = native.F8RowsPass(rows, x.data.size(0), E, k, n, topk if gather else 1, 0, 0, gather, True, x.data.data_ptr(), x.scales.data_ptr(),
                          w.data.data_ptr(), w.scales.data_ptr(), out.data_ptr(), groups.data_ptr(), perm.data_ptr(),
                          *[maps.data_ptr() + o for o in offsets], device_status(0).data_ptr(), gathered.data_ptr(), gathered_scales.data_ptr())
    steps = native.ROWS_LAYOUT | native.ROWS_GEMM | (native.ROWS_GATHER if gather else 0)
    assert native.load().moe_f8_rows_gemm(ctypes.byref(p), steps, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, there)
    assert torch.equal(m_grouped_gemm(x, MGroupedGEMMParams(w, groups, perm, gather, True, T, topk))[order[keep]], want[keep])


@gpu
def test_a_prefix_that_is_none_is_reported(native):
    from moe_explore.routing_plan import check_device_status

    g = gen(0)
    x, w = random_rows(g, 100, 128), random_weight(g, 3, 64, 128)
    groups = torch.tensor([0, 60, 40, 100], dtype=torch.int32, device="cuda")
    m_grouped_gemm(x, MGroupedGEMMParams(w, groups, None, False, False, 100, 1))
    with pytest.raises(native.MoeNativeError, match="metadata"):
        check_device_status()
    assert check_device_status() == 0


# --------------------------------------------------------------------------------------------------------- experts
def definition(x, scores, ids, p):
    """The layer in 64 bits, with the bound on what rounding in between may add: an activated value that lies within the error of its
    evaluation of the middle between two 8-bit values may go either way."""
    T, k = ids.shape
    d = p.down.data.size(1)
    out = torch.zeros(T, d, dtype=torch.float64, device="cuda")
    slack = torch.zeros_like(out)
    size = torch.zeros_like(out)
    xr = rows64(x)
    gelu = p.activation in ("geglu", "gelu")
    for e in range(p.down.data.size(0)):
        t, s = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        up = weight64(Fp8Weight(p.up.data[e], p.up.scales[e]))
        pre, terms = xr[t] @ up[0].T, xr[t].abs() @ up[0].abs().T
        err = sum_error(xr.size(1)) * terms
        act = pre * (torch.special.ndtr(pre) if gelu else torch.sigmoid(pre))
        h, e_h = act, 1.2 * err + 2.0 ** -20 * act.abs()
        if up.size(0) == 2:
            lin, e_lin = xr[t] @ up[1].T, sum_error(xr.size(1)) * (xr[t].abs() @ up[1].abs().T)
            h, e_h = act * lin, e_h * lin.abs() + (act.abs() + e_h) * e_lin + 2.0 ** -22 * (act * lin).abs()
        inter = h.size(1)
        pad = lambda v: torch.nn.functional.pad(v, (0, -inter % BLOCK)).unflatten(-1, (-1, BLOCK))
        most = pad(h).abs().amax(-1, keepdim=True).clamp_min(LEAST)
        e_most = (pad(e_h).amax(-1, keepdim=True) / most).clamp_max(1.0) + 2.0 ** -22     # relative error of the block's scale
        v = pad(h) / most * 448
        e_v = pad(e_h) / most * 448 + v.abs() * e_most
        q8 = lambda v: v.clamp(-448, 448).float().to(DTYPE).double()
        q = (q8(v) * most / 448).flatten(-2)[:, :inter]
        either = ((q8(v + e_v) - q8(v - e_v)).abs() * most / 448 + q8(v).abs() * most / 448 * e_most).flatten(-2)[:, :inter]
        w2 = weight64(Fp8Weight(p.down.data[e], p.down.scales[e]))
        y, y_terms = q @ w2.T, q.abs() @ w2.abs().T
        y_slack = either @ w2.abs().T + sum_error(inter) * y_terms
        c = scores[t, s].double()[:, None]
        out.index_add_(0, t, c * y)
        slack.index_add_(0, t, c.abs() * (y_slack + half_step(scores.dtype) * (y.abs() + y_slack)))    # the row before the fold is in 16 bits
        size.index_add_(0, t, c.abs() * y.abs())
    return out, slack, size


def check_experts(got, x, scores, ids, p, addend=None):
    want, slack, size = definition(x, scores, ids, p)
    if addend is not None:
        want = want + addend.double()
        size = size + addend.double().abs()
    f = torch.finfo(got.dtype)
    bound = f.eps / 2 * want.abs() + (1 + f.eps) * (slack + 2.0 ** -20 * size) + f.tiny * f.eps * (1 + ids.size(1))
    assert bool(((got.double() - want).abs() <= bound).all())


def make_experts(g, E, d, inter, act):
    gates = 2 if "glu" in act else 1
    return Fp8ExpertParams(random_weight(g, E, gates, inter, d), random_weight(g, E, d, inter), act)


def routing(g, T, E, k, dtype, favour=0.0):
    logits = torch.randn(T, E, generator=g, device="cuda")
    logits[:, 0] += favour
    top = torch.topk(logits, k, dim=-1)
    return torch.softmax(top.values, -1).to(dtype), top.indices


@gpu
@pytest.mark.parametrize("T,E,k,d,inter", [(1, 4, 2, 256, 512), (300, 4, 2, 272, 208), (1100, 3, 2, 512, 656)])
def test_experts_with_the_tanh_form_of_gelu(T, E, k, d, inter, native, monkeypatch):
    from moe_explore.expert_compute import fp8_expert_compute

    g = gen(T)
    p = make_experts(g, E, d, inter, "approx_gelu")
    x = torch.randn(T, d, generator=g, device="cuda").bfloat16()
    scores, ids = routing(g, T, E, k, torch.bfloat16)
    out = fp8_expert_compute(x, scores, ids, p)
    # the plain form with the tanh form in the distribution function's place; its slope, too, is below 1.2
    monkeypatch.setattr(torch.special, "ndtr", lambda v: 0.5 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (v + 0.044715 * v ** 3))))
    check_experts(out, quantize_rows(x), scores, ids, Fp8ExpertParams(p.up, p.down, "gelu"))
    # and the product by itself
    groups, owner, w, rows = grouped_case(g, [5, 0, 300], 272, 40)
    xr = random_rows(g, rows, 272)
    got = m_grouped_gemm(xr, MGroupedGEMMParams(w, groups, None, False, False, rows, 1, activation="approx_gelu"))
    for e in (0, 2):
        r64, w64 = rows64(xr)[owner == e], weight64(Fp8Weight(w.data[e], w.scales[e]))
        z, terms = r64 @ w64.T, r64.abs() @ w64.abs().T
        want = z * torch.special.ndtr(z)
        # tanh to 2^-22 of 1 (its error bound is 2 units), multiplied by z / 2
        assert bool(((got[owner == e].double() - want).abs() <= (half_step(torch.bfloat16) + 2.0 ** -20) * want.abs() + 2.0 ** -21 * z.abs()
                     + 1.2 * sum_error(272) * terms).all())


# tokens, experts, slots, d, I, pull towards expert 0: one token; a batch; many rows for one of many experts; odd widths; many rows
LAYERS = [(1, 8, 2, 256, 512, 0), (1, 1, 1, 128, 128, 0), (5, 4, 4, 16, 16, 0), (33, 16, 4, 400, 272, 0), (300, 64, 2, 256, 208, 9),
          (130, 2, 1, 528, 144, 0), (200, 2, 2, 256, 256, 0), (700, 4, 2, 272, 400, 3), (1100, 3, 2, 512, 656, 0), (64, 1, 1, 256, 1040, 0)]


@gpu
@pytest.mark.parametrize("act", ["swiglu", "geglu", "silu", "gelu"])
@pytest.mark.parametrize("T,E,k,d,inter,favour", LAYERS)
def test_experts(T, E, k, d, inter, favour, act, native):
    from moe_explore.expert_compute import fp8_expert_compute

    g = gen(T + E + d)
    p = make_experts(g, E, d, inter, act)
    dtype = torch.float16 if act in ("geglu", "silu") else torch.bfloat16
    x = torch.randn(T, d, generator=g, device="cuda").to(dtype)
    scores, ids = routing(g, T, E, k, dtype, favour)
    rows = quantize_rows(x)
    out = fp8_expert_compute(x, scores, ids, p)
    assert out.dtype is dtype
    check_experts(out, rows, scores, ids, p)
    assert torch.equal(out, fp8_expert_compute(rows, scores, ids, p))          # the same rows, already in 8 bits
    assert torch.equal(out, fp8_expert_compute(x, scores, ids, p))             # and the same bits every time
    addend = torch.randn(T, d, generator=g, device="cuda").to(dtype)
    check_experts(fp8_expert_compute(x, scores, ids, p, addend=addend), rows, scores, ids, p, addend)


# few rows and deep products: K split over clusters of 2 to 8 CTAs; fewer experts hit than there could be; one row for each of many
# experts; a wide result (more blocks than SMs); 64 rows of one expert, and 65
DEEP = [(1, 8, 2, 2048, 1024, 0), (1, 4, 1, 8192, 256, 0), (9, 8, 3, 4096, 400, 30), (4, 300, 8, 1040, 128, 0), (2, 3, 3, 256, 7168, 0),
        (21, 64, 3, 2064, 272, 0), (64, 2, 1, 1024, 1536, 30), (65, 2, 1, 1024, 1536, 30), (3, 16, 8, 128, 2560, 0)]


@gpu
@pytest.mark.parametrize("act", ["swiglu", "gelu"])
@pytest.mark.parametrize("T,E,k,d,inter,favour", DEEP)
def test_experts_of_few_rows(T, E, k, d, inter, favour, act, native):
    from moe_explore.expert_compute import fp8_expert_compute

    g = gen(T + E + d)
    p = make_experts(g, E, d, inter, act)
    x = torch.randn(T, d, generator=g, device="cuda").bfloat16()
    scores, ids = routing(g, T, E, k, torch.bfloat16, favour)
    out = fp8_expert_compute(x, scores, ids, p)
    check_experts(out, quantize_rows(x), scores, ids, p)
    ids[:] = ids[:, :1]                                   # one expert for all of a token's slots
    out = fp8_expert_compute(x, scores, ids, p)
    check_experts(out, quantize_rows(x), scores, ids, p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = fp8_expert_compute(x, scores, ids, p)
    for shift in (0, 1, 2):                               # the maps of every replay are its own
        ids.add_(shift).remainder_(E)
        graph.replay()
        assert torch.equal(again, fp8_expert_compute(x, scores, ids, p))


@gpu
@pytest.mark.parametrize("counts", [[1, 0, 3], [0] * 30 + [7], [1] * 40, [64], [30, 34, 0], [10, 55, 0], [200, 90, 110, 80]], ids=str)
@pytest.mark.parametrize("n,k", [(264, 4096), (2048, 1040)])
def test_deep_grouped_product(n, k, counts, native):
    """The product right behind the kernel that makes its maps, eager and replayed with other groups."""
    g = gen(n)
    groups, owner, w, rows = grouped_case(g, counts, k, n)
    x = random_rows(g, rows, k)
    perm = torch.randperm(rows, generator=g, device="cuda")
    plain = MGroupedGEMMParams(w, groups, None, False, False, rows, 1)
    moved = MGroupedGEMMParams(w, groups, perm, True, True, rows, 1)
    graph = torch.cuda.CUDAGraph()
    m_grouped_gemm(x, plain)
    with torch.cuda.graph(graph):
        out, there = m_grouped_gemm(x, plain), m_grouped_gemm(x, moved)
    for turn in range(2):
        if turn == 1:
            counts = counts[::-1]
            groups.copy_(torch.tensor([0] + counts, device="cuda").cumsum(0))
            owner = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), torch.tensor(counts, device="cuda"))
        graph.replay()
        assert torch.equal(out, m_grouped_gemm(x, plain))
        for e in range(len(counts)):
            if counts[e]:
                check_product(out[owner == e], rows64(x)[owner == e], weight64(Fp8Weight(w.data[e], w.scales[e])), torch.bfloat16)
                at = perm[owner == e]
                check_product(there[at], rows64(x)[at], weight64(Fp8Weight(w.data[e], w.scales[e])), torch.bfloat16)


@gpu
def test_ids_out_of_range_add_nothing_and_are_reported(native):
    from moe_explore.expert_compute import fp8_expert_compute
    from moe_explore.routing_plan import check_device_status

    g = gen(3)
    p = make_experts(g, 6, 256, 128, "swiglu")
    x = torch.randn(40, 256, generator=g, device="cuda").bfloat16()
    scores, ids = routing(g, 40, 6, 2, torch.bfloat16)
    ids[3, 0], ids[7, 1], ids[9] = -1, 6, 100
    out = fp8_expert_compute(x, scores, ids, p)
    with pytest.raises(native.MoeNativeError, match="expert id"):
        check_device_status()
    check_experts(out, quantize_rows(x), scores, ids, p)
    assert out[9].abs().max() == 0


@gpu
def test_a_token_of_nan_stays_alone(native):
    from moe_explore.expert_compute import fp8_expert_compute

    for T in (9, 600):
        g = gen(4)
        p = make_experts(g, 2, 256, 256, "swiglu")
        x = torch.randn(T, 256, generator=g, device="cuda").bfloat16()
        scores, ids = routing(g, T, 2, 1, torch.bfloat16)
        clean = fp8_expert_compute(x, scores, ids, p)
        x[4, 100] = math.nan
        x[6] = 0
        out = fp8_expert_compute(x, scores, ids, p)
        keep = [i for i in range(T) if i not in (4, 6)]
        assert torch.isnan(out[4]).all() and torch.equal(out[keep], clean[keep]) and out[6].abs().max() == 0


@gpu
def test_streams_capture_two_at_once_and_empty(native):
    from moe_explore.expert_compute import fp8_expert_compute

    g = gen(5)
    p = make_experts(g, 8, 512, 256, "swiglu")
    xs = [torch.randn(T, 512, generator=g, device="cuda").bfloat16() for T in (3, 900)]
    routes = [routing(g, x.size(0), 8, 2, torch.bfloat16) for x in xs]
    want = [fp8_expert_compute(x, *r, p) for x, r in zip(xs, routes)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for x, r, s in zip(xs, routes, streams):
            with torch.cuda.stream(s):
                got.append(fp8_expert_compute(x, *r, p))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out, want[i % 2])
    graphs, outs = [], []
    for x, r in zip(xs, routes):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fp8_expert_compute(x, *r, p))
        graphs.append(graph)
    old = [x.clone() for x in xs]
    for x in xs:
        x.mul_(-1)
    for graph in graphs:
        graph.replay()
    for x, o in zip(xs, old):
        x.copy_(o)
    torch.cuda.synchronize()
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out, w)
    assert fp8_expert_compute(xs[0][:0], routes[0][0][:0], routes[0][1][:0], p).shape == (0, 512)
    assert fp8_matmul(random_rows(g, 0, 128), random_weight(g, 64, 128)).shape == (0, 64)


# -------------------------------------------------------------------------------------------------------- refusals
def test_refusals(native):
    import ctypes

    lib = native.load()
    p = 4096
    assert lib.moe_f8_quantize_rows(p, p, p, 4, 40, 0, None) == -2 and b"multiple of 16" in lib.moe_last_error()
    assert lib.moe_f8_quantize_rows(p, p, p, -1, 64, 0, None) == -1 and lib.moe_f8_quantize_rows(p, p, p, 4, 64, 2, None) == -1
    assert lib.moe_f8_quantize_rows(p + 8, p, p, 4, 64, 0, None) == -1 and lib.moe_f8_quantize_rows(None, p, p, 4, 64, 0, None) == -1
    assert lib.moe_f8_quantize_rows(None, None, None, 0, 64, 0, None) == 0

    def gemm(rows=4, x_rows=4, E=1, k=64, n=64, act=0, dtype=0, gather=0, scatter=0, x=p, groups=None, perm=None, maps=None):
        s = native.F8RowsPass(rows, x_rows, E, k, n, 1, act, dtype, gather, scatter, x, p, p, p, p, groups, perm, maps, maps, maps, maps)
        return lib.moe_f8_rows_gemm(ctypes.byref(s), native.ROWS_GEMM, None)

    assert gemm(k=40) == -2 and gemm(n=60) == -2 and b"multiple of" in lib.moe_last_error()
    assert gemm(E=2) == -1 and b"one expert" in lib.moe_last_error()
    assert gemm(x_rows=3) == -1 and gemm(rows=0) == -1
    assert gemm(x=p + 8) == -1 and b"aligned" in lib.moe_last_error()
    assert gemm(act=3) == -1 and b"activation" in lib.moe_last_error()
    assert gemm(dtype=2) == -1
    assert gemm(groups=p) == -1 and b"null" in lib.moe_last_error()
    assert gemm(groups=p, maps=p, scatter=1) == -1 and gemm(groups=p, maps=p, gather=1) == -1
    s = native.F8Pass(4, 128, 64, 64, 2, 1, 3, 0)
    assert lib.moe_f8_expert_forward(ctypes.byref(s), 31, None) == -1 and b"bound" in lib.moe_last_error()
    s = native.F8Pass(4, native.padded_rows_bound(4, 2), 72, 64, 2, 1, 3, 0)
    assert lib.moe_f8_expert_forward(ctypes.byref(s), 31, None) == -2 and b"multiples of 16" in lib.moe_last_error()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        quantize_rows(torch.zeros(2, 16, dtype=torch.bfloat16))


@gpu
def test_refusals_of_tensors(native):
    from moe_explore.expert_compute import fp8_expert_compute

    g = gen(6)
    rows, w = random_rows(g, 4, 128), random_weight(g, 64, 128)
    with pytest.raises(ValueError, match="8-bit rows"):
        fp8_matmul(Fp8Rows(rows.data, rows.scales[:2]), w)
    with pytest.raises(TypeError):
        fp8_matmul(Fp8Rows(rows.data, rows.scales, torch.float32), w)
    with pytest.raises(ValueError, match="weight"):
        fp8_matmul(rows, Fp8Weight(w.data, w.scales.double()))
    with pytest.raises(ValueError, match="matrices"):
        fp8_matmul(rows, random_weight(g, 2, 64, 128))
    with pytest.raises(ValueError, match="columns"):
        fp8_matmul(rows, random_weight(g, 64, 256))
    groups = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError, match="both"):
        m_grouped_gemm(torch.zeros(4, 128, device="cuda", dtype=torch.bfloat16),
                       MGroupedGEMMParams(Fp8Weight(w.data[None], w.scales[None]), groups, None, False, False, 4, 1))
    with pytest.raises(ValueError, match="gated"):
        m_grouped_gemm(rows, MGroupedGEMMParams(Fp8Weight(w.data[None], w.scales[None]), groups, None, False, False, 4, 1, activation="swiglu"))
    p = make_experts(g, 2, 128, 64, "swiglu")
    x = torch.randn(4, 128, generator=g, device="cuda").bfloat16()
    scores, ids = routing(g, 4, 2, 1, torch.bfloat16)
    with pytest.raises(RuntimeError, match="no backward"):
        fp8_expert_compute(x.requires_grad_(True), scores, ids, p)
    x = x.detach()
    with pytest.raises(ValueError, match="activation"):
        fp8_expert_compute(x, scores, ids, Fp8ExpertParams(p.up, p.down, "gelu"))
    with pytest.raises(ValueError, match="shapes"):
        fp8_expert_compute(x[:, :64], scores, ids, p)
    with pytest.raises(ValueError, match="indices"):
        fp8_expert_compute(x, scores, ids.int(), p)
    with pytest.raises(ValueError, match="addend"):
        fp8_expert_compute(x, scores, ids, p, addend=x[:2])
    with pytest.raises(TypeError):
        fp8_expert_compute(x.float(), scores, ids, p)


def test_a_pass_without_its_row_map_is_refused(native):
    """Without dst_row the dispatch would leave the rows unsorted and the fold would take them so."""
    import ctypes

    lib = native.load()
    for step in (native.F8_ROUTE, native.F8_DISPATCH, native.F8_FOLD):
        s = native.F8Pass(0, native.padded_rows_bound(4, 2), 64, 64, 2, 1, 3, 0)
        s.num_tokens = 0
        s.xs = s.xs_scales = s.x = s.ys = s.out = s.scores = 4096
        assert lib.moe_f8_expert_forward(ctypes.byref(s), step, None) == -1 and b"bad sizes" in lib.moe_last_error()
        s.num_tokens = 4
        assert lib.moe_f8_expert_forward(ctypes.byref(s), step, None) == -1 and b"null" in lib.moe_last_error()


@gpu
def test_no_gradient_is_lost_in_silence(native):
    """Rows, weights or scales that ask for a gradient are refused, by every product; without gradients they are taken."""
    from moe_explore.expert_compute import fp8_expert_compute

    g = gen(8)
    rows, w = random_rows(g, 4, 128), random_weight(g, 1, 64, 128)
    groups = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    p = make_experts(g, 2, 128, 64, "swiglu")
    scores, ids = routing(g, 4, 2, 1, torch.bfloat16)
    products = (lambda: fp8_matmul(rows, w),
                lambda: m_grouped_gemm(rows, MGroupedGEMMParams(w, groups, None, False, False, 4, 1)))
    experts = (lambda: fp8_expert_compute(rows, scores, ids, p),)
    for held, calls in ((rows.scales, products + experts), (w.scales, products), (rows.data, products + experts), (w.data, products),
                        (p.up.scales, experts), (p.down.scales, experts), (p.up.data, experts), (p.down.data, experts), (scores, experts)):
        for call in calls:
            want = call()
            held.requires_grad_(True)
            with pytest.raises(RuntimeError, match="no backward"):
                call()
            with torch.no_grad():
                assert torch.equal(call(), want)
            held.requires_grad_(False)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(rows.scales, torch.ones_like(rows.scales))
        with pytest.raises(RuntimeError, match="no backward"):
            fp8_matmul(Fp8Rows(rows.data, dual), w)


def test_chained_kernels_promise_no_constant_memory():
    """The kernels that wait for the one before through await_predecessor(): see tests/test_chained_kernels.py."""
    found = 0
    for path in glob.glob(os.path.join(ROOT, "moe-explore_b200", "csrc", "f8*.cu*")):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        found += len(re.findall(r"\bawait_predecessor\(\);", text))
        assert "__restrict__" not in text and "__ldg" not in text
    assert found >= 4
