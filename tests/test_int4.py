"""Weights in 4 bits and their products with a few rows against the formulas in 64 bits; layout; refusals."""
import math

import pytest
import torch

from moe_explore.functional.int4 import Int4Weight, int4_matmul, pack_experts_int4, pack_int4, quantize_experts_int4, quantize_int4
from moe_explore.params import GLUParams, MLPParams

gpu = pytest.mark.gpu


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def raw(g, *shape, group=128, zeros=False, dtype=torch.bfloat16, device="cuda"):
    *lead, n, k = shape
    groups = -(-k // group)
    values = torch.randint(0, 256, (*lead, n, k // 2), dtype=torch.uint8, generator=g, device=device)
    scales = (0.5 + torch.rand(*lead, n, groups, generator=g, device=device)).mul_(k ** -0.5 / 5).to(dtype)
    points = torch.randint(0, 16, (*lead, n, groups), dtype=torch.uint8, generator=g, device=device) if zeros else None
    return values, scales, points


def weight64(values, scales, zeros, group):
    k = 2 * values.size(-1)
    w = torch.empty(*values.shape[:-1], k, dtype=torch.float64, device=values.device)
    w[..., 0::2], w[..., 1::2] = values % 16, values // 16
    at = torch.arange(k, device=values.device) // group
    return (w - (8 if zeros is None else zeros.double()[..., at])) * scales.double()[..., at]


def sum_error(k):
    """Of a product of depth k, relative to the sum of the terms' magnitudes: products of a group are exact and added inside the tensor cores
    at up to a unit (2^-23) of the running sum each, 128 at most; then one scaled addition per group of at least 32 (two roundings of
    2^-24) and the joining of 64 warps' sums at most."""
    return 128 * 2.0 ** -23 + (2 * (k / 32 + 1) + 64) * 2.0 ** -24


def check(out, x, w, dtype):
    want, terms = x.double() @ w.T, x.double().abs() @ w.abs().T
    f = torch.finfo(dtype)
    assert out.dtype is dtype and out.shape == want.shape
    assert bool(((out.double() - want).abs() <= f.eps / 2 * want.abs() + (1 + f.eps) * sum_error(x.size(1)) * terms + f.tiny * f.eps / 2).all())


# ---------------------------------------------------------------------------------------------------------- layout
@pytest.mark.parametrize("lead,n,k,group,zeros", [((), 16, 128, 128, False), ((), 24, 200, 32, True), ((3,), 40, 8, 64, True),
                                                  ((2, 2), 136, 1000, 128, False)])
def test_layout_and_back(lead, n, k, group, zeros):
    given = raw(gen(n, "cpu"), *lead, n, k, group=group, zeros=zeros, device="cpu")
    w = pack_int4(*given, group=group)
    back = w.unpack()
    assert torch.equal(back[0], given[0]) and torch.equal(back[1], given[1]) and (torch.equal(back[2], given[2]) if zeros else back[2] is None)
    assert bool((w.dequantize().double() == weight64(*given, group)).all())
    # every value where the description of the layout puts it
    data, values = w.data.reshape(-1, -(-n // 16), -(-k // 128), w.block), given[0].reshape(-1, n, k // 2)
    for m, r, c in torch.randint(0, 1 << 20, (200, 3), generator=gen(1, "cpu")).tolist():
        m, r, c = m % data.size(0), r % n, c % k
        i, t, low = c % 128 // 32, c % 32 // 8, c % 8
        b = (low % 2) * 2 + low // 4
        byte = int(data[m, r // 16, c // 128, (r % 16 // 8 * 32 + 4 * (r % 8) + t) * 16 + 4 * i + b])
        assert (byte >> (4 * (low % 4 // 2))) & 15 == (int(values[m, r, c // 2]) >> (4 * (c % 2))) & 15


def test_quantized_weights_are_near():
    """Half a step of the group's scale (to nearest), its rounding to 16 bits counted, plus, at the ends of the range, what the rounded scale
    leaves uncovered."""
    w = torch.randn(3, 40, 200, generator=gen(0, "cpu"))
    w[0, 3], w[1, 2, :32] = 0, 5.0
    for zeros in (False, True):
        for group in (32, 64, 128):
            q = quantize_int4(w, group, zeros)
            _, scales, points = q.unpack()
            assert q.dtype is torch.bfloat16 and scales.dtype is torch.bfloat16 and bool((scales > 0).all())
            step = scales.float().repeat_interleave(group, -1)[..., :200]
            assert bool(((q.dequantize() - w).abs() <= step * (0.5 + 15 * 2.0 ** -8 + (0.5 if zeros else 0))).all())
    glu = MLPParams(torch.randn(2, 64, 96), torch.randn(2, 48, 64), "swiglu")
    p = quantize_experts_int4(glu, 32)
    same = quantize_experts_int4(GLUParams(glu.weight1[..., 0::2], glu.weight1[..., 1::2], glu.weight2, "swiglu"), 32)
    assert torch.equal(p.up.data, same.up.data) and torch.equal(p.down.data, same.down.data)
    rows = p.up.dequantize().view(2, 6, 2, 8, 64)
    for h in range(2):
        part = glu.weight1[..., h::2].mT.reshape(2, 6, 8, 64)
        assert float((rows[:, :, h] - part).norm() / part.norm()) < 0.15


# -------------------------------------------------------------------------------------------------------- products
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("rows,k,n", [(1, 8, 8), (1, 4096, 4096), (2, 136, 24), (7, 2000, 1416), (8, 7168, 40), (9, 128, 272), (13, 776, 4096),
                                      (16, 1024, 1000), (17, 264, 64), (33, 2048, 520), (64, 392, 2048), (100, 640, 72)])
def test_product(rows, k, n, group, zeros, dtype, native):
    g = gen(rows + k + n)
    given = raw(g, n, k, group=group, zeros=zeros, dtype=dtype)
    x = torch.randn(rows, k, generator=g, device="cuda").to(dtype)
    out = int4_matmul(x, pack_int4(*given, group=group))
    check(out, x, weight64(*given, group), dtype)
    assert torch.equal(out, int4_matmul(x, pack_int4(*given, group=group)))


@gpu
def test_rows_do_not_depend_on_their_neighbours(native):
    """The rows of a call are, bit for bit, those of calls with more or fewer rows that one kernel takes at once: 1 to 8, 9 to 16."""
    given = raw(gen(5), 4096, 512)
    w = pack_int4(*given)
    x = torch.randn(16, 512, device="cuda").bfloat16()
    whole, eight = int4_matmul(x, w), int4_matmul(x[:8], w)
    for r in range(1, 16):
        assert torch.equal(int4_matmul(x[:r], w), whole[:r] if r > 8 else eight[:r])
    x[3] = math.nan
    x[4, 7] = math.inf
    other = int4_matmul(x, w)
    keep = [i for i in range(16) if i not in (3, 4)]
    assert torch.equal(other[keep], whole[keep]) and torch.isnan(other[3]).all() and not torch.isfinite(other[4]).any()


@gpu
def test_whole_numbers_are_exact(native):
    g = gen(2)
    for rows, n, k, group in ((1, 64, 1024, 128), (5, 200, 264, 32), (40, 72, 640, 64)):
        values, scales, zeros = raw(g, n, k, group=group, zeros=True, dtype=torch.float16)
        w = pack_int4(values, torch.ones_like(scales), zeros, group=group)
        x = torch.randint(-1, 2, (rows, k), generator=g, device="cuda").half()
        x[:, 32:] *= torch.rand(rows, k - 32, generator=g, device="cuda") < 0.1
        want = x.double() @ weight64(values, torch.ones_like(scales), zeros, group).T
        assert float(want.abs().max()) < 2048 and bool((int4_matmul(x, w).double() == want).all())


@gpu
def test_shapes_strides_streams_and_graphs(native):
    given = raw(gen(9), 264, 256)
    w = pack_int4(*given)
    x = torch.randn(2, 3, 300, device="cuda").bfloat16()
    part = x[:, :, 3:259]
    assert torch.equal(int4_matmul(part, w), int4_matmul(part.reshape(6, 256).contiguous(), w).view(2, 3, 264))
    assert int4_matmul(part[0, 0], w).shape == (264,) and int4_matmul(part[:0], w).shape == (0, 3, 264)
    x = torch.randn(4, 256, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = int4_matmul(x, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = int4_matmul(x, w)
    assert torch.equal(other, int4_matmul(x, w))
    x.copy_(torch.randn(4, 256, device="cuda"))
    graph.replay()
    assert torch.equal(out, int4_matmul(x, w))


@gpu
def test_offsets_past_32_bits(native):
    """A matrix of more than 2^32 values (2 GB and more of data): its last rows are what they are by themselves."""
    n, k = 270336, 16384
    x = torch.randn(1, k, device="cuda").bfloat16()
    data = torch.zeros(n // 16, k // 128, 1024 + 32, dtype=torch.uint8, device="cuda")
    tail = raw(gen(3), 48, k)
    data[-3:] = pack_int4(*tail).data
    out = int4_matmul(x, Int4Weight(data, n, k, 128, torch.bfloat16, False))
    assert not out[:, :-48].any()
    check(out[:, -48:], x, weight64(*tail, 128), torch.bfloat16)


@gpu
def test_more_rows_than_one_launch_takes(native):
    """2^21 rows are a launch's; every row is its own."""
    weight = raw(gen(5), 16, 8, group=32)
    rows = (1 << 21) + 70
    x = torch.randn(rows, 8, generator=gen(6), device="cuda").bfloat16()
    out = int4_matmul(x, pack_int4(*weight, group=32))
    w = weight64(*weight, 32)
    for part in (slice(0, 100), slice((1 << 21) - 64, rows)):
        check(out[part], x[part], w, torch.bfloat16)


# ------------------------------------------------------------------------------------------------------- refusals
def test_refusals_without_a_gpu(native):
    values, scales, zeros = raw(gen(0, "cpu"), 16, 64, group=32, zeros=True, device="cpu")
    with pytest.raises(ValueError, match="groups"):
        pack_int4(values, scales, zeros, group=16)
    with pytest.raises(ValueError, match="scales"):
        pack_int4(values, scales, zeros, group=64)
    with pytest.raises(ValueError, match="scales"):
        pack_int4(values, scales.float(), zeros, group=32)
    with pytest.raises(ValueError, match="zeros"):
        pack_int4(values, scales, zeros[:8], group=32)
    with pytest.raises(ValueError, match="values"):
        pack_int4(values.int(), scales, group=32)
    with pytest.raises(ValueError, match="multiples of 8"):
        pack_int4(values[:12], scales[:12], group=32)
    with pytest.raises(ValueError, match="multiples of 8"):
        quantize_int4(torch.randn(8, 20))
    with pytest.raises(ValueError, match="up is"):
        pack_experts_int4(raw(gen(0, "cpu"), 2, 1, 16, 64, device="cpu"), raw(gen(0, "cpu"), 2, 64, 16, device="cpu"), "swiglu")
    with pytest.raises(RuntimeError, match="CUDA"):
        int4_matmul(torch.zeros(1, 64).bfloat16(), pack_int4(values, scales, zeros, group=32))
    lib = native.load()
    assert lib.moe_int4_matmul(None, None, None, 1, 64, 64, 128, 0, 0, None) == -1 and b"null" in lib.moe_last_error()
    assert lib.moe_int4_matmul(None, None, None, 1, 64, 64, 48, 0, 0, None) == -1 and b"groups" in lib.moe_last_error()
    assert lib.moe_int4_matmul(None, None, None, 1, 60, 64, 32, 0, 0, None) == -2 and b"multiples of 8" in lib.moe_last_error()
    assert lib.moe_int4_matmul(None, None, None, -1, 64, 64, 32, 0, 0, None) == -1
    assert lib.moe_int4_expand(None, None, 1, 64, 64, 32, 0, 0, 0, None) == -1 and b"null" in lib.moe_last_error()
    assert lib.moe_int4_expand(None, None, 1, 64, 24, 32, 0, 1, 0, None) == -2 and b"gated" in lib.moe_last_error()
    assert lib.moe_int4_expand(None, None, 70000, 64, 64, 32, 0, 0, 0, None) == -1 and lib.moe_int4_expand(8, 16, 1, 64, 64, 32, 0, 0, 0, None) == -1
    assert lib.moe_int4_matmul(16, 40, 64, 1, 64, 64, 32, 0, 0, None) == -1 and b"aligned" in lib.moe_last_error()


@pytest.mark.parametrize("where", [(0, 0), (39, 4)])
def test_zero_points_that_four_bits_do_not_hold_are_refused(where):
    values, scales, points = raw(gen(3, "cpu"), 40, 136, group=32, zeros=True, device="cpu")
    assert torch.equal(pack_int4(values, scales, points, group=32).unpack()[2], points)
    points[where] = 16
    with pytest.raises(ValueError, match="0 to 15"):
        pack_int4(values, scales, points, group=32)
    points[where] = 255
    with pytest.raises(ValueError, match="0 to 15"):
        pack_experts_int4((values[None, None], scales[None, None], points[None, None]), raw(gen(4, "cpu"), 1, 136, 40, group=32, zeros=True, device="cpu"),
                          "silu", group=32)


@gpu
def test_refusals(native):
    w = pack_int4(*raw(gen(0), 16, 64, group=32), group=32)
    x = torch.randn(2, 64, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="rows of"):
        int4_matmul(x[:, :56], w)
    with pytest.raises(TypeError, match="type of the scales"):
        int4_matmul(x.half(), w)
    with pytest.raises(RuntimeError, match="no backward"):
        int4_matmul(x.requires_grad_(True), w)
    x = x.detach()
    with pytest.raises(ValueError, match="axes in front"):
        int4_matmul(x, pack_int4(*raw(gen(0), 2, 16, 64, group=32), group=32))
    with pytest.raises(ValueError, match="Int4Weight"):
        int4_matmul(x, Int4Weight(w.data, 16, 64, 128, w.dtype, False))
    with pytest.raises(ValueError, match="Int4Weight"):
        int4_matmul(x, Int4Weight(w.data, 16, 64, 32, w.dtype, True))
    two = pack_int4(*raw(gen(0), 32, 64, group=32), group=32)
    with pytest.raises(ValueError, match="contiguous"):
        int4_matmul(x, Int4Weight(two.data.repeat(1, 1, 2)[:, :, :two.block], 32, 64, 32, w.dtype, False))
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda t: int4_matmul(t, w), (x,), check_trace=False)
