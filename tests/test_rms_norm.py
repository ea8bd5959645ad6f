"""Root-mean-square norm: 16-bit and 8-bit results, residual, gradients, against a plain form in 64 bits; refusals."""
import math

import pytest
import torch

from moe_explore.functional.rms_norm import rms_norm, rms_norm_fp8

DTYPES = [torch.bfloat16, torch.float16]
COLS = [8, 16, 120, 248, 256, 776, 1024, 1032, 2048, 4096, 4104, 7168, 8192, 16384]


def plain(x, w, residual=None, eps=1e-6):
    h = x.double()
    if residual is not None:
        h = (x.double() + residual.double()).to(x.dtype).double()
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * w.double(), h


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# fp32: a sum of d squares over at most 16 pieces of a thread and 15 joins, rsqrt, two products: each 2^-24, the sum's share halved
# by the root
EVAL = 80 * 2.0 ** -24


def make(T, d, dtype, wdtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + d)
    x = (3.0 * torch.randn(T, d, generator=g, device="cuda")).to(dtype)
    r = torch.randn(T, d, generator=g, device="cuda").to(dtype)
    w = (1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(wdtype)
    return x, r, w


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", COLS)
@pytest.mark.parametrize("T", [1, 3, 700])
def test_norm_and_sum(T, d, dtype, native):
    for wdtype in (dtype, torch.float32):
        x, r, w = make(T, d, dtype, wdtype)
        y, h = rms_norm(x, w, residual=r)
        want, hs = plain(x, w, r)
        assert torch.equal(h.double(), hs)       # one rounding of an exact sum (16-bit terms of like size)
        assert bool(((y.double() - want).abs() <= (half_step(dtype) + EVAL) * want.abs() + 2.0 ** -25).all())
        y = rms_norm(x, w, eps=1e-5)
        want, _ = plain(x, w, eps=1e-5)
        assert bool(((y.double() - want).abs() <= (half_step(dtype) + EVAL) * want.abs() + 2.0 ** -25).all())


def check_fp8(rows, y, d):
    """`rows` hold y [R, d] (64 bits) to half an e4m3 step, with the scale of each block."""
    k = torch.arange(d, device=y.device) // 128
    most = torch.zeros(y.size(0), int(k[-1]) + 1, dtype=torch.float64, device=y.device).scatter_reduce_(1, k.expand_as(y), y.abs(), "amax")
    scale = most.clamp_min(2.0 ** -80) / 448
    assert rows.data.dtype is torch.float8_e4m3fn and rows.data.shape == y.shape and rows.scales.shape == scale.shape
    assert bool(((rows.scales.double() - scale).abs() <= (EVAL + 2.0 ** -22) * scale).all())
    got = rows.data.double() * rows.scales.double()[:, k]
    # half a step of e4m3: 2^-4 of the value, 2^-10 of a unit below 2^-6
    bound = 2.0 ** -4 * y.abs() + 2.0 ** -10 * scale[:, k] + 2 * (EVAL + 2.0 ** -22) * y.abs()
    assert bool(((got - y).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 112, 128, 144, 1040, 4096, 7168, 16384])
@pytest.mark.parametrize("T", [1, 5, 400])
def test_norm_in_8_bits(T, d, dtype, native):
    x, r, w = make(T, d, dtype, dtype)
    rows, y, h = rms_norm_fp8(x, w, residual=r, with_rows=True)
    want, hs = plain(x, w, r)
    check_fp8(rows, want, d)
    y2, h2 = rms_norm(x, w, residual=r)
    assert torch.equal(y, y2) and torch.equal(h, h2) and rows.dtype is dtype
    only = rms_norm_fp8(x, w)
    check_fp8(only, plain(x, w)[0], d)


@pytest.mark.gpu
def test_empty_blocks_zeros_and_what_is_not_finite(native):
    x = torch.zeros(4, 512, device="cuda", dtype=torch.bfloat16)
    x[1, 130] = 5.0
    x[2, 7] = math.nan
    x[3, 300] = math.inf
    w = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    rows, y = rms_norm_fp8(x, w, with_rows=True)
    assert y[0].abs().max() == 0 and rows.data[0].float().abs().max() == 0 and bool((rows.scales[0] > 0).all())
    back = rows.data.float() * rows.scales.repeat_interleave(128, 1)
    assert torch.allclose(back[1], y[1].float(), rtol=2.0 ** -4)
    assert torch.isnan(y[2]).all() and torch.isnan(back[2]).all()
    assert torch.isnan(y[3, 300]) and torch.isnan(back[3, 300])
    assert torch.isfinite(back[:2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,d", [(1, 64), (5, 1024), (400, 776), (3, 4096), (700, 4104), (2, 16384)])
def test_rows_whose_squares_leave_fp32(T, d, native):
    """Finite bf16 rows up to the type's largest value have a finite norm, forward and backward, beside ordinary rows."""
    g = torch.Generator(device="cuda").manual_seed(d)
    size = 10.0 ** (17 + 21.4 * torch.rand(T, 1, generator=g, device="cuda", dtype=torch.float64))
    if T > 1:
        size[1] = 1.0
    x = ((2 * torch.rand(T, d, generator=g, device="cuda", dtype=torch.float64) - 1) * size).to(torch.bfloat16)
    x[0, 5] = torch.finfo(torch.bfloat16).max
    assert torch.isfinite(x).all()
    w = 1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")
    want, _ = plain(x, w)
    y = rms_norm(x, w)
    # 1 / root mean square is at least 2^-128 and held in fp32: 21 bits where it is the least
    assert bool(((y.double() - want).abs() <= (half_step(torch.bfloat16) + EVAL + 2.0 ** -21) * want.abs() + 2.0 ** -25).all())
    rows, y2 = rms_norm_fp8(x, w, with_rows=True) if d % 16 == 0 else (None, y)
    assert torch.equal(y, y2)
    if rows is not None:
        check_fp8(rows, want, d)
    dy = torch.randn(T, d, generator=g, device="cuda").bfloat16()
    leaves = x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(rms_norm(*leaves), leaves, dy)
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    want_x, want_w = torch.autograd.grad(plain(*wide)[0], wide, dy.double())
    r = torch.rsqrt(wide[0].detach().square().mean(-1, keepdim=True) + 1e-6)
    terms = dy.double().abs() * wide[1].detach().abs()
    bound = half_step(torch.bfloat16) * want_x.abs() + 4 * (EVAL + 2.0 ** -21) * r * (terms + wide[0].detach().abs() * r * terms.mean(-1, keepdim=True) * 4)
    bound = bound + torch.finfo(torch.bfloat16).tiny * torch.finfo(torch.bfloat16).eps
    assert bool(((dx.double() - want_x).abs() <= bound).all())
    total = (dy.double() * wide[0].detach() * r).abs().sum(0)
    assert bool(((dw.double() - want_w).abs() <= 2 * (EVAL + 2.0 ** -21) * total + 1e-30).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,d", [(1, 8), (5, 248), (700, 256), (333, 1032), (1500, 2048), (601, 4104), (64, 7168), (9, 16384)])
def test_gradients(T, d, dtype, native):
    for wdtype, with_residual in ((dtype, True), (torch.float32, False)):
        x, r, w = make(T, d, dtype, wdtype)
        g = torch.Generator(device="cuda").manual_seed(5)
        dy = torch.randn(T, d, generator=g, device="cuda").to(dtype)
        dh = torch.randn(T, d, generator=g, device="cuda").to(dtype)
        leaves = [t.requires_grad_(True) for t in ((x, r, w) if with_residual else (x, w))]
        wide = [t.detach().double().requires_grad_(True) for t in leaves]
        if with_residual:
            got = torch.autograd.grad(rms_norm(x, w, residual=r), leaves, (dy, dh))
            h = (wide[0] + wide[1])
            h = h + (h.detach().to(dtype).double() - h.detach())     # the rounding, passed straight through
            y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * wide[2]
            want = torch.autograd.grad((y, h), wide, (dy.double(), dh.double()))
        else:
            got = torch.autograd.grad(rms_norm(x, w), leaves, dy)
            want = torch.autograd.grad(plain(wide[0], wide[1])[0], wide, dy.double())
        size = dy.double().abs() * w.detach().double().abs()          # terms of dx before they cancel
        for a, b in zip(got[:-1], want[:-1]):
            bound = half_step(dtype) * b.abs() + 4 * EVAL * (size + size.mean(-1, keepdim=True) + dh.double().abs()) + 2.0 ** -25
            assert a.dtype is dtype and bool(((a.double() - b).abs() <= bound).all())
        if with_residual:
            assert torch.equal(got[0], got[1])
        a, b = got[-1].double(), want[-1]
        n = plain(x.detach(), w.detach(), r.detach() if with_residual else None)[0] / w.detach().double()
        total = (dy.double() * n).abs().sum(0)                        # of the summands of dw: each addition rounds to 2^-24 of it
        assert bool(((a - b).abs() <= (half_step(wdtype) * b.abs() if wdtype is not torch.float32 else 0) + 2 * EVAL * total + 1e-30).all())


@pytest.mark.gpu
def test_gradient_against_differences(native):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(2, 64, generator=g, device="cuda").half().requires_grad_(True)
    w = torch.rand(64, generator=g, device="cuda").add_(0.5).requires_grad_(True)
    dy = torch.randn(2, 64, generator=g, device="cuda").half()
    dx, dw = torch.autograd.grad(rms_norm(x, w), (x, w), dy)
    loss = lambda a, b: float((plain(a, b)[0] * dy.double()).sum())
    xd, wd, step = x.detach().double(), w.detach().double(), 1e-6
    for row, col in ((0, 0), (1, 63), (1, 17)):
        e = torch.zeros_like(xd)
        e[row, col] = step
        difference = (loss(xd + e, wd) - loss(xd - e, wd)) / (2 * step)
        assert abs(float(dx[row, col]) - difference) <= half_step(torch.float16) * abs(difference) + 1e-5
    e = torch.zeros_like(wd)
    e[5] = step
    assert abs(float(dw[5]) - (loss(xd, wd + e) - loss(xd, wd - e)) / (2 * step)) < 1e-5


@pytest.mark.gpu
def test_gradient_of_one_result_only(native):
    x, r, w = make(7, 256, torch.bfloat16, torch.bfloat16)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y, h = rms_norm(x, w, residual=r)
    dh = torch.randn_like(h)
    dx, dw = torch.autograd.grad(h, (x, w), dh, allow_unused=True)
    assert torch.equal(dx, dh) and dw is None
    y, h = rms_norm(x, w, residual=r)
    a = torch.autograd.grad(y, (x, w), dh)
    y, h = rms_norm(x, w, residual=r)
    b = torch.autograd.grad((y, h), (x, w), (dh, torch.zeros_like(dh)))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_leading_axes_strides_empty_streams_and_capture(native):
    x, r, w = make(60, 256, torch.bfloat16, torch.bfloat16)
    want, hs = rms_norm(x, w, residual=r)
    y, h = rms_norm(x.view(3, 20, 256), w, residual=r.view(3, 20, 256))
    assert y.shape == (3, 20, 256) and torch.equal(y.view(60, 256), want) and torch.equal(h.view(60, 256), hs)
    wide = torch.zeros(60, 512, device="cuda", dtype=torch.bfloat16)
    wide[:, 256:] = x                                             # rows 1 KB apart, read in place
    assert torch.equal(rms_norm(wide[:, 256:], w, residual=r)[0], want)
    off = torch.zeros(60, 259, device="cuda", dtype=torch.bfloat16)
    off[:, 3:] = x                                                # rows no 16-byte piece begins at
    assert torch.equal(rms_norm(off[:, 3:], w, residual=r)[0], want)
    assert torch.equal(rms_norm(x.t().contiguous().t(), w, residual=r)[0], want)
    one = rms_norm(x[:1].expand(60, 256), w)
    assert torch.equal(one[59], rms_norm(x[:1], w)[0])
    empty = torch.empty(0, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    wl = w.clone().requires_grad_(True)
    y = rms_norm(empty, wl)
    dx, dw = torch.autograd.grad(y, (empty, wl), torch.empty_like(y))
    assert y.shape == (0, 256) and dx.shape == (0, 256) and dw.abs().max() == 0
    assert rms_norm_fp8(empty.detach(), w).data.shape == (0, 256)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = rms_norm(x, w, residual=r)[0]
    side.synchronize()
    assert torch.equal(z, want)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, out = rms_norm_fp8(static, w, with_rows=True)
    static.copy_(r)
    graph.replay()
    again, y2 = rms_norm_fp8(r, w, with_rows=True)
    assert torch.equal(out, y2) and torch.equal(rows.data.view(torch.uint8), again.data.view(torch.uint8)) and torch.equal(rows.scales, again.scales)


def test_one_row_has_no_stride(native, monkeypatch):
    """Torch calls a single row contiguous whatever its stride; the kernels get one that they can read."""
    from moe_explore.functional.rms_norm import _forward, _rows

    class Library:   # takes down the strides that the kernels would get
        def moe_rms_norm(self, x, x_stride, residual, residual_stride, *rest):
            self.got = x, x_stride, residual, residual_stride
            return 0

        def moe_rms_norm_backward(self, dy, dh, h, h_stride, *rest):
            self.got = dy, 0, h, h_stride
            return 0

        moe_rms_norm_partials = staticmethod(lambda rows: rows)

    library = Library()
    monkeypatch.setattr(native, "load", lambda: library)
    monkeypatch.setattr(native, "_stream", lambda: None)
    w = torch.ones(64, dtype=torch.bfloat16)
    for cut in (lambda b: b[:1, :64], lambda b: b[5:6, 3:67], lambda b: b[2:3, 1:2].expand(1, 64), lambda b: b.t()[:1, :64],
                lambda b: b[:1, None, :64], lambda b: b[0, :64]):
        x = cut(torch.arange(80 * 77, dtype=torch.float32).view(80, 77).bfloat16())
        rows = _rows(x)
        assert torch.equal(rows, x.reshape(1, 64)) and rows.stride(1) == 1
        y, h, _ = _forward(x, w, x, 1e-6, False)
        assert y.shape == h.shape == x.shape
        assert all(v % 8 == 0 for v in library.got[1::2]) and all(v % 16 == 0 for v in library.got[::2])
        native.rms_norm_backward(_rows(x).contiguous(), None, rows, w, torch.ones(1))
        assert all(v % 8 == 0 for v in library.got[1::2]) and library.got[2] % 16 == 0
    dense = torch.zeros(3, 64)
    assert _rows(dense) is dense
    wide = torch.zeros(4, 512, dtype=torch.bfloat16)
    assert _rows(wide[:1, 256:]).data_ptr() == wide[:1, 256:].data_ptr()      # read in place


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 256, 4096])
def test_one_row_of_a_wider_matrix(d, native):
    """One token's row, cut out of rows whose length is no multiple of 8, as x and as the residual, forward and backward."""
    x, r, w = make(1, d, torch.bfloat16, torch.bfloat16)
    wide = torch.zeros(2, 60, d + 13, device="cuda", dtype=torch.bfloat16)
    wide[0, :1, :d], wide[1, :1, :d] = x, r
    xs, rs = wide[0, :1, :d], wide[1, :1, :d]
    assert xs.stride(0) == d + 13 and xs.is_contiguous()
    for a, b in zip(rms_norm(xs, w, residual=rs), rms_norm(x, w, residual=r)):
        assert torch.equal(a, b)
    one, two = rms_norm_fp8(xs, w, residual=rs), rms_norm_fp8(x, w, residual=r)
    assert torch.equal(one[0].data.view(torch.uint8), two[0].data.view(torch.uint8)) and torch.equal(one[1], two[1])
    dy = torch.randn(1, 60, d + 13, device="cuda").bfloat16()[0, :1, :d]
    leaf, dense = wide.requires_grad_(True), x.clone().requires_grad_(True)
    got, = torch.autograd.grad(rms_norm(leaf[0, :1, :d], w), leaf, dy)
    want, = torch.autograd.grad(rms_norm(dense, w), dense, dy.contiguous())
    assert torch.equal(got[0, :1, :d], want)
    got[0, :1, :d] = 0
    assert got.abs().max() == 0


def test_refusals(native):
    lib = native.load()
    p = 4096
    call = lambda x=p, w=p, y=p, q=None, s=None, T=4, d=64, dtype=0, wd=0, stride=64: lib.moe_rms_norm(
        x, stride, None, 0, w, wd, None, y, q, s, None, T, d, 1e-6, dtype, None)
    assert call(d=60) == -2 and call(d=16392) == -2 and b"multiple of 8" in lib.moe_last_error()
    assert call(dtype=2) == -1 and call(wd=1) == -1 and b"weight" in lib.moe_last_error()
    assert call(T=-1) == -1 and call(d=0) == -1
    assert call(x=None) == -1 and call(y=None) == -1
    assert call(q=p) == -1 and b"scales" in lib.moe_last_error()
    assert call(x=p + 8) == -1 and call(stride=68) == -1 and b"aligned" in lib.moe_last_error()
    assert call(T=0) == 0
    back = lambda rows=4, d=64, h=p, dw=p: lib.moe_rms_norm_backward(p, None, h, 64, p, 0, p, p, dw, p, rows, d, 0, None)
    assert back(d=20) == -2 and back(h=None) == -1 and back(dw=None) == -1 and back(rows=-3) == -1
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rms_norm(torch.zeros(2, 8), torch.ones(8))


@pytest.mark.gpu
def test_refusals_of_tensors(native):
    x, r, w = make(4, 64, torch.bfloat16, torch.bfloat16)
    with pytest.raises(TypeError):
        rms_norm(x.float(), w.float())
    with pytest.raises(ValueError, match="weight"):
        rms_norm(x, w[:32])
    with pytest.raises(ValueError, match="weight"):
        rms_norm(x, w.half())
    with pytest.raises(ValueError, match="residual"):
        rms_norm(x, w, residual=r[:2])
    with pytest.raises(RuntimeError, match="no backward"):
        rms_norm_fp8(x.requires_grad_(True), w)
    with torch.no_grad():
        rms_norm_fp8(x, w)
    with pytest.raises(ValueError, match="multiple of 16"):
        rms_norm_fp8(x.detach()[:, :40].contiguous()[:, :24], w[:24])
    with pytest.raises(native.MoeNativeError, match="multiple of 8"):
        rms_norm(x.detach()[:, :60].contiguous(), w[:60].contiguous())


@pytest.mark.gpu
def test_forward_mode_is_refused(native):
    """No derivative is lost in silence: a tangent is refused where there is no formula for it, and only there."""
    x, r, w = make(4, 64, torch.bfloat16, torch.bfloat16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(Exception, match="forward"):
            rms_norm(dual, w, residual=r)
        with pytest.raises(RuntimeError, match="no backward"):
            rms_norm_fp8(dual, w)
        assert torch.equal(rms_norm(x, w), rms_norm(x.clone().requires_grad_(True), w))
