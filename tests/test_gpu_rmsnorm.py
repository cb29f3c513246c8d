"""The root-mean-square norm on the GPU against its plain 64-bit form.

Tolerances: a row's sum of squares is a chain of at most 32 fused
multiply-adds and ten additions of positive terms, so rstd is off by at most
(42 / 2 + 3) 2^-24 relative; the product adds one rounding. 32 * 2^-24 covers
it. E4M3 outputs are off by half a step of their grid on top."""
import numpy as np
import pytest
import torch

import blockscale_plain as P

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import apa
    from apa import APARMSNorm, blockscale, rms_norm

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24
EPS = 1e-6
SHAPES = [(1, 1), (3, 7), (5, 128), (9, 256), (4, 257), (6, 511), (7, 1000), (130, 384), (3, 1030), (2, 2048),
          (11, 4096), (5, 4100), (3, 8192), (2, 10001), (2, 16384), (1, 20000), (2, 32768)]


def rnd(shape, seed, dtype=torch.float32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[0], 1, generator=g))
    return x.to(dtype)


def gam(k, seed, dtype=torch.float32):
    return (1 + 0.2 * torch.randn(k, generator=torch.Generator().manual_seed(seed))).to(dtype)


def f64(t):
    return t.detach().cpu().double().numpy()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the type's smallest step."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def check_block(q, y):
    """q holds y rounded to E4M3 under its blocks' scales, y itself known to 32 * 2^-24."""
    e = P.exponents(y)
    got = q.exponents().cpu().numpy()
    low, high = P.exponents(y * (1 - 33 * U)), P.exponents(y * (1 + 33 * U))
    assert np.all((got >= low) & (got <= high))
    s = np.exp2(P.spread(got, y.shape).astype(np.float64))
    err = np.abs(f64(q.dequantize()) - y)
    assert np.all(err <= np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * s) * (1 + 2.0 ** -10) + 33 * U * np.abs(y))
    # nearly every code is the exact one: they differ only next to a border
    want, _ = P.cast(y)
    same = (e == got).repeat(128, 1)[:, :y.shape[1]]
    assert np.mean((f64(q.dequantize()) != want) & same) <= 1e-3 + 2.0 / y.size


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dtype):
    x, res, g = rnd(shape, 1, dtype), rnd(shape, 2, dtype), gam(shape[1], 3)
    xd, rd, gd = x.cuda(), res.cuda(), g.cuda()
    y, r = rms_norm(xd, gd, rd, EPS)
    r_want = (x.float() + res.float()).to(dtype)
    assert torch.equal(r.cpu(), r_want)
    want, _ = P.norm(f64(r_want), f64(g), EPS)
    assert np.all(np.abs(f64(y) - want) <= (half_step(dtype) * (1 + 2.0 ** -10) + 32 * U) * np.abs(want) + tiny(dtype))
    q, r2 = rms_norm(xd, gd, rd, EPS, quantize=True)
    assert torch.equal(r2, r)
    check_block(q, want)
    alone = rms_norm(r, gd, eps=EPS)
    assert torch.equal(alone, y)
    q2 = rms_norm(r, gd, eps=EPS, quantize=True)
    assert torch.equal(q2.data.view(torch.uint8), q.data.view(torch.uint8))
    assert torch.equal(q2.exponents(), q.exponents())


@pytest.mark.parametrize("gdtype", DTYPES)
def test_forward_weight_types_views_and_lead_shapes(gdtype):
    big = rnd((30, 700), 4, torch.bfloat16).cuda()
    g = gam(520, 5, gdtype)
    for view in (big[:, 3:523], big[::3, :520]):
        want, _ = P.norm(f64(view), f64(g), EPS)
        y = rms_norm(view, g.cuda(), eps=EPS)
        assert np.all(np.abs(f64(y) - want) <= (2.0 ** -8 * (1 + 2.0 ** -8)) * np.abs(want) + 1e-30)
    x = rnd((24, 520), 6, torch.bfloat16).cuda()
    y, r = rms_norm(x.view(2, 12, 520), g.cuda(), x.view(2, 12, 520))
    assert y.shape == (2, 12, 520) and torch.equal(r.view(24, 520), x + x)
    assert rms_norm(x[:0], g.cuda()).shape == (0, 520)


def test_rows_that_are_zero_huge_or_not_finite():
    x = rnd((6, 300), 7)
    x[0] = 0
    x[1] *= 1e30 / x[1].abs().max()      # its squares pass fp32
    x[2, 5] = float("inf")
    x[3, 6] = float("nan")
    x[4] *= 1e-25 / x[4].abs().max()     # its squares are below fp32
    y = f64(rms_norm(x.cuda(), torch.ones(300, device="cuda"), eps=EPS))
    assert np.all(y[0] == 0)
    assert np.all(y[1] == 0)                              # as the fp32 form: 1 / sqrt(inf)
    assert np.isnan(y[2, 5]) and np.all(y[2, :5] == 0)    # inf * 0, finite * 0
    assert np.isnan(y[3]).all()
    assert np.all(np.abs(y[4] - f64(x)[4] * 1e3) <= 32 * U * np.abs(f64(x)[4]) * 1e3 + 1e-30)
    want, _ = P.norm(f64(x)[5:], np.ones(300), EPS)
    assert np.all(np.abs(y[5:] - want) <= 33 * U * np.abs(want))
    q = rms_norm(x.cuda(), torch.ones(300, device="cuda"), eps=EPS, quantize=True)
    v = f64(q.dequantize())
    assert np.isnan(v[3]).all() and np.all(v[0] == 0) and np.isfinite(v[[0, 1, 4, 5]]).all()


def check_backward(shape, dtype, gdtype, with_res):
    x, dy, g = rnd(shape, 1, dtype), rnd(shape, 2, dtype, 0.3), gam(shape[1], 3, gdtype)
    res, dr = rnd(shape, 4, dtype), rnd(shape, 5, dtype, 0.3)
    xd = x.cuda().requires_grad_(True)
    gd = g.cuda().requires_grad_(True)
    rd = res.cuda().requires_grad_(True)
    if with_res:
        y, r = rms_norm(xd, gd, rd, EPS)
        torch.autograd.backward([y, r], [dy.cuda(), dr.cuda()])
        assert torch.equal(rd.grad, xd.grad)
    else:
        y = rms_norm(xd, gd, eps=EPS)
        y.backward(dy.cuda())
        r = xd
    r64, g64, dy64 = f64(r), f64(g), f64(dy)
    dx, dg = P.norm_backward(r64, g64, EPS, dy64, f64(dr) if with_res else None)
    rstd = 1.0 / np.sqrt((r64 * r64).mean(1, keepdims=True) + EPS)
    hat, gdy = np.abs(r64 * rstd), np.abs(g64 * dy64)
    size = rstd * (gdy + hat * (gdy * hat).mean(1, keepdims=True)) + (np.abs(f64(dr)) if with_res else 0)
    err = np.abs(f64(xd.grad) - dx)
    assert np.all(err <= 100 * U * size + half_step(dtype) * (1 + 2.0 ** -9) * np.abs(dx) + tiny(dtype))
    terms = (np.abs(dy64) * hat).sum(0)
    chain = shape[0] / 100 + 120      # rows per CTA, then the partials; and rstd's own error
    err = np.abs(f64(gd.grad) - dg)
    assert gd.grad.dtype == gdtype
    assert np.all(err <= chain * U * terms + half_step(gdtype) * (1 + 2.0 ** -9) * np.abs(dg) + tiny(gdtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES + [(2000, 384), (1777, 1100), (5000, 16)])
def test_backward(shape, dtype):
    check_backward(shape, dtype, torch.float32, True)


@pytest.mark.parametrize("gdtype", DTYPES)
def test_backward_without_residual(gdtype):
    check_backward((300, 520), torch.bfloat16, gdtype, False)


def test_backward_against_differences():
    """Directional differences of the kernel's forward against its gradient;
    the formula's own differences, in 64 bits, take the same step, so what is
    left is the forward's rounding."""
    M, K, h = 7, 300, 2.0 ** -6
    x, v, dy, g = rnd((M, K), 1), rnd((M, K), 2, spread=0), rnd((M, K), 3, spread=0), gam(K, 4)
    xd = x.cuda().requires_grad_(True)
    gd = g.cuda()
    rms_norm(xd, gd, eps=EPS).backward(dy.cuda())
    up, down = (x + h * v), (x - h * v)
    got = (f64(dy) * (f64(rms_norm(up.cuda(), gd)) - f64(rms_norm(down.cuda(), gd)))).sum(1) / (2 * h)
    a, b = P.norm(f64(up), f64(g), EPS)[0], P.norm(f64(down), f64(g), EPS)[0]
    want = (f64(dy) * (a - b)).sum(1) / (2 * h)
    noise = (np.abs(f64(dy)) * (np.abs(a) + np.abs(b)) * 33 * U).sum(1) / (2 * h)
    assert np.all(np.abs(got - want) <= noise)
    slope = (f64(xd.grad) * f64(v)).sum(1)
    small = 2.0 ** -16
    a, b = P.norm(f64(x) + small * f64(v), f64(g), EPS)[0], P.norm(f64(x) - small * f64(v), f64(g), EPS)[0]
    limit = (f64(dy) * (a - b)).sum(1) / (2 * small)
    scale = (np.abs(f64(xd.grad)) * np.abs(f64(v))).sum(1)
    assert np.all(np.abs(slope - limit) <= 1e-5 * scale + 1e-6)


def test_only_one_output_used():
    x = rnd((20, 256), 1).cuda().requires_grad_(True)
    res = rnd((20, 256), 2).cuda().requires_grad_(True)
    norm = APARMSNorm(256, config=apa.APAConfig(device="cuda"))
    y, r = norm(x, res)
    r.backward(torch.ones_like(r))
    assert torch.equal(x.grad, torch.ones_like(x)) and torch.equal(res.grad, x.grad) and norm.weight.grad is None
    x.grad = res.grad = None
    y, r = norm(x, res)
    y.sum().backward()
    want, _ = P.norm_backward(f64(r), np.ones(256), 1e-6, np.ones((20, 256)))
    assert np.all(np.abs(f64(x.grad) - want) <= 1e-4 * np.abs(want).max())
    norm.weight.requires_grad_(False)
    x.grad = None
    norm(x, res)[0].sum().backward()
    assert norm.weight.grad is not None and x.grad is not None


def test_recomputed_cols_cast():
    """The transposed cast of the norm's output from the stream is the norm's output."""
    for dtype, shape in ((torch.bfloat16, (300, 520)), (torch.float32, (130, 257))):
        r, g = rnd(shape, 1, dtype).cuda(), gam(shape[1], 2).cuda()
        _, _, rstd = blockscale._norm_forward(r, g, None, EPS, True, True)
        _, qt = blockscale._cast(r, False, True, row_mul=rstd, col_mul=g)
        want, _ = P.norm(f64(r), f64(g), EPS)
        check_block(qt, np.ascontiguousarray(want.T))


def test_deterministic_and_captured():
    r, dy, g = rnd((900, 640), 1).cuda(), rnd((900, 640), 2).cuda(), gam(640, 3).cuda()

    def run():
        x = r.clone().requires_grad_(True)
        w = g.clone().requires_grad_(True)
        return (*torch.autograd.grad(rms_norm(x, w), [x, w], dy),)

    a, b = run(), run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        c = run()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


def test_offsets_past_32_bits():
    """Rows behind 2^31 elements equal those of a call on them alone."""
    m, k = 525_000, 4096
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(m, k, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    assert x.numel() > 2 ** 31
    w = torch.rand(k, generator=g, device="cuda")
    lo = m - 512
    tail = x[lo:].clone()
    y, r = rms_norm(x, w, residual=x)
    y1, r1 = rms_norm(tail, w, residual=tail)
    assert torch.equal(y[lo:], y1) and torch.equal(r[lo:], r1)
    del y
    q = rms_norm(r, w, quantize=True)
    assert torch.equal(q.dequantize()[lo:], rms_norm(r1, w, quantize=True).dequantize())
    del q
    rstd = torch.rand(m, generator=g, device="cuda")
    dx, _ = blockscale._norm_backward(x, r, rstd, w, x)
    dx1, _ = blockscale._norm_backward(tail, r1, rstd[lo:].clone(), w, tail)
    assert torch.equal(dx[lo:], dx1)
