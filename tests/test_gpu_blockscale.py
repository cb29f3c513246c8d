"""Block-scaled FP8 casts and products on the GPU against plain 64-bit forms."""
import numpy as np
import pytest
import torch

import blockscale_plain as P

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import apa
    from apa import APABlockTensor, block_cast, block_linear, block_matmul

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def rnd(shape, seed, dtype=torch.float32, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[0], 1, generator=g))
    return x.to(dtype)


def f64(t):
    return t.detach().cpu().double().numpy()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_equal_nan(got, want):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert np.array_equal(got[ok], want[ok])


def check_cast(q, want, e):
    """Codes, scales and dequantised values are those of the definition, bit for bit.
    Every value code * 2^p is an fp32 number (a multiple of 2^-9 2^-126, four
    significant bits) but for one: magnitudes above 248 * 2^120 round to the
    code 256 under the scale 2^120, and 2^128 is fp32's infinity."""
    assert np.array_equal(q.exponents().cpu().numpy(), e)
    with np.errstate(over="ignore"):
        want = np.asarray(want).astype(np.float32).astype(np.float64)
    assert_equal_nan(f64(q.dequantize(torch.float32)), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 7), (128, 128), (129, 130), (200, 520), (64, 1000), (513, 33)])
def test_cast_forms(shape, dtype):
    x = rnd(shape, 1, dtype)
    xd = x.cuda()
    q, qt = block_cast(xd, "both")
    want, _ = P.cast(f64(x))
    check_cast(q, want, P.exponents(f64(x)))
    xt = np.ascontiguousarray(f64(x).T)
    want, _ = P.cast(xt)
    check_cast(qt, want, P.exponents(xt))
    for form, ref in (("rows", q), ("cols", qt)):
        one = block_cast(xd, form)
        assert torch.equal(one.data.view(torch.uint8), ref.data.view(torch.uint8))
    s, st = block_cast(xd, "both", square=True)
    e = P.exponents(f64(x), 128)
    want, _ = P.cast(f64(x), 128)
    rows = np.repeat(e, 128, 0)[:shape[0]]
    check_cast(s, want, rows)
    check_cast(st, want.T, np.repeat(e.T, 128, 0)[:shape[1]])


def test_cast_special_values():
    x = torch.zeros(6, 260)
    x[0, 3] = float("inf")
    x[0, 4] = 7.0
    x[1, 130] = float("nan")
    x[1, 131] = -1e-30
    x[2, :] = 448.0
    x[3, :] = 448.0 * (1 + 2.0 ** -23)
    x[4, 0] = 3.4e38
    x[4, 200] = 1e-45
    x[5, 5] = -0.0
    q, qt = block_cast(x.cuda(), "both")
    want, _ = P.cast(f64(x))
    check_cast(q, want, P.exponents(f64(x)))
    want, _ = P.cast(f64(x).T)
    check_cast(qt, want, P.exponents(f64(x).T))


def test_cast_every_border():
    """Values on and next to every rounding border of E4M3, and amax next to the scale's border."""
    grid = np.unique(P.round_e4m3(np.linspace(0, 448, 100001)))
    mids = (grid[1:] + grid[:-1]) / 2
    v = np.concatenate([grid, mids, np.nextafter(mids.astype(np.float32), np.float32(0)),
                        np.nextafter(mids.astype(np.float32), np.float32(1e9))]).astype(np.float32)
    v = np.concatenate([v, -v])
    rows = [np.concatenate([[448.0], v[i:i + 127], np.zeros(max(0, 127 - len(v[i:i + 127])))])
            for i in range(0, len(v), 127)]
    x = np.stack(rows).astype(np.float32)
    x = np.concatenate([x * np.float32(2.0 ** k) for k in (-20, 0, 13)])
    q = block_cast(torch.from_numpy(x).cuda())
    want, _ = P.cast(x)
    check_cast(q, want, P.exponents(x))


def test_cast_strided_and_flattened():
    big = rnd((70, 400), 3, torch.bfloat16).cuda()
    for view in (big[:, 3:201], big[::2, :300], big.t()[:130, :64], big[5:6]):
        q = block_cast(view)
        want, _ = P.cast(f64(view))
        check_cast(q, want, P.exponents(f64(view)))
    x = rnd((24, 160), 4).cuda().view(2, 3, 4, 160)
    assert tuple(block_cast(x).shape) == (24, 160)
    assert tuple(block_cast(torch.empty(0, 8, device="cuda")).shape) == (0, 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantize_types(dtype):
    x = rnd((37, 300), 5, spread=0.5)
    want, _ = P.cast(f64(x))
    got = f64(block_cast(x.cuda()).dequantize(dtype))
    # exact but for what the type cannot hold (float16's range and subnormals)
    lim = np.finfo(np.float16).tiny * 2.0 ** -10 if dtype == torch.float16 else 0.0
    assert np.all(np.abs(got - want) <= half_step(dtype) * (0 if dtype != torch.float16 else 1) * np.abs(want) + lim)


def matmul_bound(a, b, steps_k, out, dtype):
    """|error| allowed: every step adds 32 exact products to an fp32 accumulator
    (each step off by at most an ulp, 2^-23, of the running magnitude, and the
    aligned sum of its products by 2^-21 of theirs), then one rounding."""
    mag = np.abs(a) @ np.abs(b).T
    steps = -(-steps_k // 32) + 8
    return (4 + steps) * 2.0 ** -23 * mag + half_step(dtype) * np.abs(out) * (1 + 2.0 ** -10) + 1e-37


def check_matmul(x, w, square, out_dtype, bias=None):
    a = block_cast(x.cuda())
    b = block_cast(w.cuda(), square=square)
    av, bv = f64(a.dequantize()), f64(b.dequantize())
    y = block_matmul(a, b, None if bias is None else bias.cuda(), out_dtype=out_dtype)
    want = av @ bv.T + (0.0 if bias is None else f64(bias))
    tol = matmul_bound(av, bv, x.shape[1], np.abs(want) + (0.0 if bias is None else np.abs(f64(bias))), out_dtype)
    if bias is not None:
        tol = tol + 2.0 ** -23 * np.abs(want)
    err = np.abs(f64(y) - want)
    assert y.dtype == out_dtype and np.all(err <= tol), (err / tol).max()


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 128, 128), (2, 200, 130), (16, 4096, 512), (17, 96, 1000), (33, 512, 4096), (64, 130, 384),
    (65, 65, 65), (128, 128, 2048), (129, 127, 640), (200, 16, 520), (300, 31, 1500), (256, 256, 256),
    (384, 1536, 1111), (1000, 777, 1000), (777, 300, 16)])
@pytest.mark.parametrize("square", [False, True])
def test_matmul(m, n, k, square):
    check_matmul(rnd((m, k), m + k), rnd((n, k), n + 7), square, torch.float32)


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("bias_dtype", DTYPES)
@pytest.mark.parametrize("m,n", [(5, 264), (150, 72), (70, 33)])
def test_matmul_types_and_bias(m, n, out_dtype, bias_dtype):
    check_matmul(rnd((m, 300), 1, spread=0.3), rnd((n, 300), 2, spread=0.3), True, out_dtype,
                 rnd((n, 1), 3, spread=0.0)[:, 0].to(bias_dtype))


@pytest.mark.parametrize("m,n,k", [(3, 160, 700), (260, 130, 300), (130, 257, 4096)])
def test_matmul_exact_operands(m, n, k):
    """Small whole numbers with power-of-two row and block scales: every partial sum is exact, so is the result."""
    g = torch.Generator().manual_seed(m)
    a = torch.randint(-4, 5, (m, k), generator=g).float()
    b = torch.randint(-4, 5, (n, k), generator=g).float()
    ea = torch.randint(-2, 3, (m, (k + 127) // 128), generator=g)
    eb = torch.randint(-2, 3, (n, (k + 127) // 128), generator=g)
    A = APABlockTensor.from_parts(a.to(torch.float8_e4m3fn).cuda(), ea.cuda())
    B = APABlockTensor.from_parts(b.to(torch.float8_e4m3fn).cuda(), eb.cuda())
    assert torch.equal(A.exponents().cpu(), ea.int())
    av = a.numpy().astype(np.float64) * np.exp2(P.spread(ea.numpy(), (m, k)))
    bv = b.numpy().astype(np.float64) * np.exp2(P.spread(eb.numpy(), (n, k)))
    assert np.array_equal(f64(block_matmul(A, B, out_dtype=torch.float32)), av @ bv.T)


def test_matmul_out_and_accumulate():
    m, n, k = 140, 200, 260
    a, b = block_cast(rnd((m, k), 1, spread=0.1).cuda()), block_cast(rnd((n, k), 2, spread=0.1).cuda())
    y = block_matmul(a, b, out_dtype=torch.float32)
    for pitch, off in ((n, 0), (n + 3, 1), (n + 8, 4)):
        buf = torch.full((m + 2, pitch + 8), 7.0, device="cuda")
        out = buf[1:m + 1, off:off + n]
        r = block_matmul(a, b, out=out)
        assert r.data_ptr() == out.data_ptr() and torch.equal(out, y)
        block_matmul(a, b, out=out, accumulate=True)
        assert torch.equal(out, y + y)
        buf[1:m + 1, off:off + n] = 7.0
        assert bool((buf == 7.0).all())          # nothing around it was written
    buf = torch.full((m, n + 5), 7.0, dtype=torch.bfloat16, device="cuda")
    block_matmul(a, b, out=buf[:, :n])
    assert torch.equal(buf[:, :n], y.bfloat16()) and bool((buf[:, n:] == 7.0).all())


def test_matmul_nan_stays_in_its_row():
    x, w = rnd((200, 300), 1, spread=0.1), rnd((150, 300), 2, spread=0.1)
    x[7, 150] = float("inf")
    y = f64(block_matmul(block_cast(x.cuda()), block_cast(w.cuda(), square=True), out_dtype=torch.float32))
    assert np.isnan(y[7]).all() and np.isfinite(np.delete(y, 7, 0)).all()


@pytest.mark.parametrize("lead", [(1,), (5,), (2, 3), (4, 50)])
def test_linear_shapes(lead):
    w, b = rnd((70, 200), 1, spread=0.1), rnd((70, 1), 2, spread=0.0)[:, 0]
    x = rnd((int(np.prod(lead)), 200), 3, torch.bfloat16).cuda().view(*lead, 200)
    wq = block_cast(w.cuda(), square=True)
    y = block_linear(x, wq, b.cuda())
    assert y.shape == (*lead, 70) and y.dtype == torch.bfloat16
    q = block_cast(x)
    assert torch.equal(block_linear(q, wq, b.cuda()), y.view(-1, 70))
    assert torch.equal(block_matmul(q, wq, b.cuda()), y.view(-1, 70))
    assert tuple(block_linear(x[:0], wq).shape) == (0, *lead[1:], 70)


def test_repeatable_and_streams():
    a = block_cast(rnd((300, 2000), 1).cuda())
    b = block_cast(rnd((500, 2000), 2).cuda())
    y = block_matmul(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [block_matmul(a, b) for _ in range(3)]
    again = block_matmul(a, b)
    torch.cuda.synchronize()
    assert torch.equal(again, y) and all(torch.equal(o, y) for o in outs)


def test_graph_capture():
    x = rnd((40, 512), 1, torch.bfloat16).cuda()
    wq = block_cast(rnd((256, 512), 2).cuda(), square=True)
    ref = block_linear(x, wq)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = block_linear(x, wq)
    for seed in (1, 5):
        x.copy_(rnd((40, 512), seed, torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, block_linear(x, wq))
    assert not torch.equal(ref, y)


# plans of apa_block_gemm: CTA pairs (epilogue warps, units per tile), and
# the split tile (columns, CTAs per tile, swapped)
def pair_plan(ew, split=1):
    return split << 7 | ew << 15


def split_plan(bn, split, swap):
    return bn | split << 7 | swap << 14


def exact_operands(m, n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randint(-4, 5, (m, k), generator=g, device="cuda").float()
    b = torch.randint(-4, 5, (n, k), generator=g, device="cuda").float()
    ea = torch.randint(-1, 2, (m, (k + 127) // 128), generator=g, device="cuda")
    eb = torch.randint(-1, 2, (n, (k + 127) // 128), generator=g, device="cuda")
    A = APABlockTensor.from_parts(a.to(torch.float8_e4m3fn), ea)
    B = APABlockTensor.from_parts(b.to(torch.float8_e4m3fn), eb)
    want = A.dequantize().double() @ B.dequantize().double().t()
    return A, B, want


@pytest.mark.parametrize("ew", [4, 8])
@pytest.mark.parametrize("m,n,k", [
    (256, 256, 128), (257, 1, 1), (1, 257, 600), (300, 500, 1000), (1023, 777, 520),
    (2560, 2560, 256),      # 100 tiles: more than one on some CTA pairs
    (5000, 2600, 384),      # 220 tiles: both accumulators of a pair reused
    (4096, 4096, 128)])     # 256 tiles of one slab: the epilogue is the bound
@pytest.mark.parametrize("dtype", DTYPES)
def test_pair_plan_exact(ew, m, n, k, dtype):
    from apa import blockscale
    A, B, want = exact_operands(m, n, k, m + n)
    out = torch.empty(m, n, dtype=dtype, device="cuda")
    blockscale._matmul(A, B, None, out, False, pair_plan(ew))
    assert torch.equal(out, want.to(dtype))
    bias = torch.randint(-9, 9, (n,), device="cuda").float()
    blockscale._matmul(A, B, bias, out, False, pair_plan(ew))
    assert torch.equal(out, (want + bias.double()).to(dtype))


@pytest.mark.parametrize("plan", [pair_plan(4), pair_plan(8), pair_plan(4, 3), pair_plan(8, 9), split_plan(64, 1, 0),
                                  split_plan(64, 4, 0), split_plan(64, 2, 1)])
@pytest.mark.parametrize("pitch,off", [(0, 0), (1, 0), (8, 4), (5, 3)])
def test_plans_write_inside_their_output(plan, pitch, off):
    """Aligned and unaligned rows, overwrite and accumulate: the bytes around stay."""
    from apa import blockscale
    m, n, k = 700, 333, 1100
    A, B, want = exact_operands(m, n, k, 5)
    for dtype in DTYPES:
        buf = torch.full((m + 2, n + pitch + off + 3), 3.0, dtype=dtype, device="cuda")
        out = buf[1:m + 1, off:off + n]
        blockscale._matmul(A, B, None, out, False, plan)
        assert torch.equal(out, want.to(dtype))
        if dtype == torch.float32:
            blockscale._matmul(A, B, None, out, True, plan)
            assert torch.equal(out, (2 * want).float())
        out.fill_(3.0)
        assert bool((buf == 3.0).all())


@pytest.mark.parametrize("bn", [16, 32, 64])
@pytest.mark.parametrize("split", [1, 2, 3, 4, 6, 8])
@pytest.mark.parametrize("swap", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_split_plan_exact(bn, split, swap, dtype):
    """Every tile width, split and orientation, over ragged sizes and uneven splits of the slabs."""
    from apa import blockscale
    small = {16: 13, 32: 29, 64: 139}[bn]
    for big, k in ((200, 1024), (129, 1157)):
        m, n = (small, big) if swap else (big, small)
        A, B, want = exact_operands(m, n, k, bn + split)
        bias = torch.randint(-9, 9, (n,), device="cuda").float()
        out = torch.empty(m, n, dtype=dtype, device="cuda")
        blockscale._matmul(A, B, bias, out, False, split_plan(bn, split, swap))
        assert torch.equal(out, (want + bias.double()).to(dtype))


def test_plans_agree_on_real_data():
    from apa import blockscale
    a = block_cast(rnd((1500, 1300), 1).cuda())
    b = block_cast(rnd((900, 1300), 2).cuda(), square=True)
    av, bv = f64(a.dequantize()), f64(b.dequantize())
    want, tol = av @ bv.T, None
    for plan in (pair_plan(4), pair_plan(8), pair_plan(8, 5), split_plan(64, 1, 0), split_plan(64, 8, 1)):
        out = torch.empty(1500, 900, device="cuda")
        blockscale._matmul(a, b, None, out, False, plan)
        tol = matmul_bound(av, bv, 1300, want, torch.float32) if tol is None else tol
        assert np.all(np.abs(f64(out) - want) <= tol)


@pytest.mark.parametrize("plan", [pair_plan(4), pair_plan(8, 4), split_plan(64, 2, 0), split_plan(32, 1, 1)])
def test_codes_past_the_last_column_do_not_count(plan):
    """The bytes between a row's last code and its pitch, and the scales of rows and blocks past the end, hold NaN."""
    from apa import blockscale
    m, n, k = 30, 200, 1157
    A, B, want = exact_operands(m, n, k, 3)
    for t in (A, B):
        pitch = (k + 15) // 16 * 16
        full = t.buffer[:t.rows * pitch].view(t.rows, pitch)
        full[:, k:] = 0x7F
        rp, kb = (t.shape[0] + 127) // 128 * 128, (k + 127) // 128
        v = t.scales.view((kb + 3) // 4, rp // 128, 32, 4, 4)
        live = torch.zeros(rp, (kb + 3) // 4 * 4, dtype=torch.bool, device="cuda")
        live[:t.shape[0], :kb] = True
        v[~live.view(rp // 128, 4, 32, -1, 4).permute(3, 0, 2, 1, 4)] = 0xFF
    out = torch.empty(m, n, device="cuda")
    blockscale._matmul(A, B, None, out, False, plan)
    assert torch.equal(out, want.float())


@pytest.mark.parametrize("ew", [4, 8])
@pytest.mark.parametrize("split", [2, 3, 7, 10])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(300, 270, 1280), (513, 100, 1300), (2600, 1100, 1281)])
def test_pair_split_exact(ew, split, dtype, m, n, k):
    """Units of a tile on several pairs, slices added in order, with bias and accumulation."""
    from apa import blockscale
    A, B, want = exact_operands(m, n, k, m)
    bias = torch.randint(-9, 9, (n,), device="cuda").float()
    out = torch.empty(m, n, dtype=dtype, device="cuda")
    blockscale._matmul(A, B, bias, out, False, pair_plan(ew, split))
    assert torch.equal(out, (want + bias.double()).to(dtype))
    if dtype == torch.float32:
        blockscale._matmul(A, B, bias, out, True, pair_plan(ew, split))
        assert torch.equal(out, (2 * (want + bias.double())).float())


@pytest.mark.parametrize("plan", [0, pair_plan(4), pair_plan(8), pair_plan(8, 2)])
@pytest.mark.parametrize("n", [300, 301])
def test_long_reductions(plan, n):
    """More than 64 slabs: an fp32 output is summed in rounded chunks (aligned rows by TMA reductions, others by
    plain additions), each chunk's chain at most 8192 columns long; 16-bit outputs in one chain."""
    from apa import blockscale
    m, k = 270, 20000
    A, B, want = exact_operands(m, n, k, 4)
    for dtype in DTYPES:
        out = torch.full((m, n), 5.0, dtype=dtype, device="cuda")
        blockscale._matmul(A, B, None, out, False, plan)
        assert torch.equal(out, want.to(dtype))
    blockscale._matmul(A, B, None, out, True, plan)
    assert torch.equal(out, (2 * want).float())
    a, b = block_cast(rnd((m, k), 1, spread=0).cuda()), block_cast(rnd((n, k), 2, spread=0).cuda())
    out = torch.empty(m, n, device="cuda")
    blockscale._matmul(a, b, None, out, False, plan)
    want = a.dequantize().double() @ b.dequantize().double().t()
    assert float((out - want).norm() / want.norm()) < 1e-6


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 15, 16, 17])
@pytest.mark.parametrize("n,k", [(64, 100), (300, 128), (513, 1157), (4096, 1024), (260, 4096)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_tokens(m, n, k, dtype):
    """Up to 16 tokens are cast inside the product: the same bits as cast and product apart."""
    x, w, b = rnd((m, k), m + k, dtype).cuda(), rnd((n, k), 2).cuda(), rnd((n, 1), 3)[:, 0].cuda()
    wq = block_cast(w, square=True)
    y = block_linear(x, wq, b, out_dtype=torch.float32)
    assert torch.equal(y, block_matmul(block_cast(x), wq, b, out_dtype=torch.float32))
    wide = torch.full((m, k + 9), 3.0, dtype=dtype, device="cuda")
    wide[:, 5:5 + k] = x
    assert torch.equal(block_linear(wide[:, 5:5 + k], wq, b, out_dtype=torch.float32), y)
    x[0, k // 2] = float("inf")
    z = block_linear(x, wq, b, out_dtype=torch.float32)
    assert bool(torch.isnan(z[0]).all()) and torch.equal(z[1:], y[1:])


@pytest.mark.parametrize("plan", [pair_plan(4), pair_plan(8, 2), split_plan(64, 1, 0), split_plan(16, 2, 1)])
def test_extreme_scales(plan):
    """Scales from 2^-127 to 2^127: the exponents of the two sides add."""
    from apa import blockscale
    m, n, k = 16, 200, 512
    g = torch.Generator().manual_seed(1)
    a = torch.randint(1, 5, (m, k), generator=g).float()
    b = torch.randint(1, 5, (n, k), generator=g).float()
    for ea in (-127, -126, -1, 0, 126, 127):
        A = APABlockTensor.from_parts(a.to(torch.float8_e4m3fn).cuda(), torch.full((m, 4), ea).cuda())
        B = APABlockTensor.from_parts(b.to(torch.float8_e4m3fn).cuda(), torch.full((n, 4), -ea).cuda())
        out = torch.empty(m, n, device="cuda")
        blockscale._matmul(A, B, None, out, False, plan)
        assert torch.equal(out.cpu(), a @ b.t()), ea


def test_column_sums_of_infinite_gradients():
    """A bias gradient sums the gradient as it comes: an infinity stays one."""
    from apa import blockscale
    x = torch.ones(300, 40)
    x[5, 3] = float("inf")
    x[200, 4] = float("nan")
    sums = torch.empty(3, 40, device="cuda")
    blockscale._cast(x.cuda(), True, True, colsum=sums)
    got = sums.sum(0).cpu()
    assert got[3] == float("inf") and torch.isnan(got[4]) and bool((got[5:] == 300).all())


def whole_rows(m, k, seed, top):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-top, top + 1, (m, k), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)


def test_offsets_past_32_bits():
    """More than 2^31 elements in the source, the codes, the transposed codes
    and the output: whole numbers, so every row is exact."""
    from apa import blockscale
    m, k, n = 525_000, 4096, 4104
    x = whole_rows(m, k, 1, 7)
    assert x.numel() > 2 ** 31
    q, t = blockscale._cast(x, True, True)
    back = q.dequantize(torch.bfloat16)
    assert torch.equal(back, x)
    del back
    back = t.dequantize(torch.bfloat16)
    for c in (0, 2049, 4095):
        assert torch.equal(back[c], x[:, c])
    del back
    w = whole_rows(72, k, 2, 3)
    y = block_matmul(q, block_cast(w, square=True), out_dtype=torch.float32)
    for lo in (0, 262_100, m - 300):
        assert torch.equal(y[lo:lo + 300].double(), x[lo:lo + 300].double() @ w.double().T)
    del q, t, y, x
    a, b = whole_rows(m, 128, 3, 7), whole_rows(n, 128, 4, 3)
    out = block_matmul(block_cast(a), block_cast(b, square=True), out_dtype=torch.bfloat16)
    assert out.numel() > 2 ** 31
    for lo in (0, 262_100, m - 300):
        want = (a[lo:lo + 300].double() @ b.double().T).to(torch.bfloat16)
        assert torch.equal(out[lo:lo + 300], want)


def test_linear_refuses_inputs_that_want_gradients():
    x = torch.randn(3, 64, device="cuda", requires_grad=True)
    w = block_cast(torch.randn(40, 64, device="cuda"), square=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        block_linear(x, w)
    with torch.no_grad():
        y = block_linear(x, w)
    assert torch.equal(block_linear(x.detach(), w), y)
