"""Block-scaled operators without a GPU: layouts, refusals, and the C entry points' checks."""
import ctypes

import numpy as np
import pytest
import torch

import blockscale_plain as P
from apa import (APABlockLinear, APABlockTensor, APAConfig, APARMSNorm, _lib, block_cast, block_linear, block_matmul,
                 rms_norm)

CPU = APAConfig(device="cpu")


def block(rows, cols, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(rows, cols, generator=g).to(torch.float8_e4m3fn)
    e = torch.randint(-20, 20, (rows, (cols + 127) // 128), generator=g)
    return APABlockTensor.from_parts(q, e), q, e


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 128), (127, 129), (128, 512), (200, 1300), (300, 700)])
def test_scale_layout(rows, cols):
    t, q, e = block(rows, cols)
    assert torch.equal(t.exponents(), e.int())
    assert t.data.stride(0) % 16 == 0 or rows == 1
    rp = (rows + 127) // 128 * 128
    raw = t.scales.numpy()
    assert raw.size == (cols + 511) // 512 * rp * 4
    for r in range(0, rows, 17):
        for kb in range(e.shape[1]):
            at = 4 * ((kb // 4) * rp + r // 128 * 128 + r % 32 * 4 + r % 128 // 32) + kb % 4
            assert int(raw[at]) - 127 == int(e[r, kb])


def test_square_exponents_and_bad_parts():
    q = torch.zeros(200, 300).to(torch.float8_e4m3fn)
    e = torch.tensor([[1, 2, 3], [4, 5, 6]])
    t = APABlockTensor.from_parts(q, e)
    assert torch.equal(t.exponents()[127], torch.tensor([1, 2, 3], dtype=torch.int32))
    assert torch.equal(t.exponents()[128], torch.tensor([4, 5, 6], dtype=torch.int32))
    for bad in (e[:1], e.float(), torch.full((2, 3), 128), torch.full((2, 3), -128)):
        with pytest.raises((ValueError, TypeError)):
            APABlockTensor.from_parts(q, bad)
    with pytest.raises(ValueError):
        APABlockTensor.from_parts(torch.zeros(2, 3), e)
    with pytest.raises(ValueError):
        APABlockTensor.from_parts(q[:0], e[:0])


def test_refusals():
    x = torch.randn(4, 64)
    t, _, _ = block(5, 64)
    for call in (lambda: block_cast(x), lambda: block_matmul(t, t), lambda: block_linear(x, t), lambda: t.dequantize(),
                 lambda: rms_norm(x, torch.ones(64)), lambda: rms_norm(x, torch.ones(64), quantize=True),
                 lambda: APABlockLinear(64, 8, config=CPU)(x), lambda: APARMSNorm(64, config=CPU)(x)):
        with pytest.raises(_lib.APAKernelError, match="CUDA"):
            call()
    for call in (lambda: block_cast(x.int()), lambda: block_cast(x.double()), lambda: block_cast([1.0]),
                 lambda: block_linear(x, x), lambda: block_matmul(x, t), lambda: t.dequantize(torch.int32),
                 lambda: rms_norm(x.double(), torch.ones(64)), lambda: APABlockLinear(64, 8, config=CPU)(t),
                 lambda: APABlockLinear(8, 8, dtype=torch.float64, config=CPU),
                 lambda: APARMSNorm(8, dtype=torch.int8, config=CPU)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: block_cast(x, "columns"), lambda: block_cast(torch.empty(3, 0)),
                 lambda: block_cast(torch.tensor(1.0)), lambda: rms_norm(x, torch.ones(64), eps=-1.0),
                 lambda: rms_norm(x, torch.ones(64), eps=float("nan")),
                 lambda: APABlockLinear(0, 8, config=CPU), lambda: APARMSNorm(0, config=CPU),
                 lambda: APARMSNorm(32769, config=CPU), lambda: APABlockLinear(64, 8, config=CPU)(x[:, :63]),
                 lambda: APABlockLinear(64, 8, config=CPU)(x, residual=x),
                 lambda: APABlockLinear(64, 8, config=CPU)(x, norm=APARMSNorm(32, config=CPU))):
        with pytest.raises(ValueError):
            call()


def test_plain_forms_used_by_the_tests():
    """The tests' plain norm gradient against differences in 64 bits."""
    rng = np.random.default_rng(0)
    r, g, dy, v = (rng.standard_normal((3, 40)) for _ in range(4))
    dx, dg = P.norm_backward(r, g[0], 1e-6, dy)
    h = 1e-6
    num = ((P.norm(r + h * v, g[0], 1e-6)[0] - P.norm(r - h * v, g[0], 1e-6)[0]) * dy).sum() / (2 * h)
    assert abs(num - (dx * v).sum()) <= 1e-7 * np.abs(dx * v).sum()
    num = ((P.norm(r, g[0] + h * v[0], 1e-6)[0] - P.norm(r, g[0] - h * v[0], 1e-6)[0]) * dy).sum() / (2 * h)
    assert abs(num - (dg * v[0]).sum()) <= 1e-7 * np.abs(dg * v[0]).sum()
    x = torch.randn(50) * 30
    assert np.array_equal(P.round_e4m3(x.numpy()), x.to(torch.float8_e4m3fn).float().numpy())


def test_entry_points_check_their_arguments():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib, I, A, U = _lib.lib(), _lib.ERR_INVALID, _lib.ERR_ALIGN, _lib.ERR_UNSUPPORTED

    def cast(src=16, dt=0, rows=4, cols=32, ld=32, rm=None, cm=None, cmd=0, sq=0, dst=16, ldd=32, sc=16, dt_=None,
             ldt=0, sct=None):
        return lib.apa_block_cast(src, dt, rows, cols, ld, rm, cm, cmd, sq, dst, ldd, sc, dt_, ldt, sct, None, None)

    assert cast(src=None) == I and cast(rows=0) == I and cast(cols=-1) == I and cast(ld=31) == I
    assert cast(sc=None) == I and cast(dst=None, sc=None) == I and cast(ldd=16) == I and cast(rm=16) == I
    assert cast(dt_=16, ldt=3, sct=16) == I and cast(rows=1 << 31) == I
    assert cast(dt=3) == U and cast(rm=16, cm=16, cmd=3) == U
    assert cast(dst=17) == A and cast(ldd=40) == A and cast(dt_=16, ldt=8, sct=16) == A

    def gemm(a=16, lda=32, sa=16, b=16, ldb=32, sb=16, bias=None, bd=0, out=16, od=0, ldo=8, M=4, N=8, K=32, acc=0, plan=0, ws=None, wb=0):
        return lib.apa_block_gemm(a, lda, sa, b, ldb, sb, bias, bd, out, od, ldo, M, N, K, acc, plan, ws, wb, None)

    assert gemm(a=None) == I and gemm(sa=None) == I and gemm(out=None) == I and gemm(M=0) == I and gemm(K=0) == I
    assert gemm(lda=16) == I and gemm(ldo=7) == I and gemm(N=1 << 31, ldo=1 << 31) == I
    assert gemm(od=3) == U and gemm(bias=16, bd=3) == U and gemm(od=1, acc=1) == U
    def split(bn, n, swap=0):
        return bn | n << 7 | swap << 14

    def pair(ew, n):
        return n << 7 | ew << 15

    for bad in (-1, 1, 3, split(16, 0), split(48, 1), split(64, 2), pair(4, 0), pair(5, 1), pair(4, 2), pair(0, 1),
                pair(4, 1) | 1 << 14, split(64, 1) | 4 << 15, 1 << 19 | pair(4, 1)):
        assert gemm(plan=bad) == I, bad
    assert gemm(plan=split(64, 9), K=4096, lda=4096, ldb=4096) == I
    # tiles of 16 and 32 rows only for a side of one tile
    assert gemm(plan=split(16, 1), N=17, ldo=17) == I and gemm(plan=split(32, 1), N=33, ldo=33) == I
    assert gemm(plan=split(16, 1, 1), M=17) == I and gemm(plan=split(32, 1, 1), M=33) == I
    # a forced split needs its workspace
    big = dict(K=4096, lda=4096, ldb=4096, plan=pair(4, 2))
    assert gemm(**big) == I and gemm(**big, ws=16, wb=2 * 256 * 8 * 4 - 1) == I
    n = ctypes.c_int64(0)
    at = ctypes.addressof(n)
    assert lib.apa_block_gemm_workspace(4, 8, 4096, 0, pair(4, 2), at) == _lib.OK and n.value == 2 * 256 * 8 * 4
    assert lib.apa_block_gemm_workspace(4, 8, 4096, 0, pair(4, 2), None) == I
    assert lib.apa_block_gemm_workspace(4, 0, 4096, 0, 0, at) == I
    assert lib.apa_block_gemm_workspace(4, 8, 4096, 3, 0, at) == U
    assert gemm(ws=8, wb=64) == A
    assert gemm(a=8) == A and gemm(ldb=40) == A and gemm(sb=8) == A

    def fwd(x=16, res=None, g=16, gd=0, dt=0, rows=2, cols=32, st=None, y=16, q=None, sc=None, ldq=32):
        return lib.apa_rmsnorm_fwd(x, 32, res, 32, g, gd, dt, rows, cols, 1e-6, st, 32, y, 32, q, ldq, sc, None, None)

    assert fwd(x=None) == I and fwd(rows=0) == I and fwd(cols=33) == I and fwd(res=16) == I and fwd(st=16) == I
    assert fwd(y=None) == I and fwd(q=16, sc=16) == I and fwd(y=None, q=16) == I
    assert fwd(gd=3) == U and fwd(dt=3) == U and fwd(cols=32769) == U
    assert fwd(y=None, q=8, sc=16) == A
    n = ctypes.c_int64(0)
    assert lib.apa_rmsnorm_bwd_workspace(2, 32, None) == I
    assert lib.apa_rmsnorm_bwd_workspace(0, 32, ctypes.addressof(n)) == I

    def bwd(dy=16, dx=16, dg=16, ws=16, wb=1 << 30, cols=32, dt=0, gd=0, dyt=0):
        return lib.apa_rmsnorm_bwd(dy, dyt, 32, 16, 32, 16, 16, gd, None, 0, dx, 32, dt, 2, cols, dg, ws, wb, None)

    assert bwd(dy=None) == I and bwd(dx=None) == I and bwd(dg=None) == I and bwd(ws=None) == I and bwd(cols=33) == I
    assert bwd(dyt=2) == U and bwd(dt=2, dyt=1) == U
    assert bwd(dt=3) == U and bwd(gd=3) == U and bwd(ws=8) == A
    assert lib.apa_block_dequant(None, 32, 16, 2, 32, 16, 0, 32, None) == I
    assert lib.apa_block_dequant(16, 32, 16, 2, 32, 16, 3, 32, None) == U
    assert lib.apa_block_dequant(8, 32, 16, 2, 32, 16, 0, 32, None) == A
    assert lib.apa_block_colsum(None, 2, 32, 16, 0, None) == I and lib.apa_block_colsum(16, 2, 32, 16, 3, None) == U
