"""Block-scaled FP8: E4M3 tensors with one power-of-two scale per 128 elements,
their products, and the root-mean-square norm that feeds them.

``APALinear`` keeps the reference's arithmetic, which casts to E4M3 without a
scale and climbs to wider types when that loses too much. The operators here
scale every block of 128 elements into E4M3's range instead, so a layer stays
in FP8 whatever the size of its activations, weights and gradients:

    x   activations   one scale per token and 128 features
    W   weights       one scale per 128 x 128
    dy  gradients     one scale per token and 128 features; for the weight
                      gradient one per feature and 128 tokens

Serving:

    wq = block_cast(weight, square=True)            # once
    y = block_linear(x, wq, bias)                   # every call
    q, r = rms_norm(x, gamma, residual=r, quantize=True)
    y = block_linear(q, wq)                         # the norm's E4M3 output as it is

Training (any optimizer; beside ``APALinear`` under one ``APAManager``, whose
overflow checks see these layers' output gradients through its leaf hooks):

    norm = APARMSNorm(d)
    lin = APABlockLinear(d, 4 * d)
    y = lin(x)                                      # or
    y, r = lin(x, norm=norm, residual=r)            # r = x + r; y = lin(norm(r))

All functions run on the current stream of their tensors' device, allocate
with torch's caching allocator, and can be captured in a CUDA graph. Scales
and codes are those of the definition, bit for bit: the smallest power of two
that brings a block's largest finite magnitude to 448 or below (not below
2^-126), and round to nearest even. NaN and infinities become NaN codes and do
not affect the scale.
"""
from __future__ import annotations

import ctypes
import functools
import math
import threading
from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable
from torch.optim.optimizer import register_optimizer_step_post_hook

from . import _lib
from .config import APAConfig

BLOCK = 128
MAX_NORM_FEATURES = 32768

_E4M3 = torch.float8_e4m3fn
_REAL = {torch.float32: _lib.DT_F32, torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}


_fns: dict = {}
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(device: torch.device, name: str, *args) -> None:
    """One library call on the current stream of the tensors' device, which
    need not be the current device. The stream is the call's last argument."""
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_lib.lib(), name)
    if device.index == _current_device():
        _lib.check(fn(*args, _lib.stream_handle(device)), name)
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, _lib.stream_handle(device)), name)


def _sizes(device: int, name: str, *args) -> int:
    """A size that the library computes for a device."""
    n = ctypes.c_int64(0)
    with torch.cuda.device(device):
        _lib.check(getattr(_lib.lib(), name)(*args, ctypes.addressof(n)), name)
    return n.value


def _real(dtype: torch.dtype, what: str) -> int:
    code = _REAL.get(dtype)
    if code is None:
        raise TypeError(f"{what}: expected float32, float16 or bfloat16, got {dtype}")
    return code


def _matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    """x as a 2-D matrix with unit column stride, rows a positive distance apart."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(x).__name__}")
    d = x.dim()
    if d < 1:
        raise ValueError(f"{what}: expected at least one dimension")
    n = x.shape[-1]
    if n == 0:
        raise ValueError(f"{what}: has no columns")
    m = x if d == 2 else x.reshape(-1, n)
    if not m.is_contiguous() and ((n > 1 and m.stride(1) != 1) or (m.shape[0] > 1 and m.stride(0) < n)):
        m = m.contiguous()
    return m


def _ld(m: torch.Tensor) -> int:
    """Row pitch of a matrix from _matrix (a single row's stride may be anything)."""
    return m.stride(0) if m.shape[0] > 1 else m.shape[1]


def _same_device(what: str, device: torch.device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: tensors on {device} and {t.device}")


def _vector(t: torch.Tensor, n: int, device: torch.device, what: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{what}: expected shape [{n}], got {list(t.shape)}")
    _real(t.dtype, what)
    _same_device(what, device, t)
    return t if t.stride(0) == 1 else t.contiguous()


def _pitch(cols: int) -> int:
    return (cols + 15) & ~15


def _packed_bytes(rows: int, cols: int) -> int:
    """Codes with a row pitch of 16 bytes' multiple, then the scales: a 32-bit
    word per row (rounded up to 128 rows) and 512 columns."""
    return rows * _pitch(cols) + ((cols + 511) >> 9) * ((rows + 127) & ~127) * 4


class APABlockTensor:
    """A [rows, cols] matrix held as E4M3 codes with one scale per row and 128
    columns. ``data`` holds the codes; ``scales`` one byte per block (2^(b-127))
    in the order the tensor cores take, see ``exponents()`` for the plain one.
    ``buffer`` is a flat uint8 tensor on a 16-byte boundary: the codes, row by
    row with a pitch of ``cols`` rounded up to 16, then the scales.
    """

    __slots__ = ("buffer", "rows", "cols")

    def __init__(self, buffer: torch.Tensor, rows: int, cols: int):
        # the kernels read as many bytes as rows and cols say
        if not isinstance(buffer, torch.Tensor) or buffer.dtype != torch.uint8 or buffer.dim() != 1:
            raise TypeError("APABlockTensor: buffer must be a flat uint8 tensor")
        if rows < 0 or cols <= 0:
            raise ValueError(f"APABlockTensor: bad shape [{rows}, {cols}]")
        if buffer.numel() < _packed_bytes(rows, cols) or not buffer.is_contiguous() or buffer.data_ptr() % 16:
            raise ValueError(f"APABlockTensor: [{rows}, {cols}] takes {_packed_bytes(rows, cols)} contiguous bytes "
                             "on a 16-byte boundary")
        self.buffer, self.rows, self.cols = buffer, rows, cols

    @property
    def data(self) -> torch.Tensor:
        pitch = _pitch(self.cols)
        return self.buffer[:self.rows * pitch].view(_E4M3).view(self.rows, pitch)[:, :self.cols]

    @property
    def scales(self) -> torch.Tensor:
        return self.buffer[self.rows * _pitch(self.cols):_packed_bytes(self.rows, self.cols)]

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.rows, self.cols))

    @property
    def device(self) -> torch.device:
        return self.buffer.device

    def _at(self) -> Tuple[int, int, int]:
        """Addresses of codes and scales, and the codes' pitch."""
        p, pitch = self.buffer.data_ptr(), _pitch(self.cols)
        return p, pitch, p + self.rows * pitch

    def __repr__(self) -> str:
        return f"APABlockTensor({list(self.shape)}, device={self.device})"

    @classmethod
    def from_parts(cls, data: torch.Tensor, exponents: torch.Tensor) -> "APABlockTensor":
        """From E4M3 codes [rows, cols] and integer exponents p (scale 2^p,
        -127 <= p <= 127) of shape [rows, ceil(cols / 128)], or
        [ceil(rows / 128), ceil(cols / 128)] for 128 x 128 blocks."""
        if data.dim() != 2 or data.dtype != _E4M3:
            raise ValueError("APABlockTensor.from_parts: data must be a 2-D float8_e4m3fn tensor")
        rows, cols = data.shape
        if rows == 0 or cols == 0:
            raise ValueError("APABlockTensor.from_parts: data is empty")
        kb = (cols + 127) // 128
        e = exponents
        if e.is_floating_point() or e.is_complex() or e.dtype == torch.bool:
            raise TypeError("APABlockTensor.from_parts: exponents must be integers")
        _same_device("APABlockTensor.from_parts", data.device, e)
        if tuple(e.shape) == (rows, kb):
            pass
        elif tuple(e.shape) == ((rows + 127) // 128, kb):
            e = e.repeat_interleave(128, dim=0)[:rows]
        else:
            raise ValueError(f"APABlockTensor.from_parts: exponents of shape {list(exponents.shape)} for codes "
                             f"{list(data.shape)}")
        e = e.to(torch.int32)
        if int(e.min()) < -127 or int(e.max()) > 127:
            raise ValueError("APABlockTensor.from_parts: exponents must lie in -127 .. 127")
        rp, kp = (rows + 127) & ~127, (kb + 3) & ~3
        full = torch.full((rp, kp), 127, dtype=torch.uint8, device=data.device)
        full[:rows, :kb] = (e + 127).to(torch.uint8)
        # [row group, quarter, lane, word, byte] -> [word, row group, lane, quarter, byte]
        t = _new_block(rows, cols, data.device)
        t.scales.copy_(full.view(rp // 128, 4, 32, kp // 4, 4).permute(3, 0, 2, 1, 4).reshape(-1))
        t.data.view(torch.uint8).copy_(data.view(torch.uint8))
        return t

    def exponents(self) -> torch.Tensor:
        """int32 [rows, ceil(cols / 128)]: block b of row r has the scale 2^exponents[r, b]."""
        rows, cols = self.shape
        rp, kb = (rows + 127) & ~127, (cols + 127) // 128
        kg = (kb + 3) // 4
        full = self.scales.view(kg, rp // 128, 32, 4, 4).permute(1, 3, 2, 0, 4).reshape(rp, kg * 4)
        return full[:rows, :kb].to(torch.int32) - 127

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values code * scale, in ``dtype`` (exact in float32 and, within
        its range, bfloat16)."""
        code = _real(dtype, "APABlockTensor.dequantize")
        _lib.require_cuda(self.buffer, "APABlockTensor.dequantize")
        rows, cols = self.rows, self.cols
        out = torch.empty(rows, cols, dtype=dtype, device=self.device)
        if rows:
            p, pitch, sc = self._at()
            _call(self.device, "apa_block_dequant", p, pitch, sc, rows, cols, out.data_ptr(), code, cols)
        return out


def _new_block(rows: int, cols: int, device) -> APABlockTensor:
    t = object.__new__(APABlockTensor)       # what the constructor checks holds
    t.buffer = torch.empty(_packed_bytes(rows, cols), dtype=torch.uint8, device=device)
    t.rows, t.cols = rows, cols
    return t


_NONE = (None, 0, None)


def _cast(x2: torch.Tensor, rows_form: bool, cols_form: bool, square: bool = False, colsum=None, row_mul=None,
          col_mul=None, into: Optional[APABlockTensor] = None):
    rows, cols = x2.shape
    dev = x2.device
    q = (into or _new_block(rows, cols, dev)) if rows_form else None
    qt = _new_block(cols, rows, dev) if cols_form else None
    if rows == 0:
        return q, qt
    _call(dev, "apa_block_cast", x2.data_ptr(), _REAL[x2.dtype], rows, cols, _ld(x2), _lib.ptr(row_mul),
          _lib.ptr(col_mul), _REAL[col_mul.dtype] if col_mul is not None else 0, int(square),
          *(q._at() if q else _NONE), *(qt._at() if qt else _NONE), _lib.ptr(colsum))
    return q, qt


def block_cast(x: torch.Tensor, form: str = "rows", square: bool = False):
    """Cast a matrix (leading dimensions are flattened) to an APABlockTensor.

    ``form`` "rows": x itself, scales per row and 128 columns; "cols": its
    transpose [cols, rows], scales per column of x and 128 rows (the operand
    of a product that reduces over x's rows); "both": the pair. ``square``:
    one scale per 128 x 128 block (weights), so both forms hold the same
    values. Not differentiable; ``APABlockLinear`` is.
    """
    if form not in ("rows", "cols", "both"):
        raise ValueError(f"block_cast: form must be 'rows', 'cols' or 'both', got {form!r}")
    x2 = _matrix(x, "block_cast")
    _real(x2.dtype, "block_cast")
    _lib.require_cuda(x2, "block_cast")
    if x2.shape[0] == 0 and form != "rows":
        raise ValueError("block_cast: the transpose of a matrix without rows has no columns")
    q, qt = _cast(x2, form != "cols", form != "rows", square)
    return (q, qt) if form == "both" else q if form == "rows" else qt


@functools.lru_cache(maxsize=1024)
def _matmul_workspace(M: int, N: int, K: int, dtype: int, plan: int, device: int) -> int:
    return _sizes(device, "apa_block_gemm_workspace", M, N, K, dtype, plan)


def _matmul(a: APABlockTensor, b: APABlockTensor, bias, out: torch.Tensor, accumulate: bool, plan: int = 0) -> None:
    M, K, N = a.rows, a.cols, b.rows
    dt = _REAL[out.dtype]
    n = _matmul_workspace(M, N, K, dt, plan, a.device.index)
    ws = torch.empty(n, dtype=torch.uint8, device=a.device) if n else None
    _call(a.device, "apa_block_gemm", *a._at(), *b._at(), _lib.ptr(bias), _REAL[bias.dtype] if bias is not None else 0,
          out.data_ptr(), dt, _ld(out), M, N, K, int(accumulate), plan, _lib.ptr(ws), n)


def _no_gradient(what: str, a, b) -> None:
    """Refuses what wants a gradient (each may be None)."""
    if ((a is not None and a.requires_grad) or (b is not None and b.requires_grad)) and torch.is_grad_enabled():
        raise RuntimeError(f"{what}: has no gradient; call it under torch.no_grad(), or train through APABlockLinear")


def block_matmul(a: APABlockTensor, b: APABlockTensor, bias: Optional[torch.Tensor] = None,
                 out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None,
                 accumulate: bool = False) -> torch.Tensor:
    """a [M, K] times the transpose of b [N, K], plus bias [N]: [M, N].

    Accumulated in fp32 and rounded once to ``out_dtype`` (float32, float16
    or bfloat16). ``out``: written in place (unit column stride); with
    ``accumulate`` the product is added to a float32 ``out``. Not
    differentiable (a bias or an ``out`` that wants a gradient is refused)."""
    if not isinstance(a, APABlockTensor) or not isinstance(b, APABlockTensor):
        raise TypeError("block_matmul: both operands must be APABlockTensors")
    _lib.require_cuda(a.buffer, "block_matmul")
    _same_device("block_matmul", a.device, b.buffer)
    M, K, N = a.rows, a.cols, b.rows
    if b.cols != K:
        raise ValueError(f"block_matmul: operands reduce over {K} and {b.cols} columns")
    if N == 0:
        raise ValueError("block_matmul: the second operand has no rows")
    if bias is not None:
        bias = _vector(bias, N, a.device, "block_matmul: bias")
    _no_gradient("block_matmul", bias, out)
    if accumulate and out is None:
        raise ValueError("block_matmul: accumulate needs out")
    given = out is not None
    if not given:
        _real(out_dtype, "block_matmul: out_dtype")
        out = torch.empty(M, N, dtype=out_dtype, device=a.device)
    else:
        _real(out.dtype, "block_matmul: out")
        _same_device("block_matmul: out", a.device, out)
        if tuple(out.shape) != (M, N) or (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
            raise ValueError(f"block_matmul: out must be a row-major [{M}, {N}] tensor")
        if accumulate and out.dtype != torch.float32:
            raise ValueError("block_matmul: accumulate needs a float32 out")
    if M:
        _matmul(a, b, bias, out, accumulate)
        if given and not out.is_inference():
            # autograd refuses a backward that would read the values from before
            torch.autograd.graph.increment_version(out)
    return out


def block_linear(x: Union[torch.Tensor, APABlockTensor], weight: APABlockTensor, bias: Optional[torch.Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x W^T + bias for serving. x [..., K] is cast to E4M3 here, or comes as an
    APABlockTensor (from ``rms_norm(..., quantize=True)``); ``weight`` [N, K] is
    ``block_cast(w, square=True)``. ``out_dtype`` defaults to x's type
    (bfloat16 for an APABlockTensor). Not differentiable (an x or a bias that
    wants a gradient is refused)."""
    if isinstance(x, APABlockTensor):
        return block_matmul(x, weight, bias, out_dtype or torch.bfloat16)
    if not isinstance(weight, APABlockTensor):
        raise TypeError("block_linear: the weight must be an APABlockTensor (block_cast(w, square=True))")
    x2 = _matrix(x, "block_linear")
    code = _real(x2.dtype, "block_linear")
    _lib.require_cuda(x2, "block_linear")
    M, K = x2.shape
    N = weight.rows
    dev = x2.device
    if K != weight.cols:
        raise ValueError(f"block_linear: x has {K} features, the weight {weight.cols}")
    _same_device("block_linear", dev, weight.buffer)
    if bias is not None:
        bias = _vector(bias, N, dev, "block_linear: bias")
    _no_gradient("block_linear", x, bias)
    out_code = code if out_dtype is None else _real(out_dtype, "block_linear: out_dtype")
    y = torch.empty(M, N, dtype=out_dtype or x2.dtype, device=dev)
    if M:
        _linear_forward(x2, code, None, None, 0.0, None, None, None, None, weight.buffer.data_ptr(), None, bias, y,
                        out_code, M, N, K)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


@functools.lru_cache(maxsize=4096)
def _forward_workspace(M: int, N: int, K: int, flags: int, dtype: int, device: int) -> int:
    return _sizes(device, "apa_block_linear_fwd_workspace", M, N, K, flags, dtype)


def _linear_forward(x2, code, res2, gamma, eps, stream, rstd, w2, xt, wq, wt, bias, y, out_code, M, N, K) -> None:
    """apa_block_linear_fwd with its temporaries in one buffer. The weight is
    w2, or wq, the address of its packed cast; xt, wt: addresses for the
    transposed casts."""
    dev = x2.device
    flags = (0 if w2 is None else 1) | (0 if gamma is None else 2) | (0 if xt is None else 4)
    n = _forward_workspace(M, N, K, flags, out_code, dev.index)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _call(dev, "apa_block_linear_fwd", x2.data_ptr(), code, _ld(x2),
          _lib.ptr(res2), _ld(res2) if res2 is not None else 0,
          _lib.ptr(gamma), _REAL[gamma.dtype] if gamma is not None else 0, eps, _lib.ptr(stream), K, _lib.ptr(rstd),
          xt, _lib.ptr(w2), _REAL[w2.dtype] if w2 is not None else 0, _ld(w2) if w2 is not None else 0, wq, wt,
          _lib.ptr(bias), _REAL[bias.dtype] if bias is not None else 0, y.data_ptr(), out_code, N, M, N, K,
          _lib.ptr(ws), n)


# ---------------------------------------------------------------------------
# root-mean-square norm
# ---------------------------------------------------------------------------
def _norm_weight(norm: nn.Module):
    """A norm module's weight. nn.Module's own lookup takes a microsecond; it
    serves a weight that something else computes (a parametrization, pruning, a
    replica of DataParallel)."""
    try:
        return norm._parameters["weight"]
    except KeyError:
        return norm.weight


def _norm_args(x, weight, residual, what: str):
    x2 = _matrix(x, what)
    _real(x2.dtype, what)
    _lib.require_cuda(x2, what)
    K = x2.shape[1]
    if K > MAX_NORM_FEATURES:
        raise ValueError(f"{what}: at most {MAX_NORM_FEATURES} features, got {K}")
    g = _vector(weight, K, x2.device, f"{what}: weight")
    r2 = None
    if residual is not None:
        if not isinstance(residual, torch.Tensor):
            raise TypeError(f"{what}: residual: expected a tensor, got {type(residual).__name__}")
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"{what}: residual {residual.dtype} {list(residual.shape)} does not match x {x.dtype} "
                             f"{list(x.shape)}")
        _same_device(what, x2.device, residual)
        r2 = _matrix(residual, what)
    return x2, g, r2


def _check_eps(eps: float, what: str) -> float:
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"{what}: eps must be finite and not negative")
    return float(eps)


def _norm_forward(x2, g, res2, eps: float, quantize: bool, want_rstd: bool):
    """(output, stream, rstd): output an APABlockTensor or a matrix of x's type."""
    M, K = x2.shape
    dev = x2.device
    stream = torch.empty(M, K, dtype=x2.dtype, device=dev) if res2 is not None else None
    q = _new_block(M, K, dev) if quantize else None
    y = None if quantize else torch.empty(M, K, dtype=x2.dtype, device=dev)
    rstd = torch.empty(M, dtype=torch.float32, device=dev) if want_rstd else None
    if M:
        _call(dev, "apa_rmsnorm_fwd", x2.data_ptr(), _ld(x2), _lib.ptr(res2), _ld(res2) if res2 is not None else 0,
              g.data_ptr(), _REAL[g.dtype], _REAL[x2.dtype], M, K, eps, _lib.ptr(stream), K, _lib.ptr(y), K,
              *(q._at() if q else _NONE), _lib.ptr(rstd))
    return (q if quantize else y), stream, rstd


@functools.lru_cache(maxsize=1024)
def _norm_workspace(M: int, K: int, device: int) -> int:
    return _sizes(device, "apa_rmsnorm_bwd_workspace", M, K)


def _norm_backward(dh2, r2, rstd, g, dr2):
    """(dx, dgamma)."""
    M, K = r2.shape
    dev = r2.device
    dx = torch.empty(M, K, dtype=r2.dtype, device=dev)
    dg = torch.empty(K, dtype=g.dtype, device=dev)
    if M == 0:
        return dx, dg.zero_()
    n = _norm_workspace(M, K, dev.index)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _call(dev, "apa_rmsnorm_bwd", dh2.data_ptr(), _REAL[dh2.dtype], _ld(dh2), r2.data_ptr(), _ld(r2), rstd.data_ptr(),
          g.data_ptr(), _REAL[g.dtype], _lib.ptr(dr2), _ld(dr2) if dr2 is not None else 0, dx.data_ptr(), K,
          _REAL[r2.dtype], M, K, dg.data_ptr(), ws.data_ptr(), n)
    return dx, dg


def _grad_matrix(g, dtype, K: int):
    """A gradient from autograd as a matrix of the operator's type (None stays None)."""
    if g is None:
        return None
    if g.dtype != dtype:
        g = g.to(dtype)
    return _matrix(g if g.dim() == 2 else g.reshape(-1, K), "gradient")


def _first_order(fn):
    """A backward without a second derivative. torch's decorator costs two
    microseconds a call, so it is used only where a graph of the gradient is
    being built."""
    graphed = once_differentiable(fn)

    @functools.wraps(fn)
    def backward(ctx, *grads):
        return graphed(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return backward


class _RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        x2, g, res2 = _norm_args(x, weight, residual, "rms_norm")
        y, stream, rstd = _norm_forward(x2, g, res2, eps, False, True)
        ctx.set_materialize_grads(False)
        ctx.has_res = residual is not None
        ctx.shape = x.shape
        flat = x.dim() == 2
        if not flat:
            y = y.view(x.shape)
        if residual is None:
            ctx.save_for_backward(x, weight, rstd)
            return y
        if not flat:
            stream = stream.view(x.shape)
        ctx.save_for_backward(stream, weight, rstd)
        return y, stream

    @staticmethod
    @_first_order
    def backward(ctx, dy, dr=None):
        r, weight, rstd = ctx.saved_tensors
        K = weight.shape[0]
        if dy is None:
            return dr, None, dr if ctx.has_res else None, None
        dx, dg = _norm_backward(_grad_matrix(dy, r.dtype, K), _matrix(r, "rms_norm"), rstd, weight.contiguous(),
                                _grad_matrix(dr, r.dtype, K))
        if dx.shape != ctx.shape:
            dx = dx.view(ctx.shape)
        return dx, dg, dx if ctx.has_res else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
             quantize: bool = False):
    """Root-mean-square norm over the last dimension, with the residual's
    addition: r = x + residual (rounded to x's type), y = r / sqrt(mean(r^2) +
    eps) * weight. Returns y, or (y, r) when a residual is given.

    ``quantize``: y as an APABlockTensor [rows, K], rounded once from fp32 to
    E4M3 under its blocks' scales (not differentiable; use ``APABlockLinear``
    with ``norm=`` for training). Otherwise y has x's type and gradients flow
    to x, residual and weight."""
    eps = _check_eps(eps, "rms_norm")
    if not quantize:
        return _RMSNormFn.apply(x, weight, residual, eps)
    x2, g, res2 = _norm_args(x, weight, residual, "rms_norm")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        raise RuntimeError("rms_norm: the E4M3 output has no gradient; call it under torch.no_grad(), or train through "
                           "APABlockLinear(...)(x, norm=norm, residual=residual)")
    q, stream, _ = _norm_forward(x2, g, res2, eps, True, False)
    return q if residual is None else (q, stream.view(x.shape))


class APARMSNorm(nn.Module):
    """``rms_norm`` with its weight: ``norm(x)`` or ``y, r = norm(x, residual)``."""

    def __init__(self, features: int, eps: float = 1e-6, dtype: torch.dtype = torch.float32,
                 config: APAConfig = APAConfig()):
        super().__init__()
        if not 0 < features <= MAX_NORM_FEATURES:
            raise ValueError(f"APARMSNorm: features must lie in 1 .. {MAX_NORM_FEATURES}, got {features}")
        _real(dtype, "APARMSNorm")
        self.features = features
        self.eps = _check_eps(eps, "APARMSNorm")
        self.weight = nn.Parameter(torch.ones(features, dtype=dtype, device=torch.device(config.device)))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, quantize: bool = False):
        return rms_norm(x, _norm_weight(self), residual, self.eps, quantize)

    def extra_repr(self) -> str:
        return f"{self.features}, eps={self.eps}"


# ---------------------------------------------------------------------------
# linear layer
# ---------------------------------------------------------------------------
@functools.lru_cache(maxsize=1024)
def _linear_workspace(M: int, N: int, K: int, flags: int, dtype: int, dw_dtype: int, device: int) -> int:
    return _sizes(device, "apa_block_linear_bwd_workspace", M, N, K, flags, dtype, dw_dtype)


class _BlockLinearFn(torch.autograd.Function):
    """y = (norm of x + residual, or x) W^T + b with E4M3 operands; the casts
    pass gradients straight through."""

    @staticmethod
    def forward(ctx, x, residual, gamma, weight, bias, eps):
        ctx.set_materialize_grads(False)
        need = ctx.needs_input_grad
        need_in = need[0] or need[1] or need[2]
        N, K = weight.shape
        dev = x.device
        has_norm = gamma is not None
        if has_norm:
            x2, g, res2 = _norm_args(x, gamma, residual, "APABlockLinear")
        else:
            x2, g, res2 = _matrix(x, "APABlockLinear"), None, None
        M = x2.shape[0]
        y = torch.empty(M, N, dtype=x.dtype, device=dev)
        stream = torch.empty(M, K, dtype=x.dtype, device=dev) if res2 is not None else None
        rstd = torch.empty(M, dtype=torch.float32, device=dev) if has_norm else None
        # what the backward reads: the transposed cast of x (recomputed behind a
        # norm) and of the weight, in one buffer
        n_xt = (_packed_bytes(K, M) + 255) & ~255 if need[3] and not has_norm and M else 0
        n_wt = _packed_bytes(K, N) if need_in and M else 0
        keep = torch.empty(n_xt + n_wt, dtype=torch.uint8, device=dev) if n_xt + n_wt else None
        if M:
            p = keep.data_ptr() if keep is not None else 0
            code = _REAL[x.dtype]
            _linear_forward(x2, code, res2, g, eps, stream, rstd, _matrix(weight, "APABlockLinear: weight"),
                            p if n_xt else None, None, p + n_xt if n_wt else None,
                            _vector(bias, N, dev, "APABlockLinear: bias") if bias is not None else None, y, code, M, N,
                            K)
        ctx.n_xt = n_xt
        ctx.has_res, ctx.has_norm = residual is not None, has_norm
        ctx.meta = (x.shape, M, N, K, x.dtype, weight.dtype, bias.dtype if bias is not None else None)
        if y.shape[:-1] != x.shape[:-1]:
            y = y.view(*x.shape[:-1], N)
        # saved as tensors: freed by the backward, refused to a second one, and
        # seen by hooks (checkpointing, offloading)
        if not has_norm:
            ctx.save_for_backward(keep)
            return y
        stream = x if stream is None else stream.view(x.shape)
        ctx.save_for_backward(keep, rstd, stream, gamma)
        return (y, stream) if residual is not None else y

    @staticmethod
    @_first_order
    def backward(ctx, dy, dr=None):
        need = ctx.needs_input_grad
        has_norm, has_res = ctx.has_norm, ctx.has_res
        if dy is None:
            return (dr if need[0] else None, dr if has_res and need[1] else None, None, None, None, None)
        saved = ctx.saved_tensors
        keep = saved[0]
        shape, M, N, K, dtype, wdtype, bdtype = ctx.meta
        need_in = need[0] or need[1] or need[2]
        dev = dy.device
        dx = torch.empty(M, K, dtype=dtype, device=dev) if need_in else None
        dw = torch.empty(N, K, dtype=wdtype, device=dev) if need[3] else None
        db = torch.empty(N, dtype=bdtype, device=dev) if need[4] else None
        dg = None
        rstd = stream = gamma = None
        if has_norm:
            _, rstd, stream, gamma = saved
            if need_in:
                dg = torch.empty(K, dtype=gamma.dtype, device=dev)
        if M:
            dy2 = _grad_matrix(dy, dtype, N)
            dr2 = _grad_matrix(dr, dtype, K) if has_norm and need_in else None
            if has_norm:
                stream, gamma = _matrix(stream, "APABlockLinear"), gamma.contiguous()
            code, wcode = _REAL[dtype], _REAL[wdtype]
            flags = (1 if need_in else 0) | (2 if need[3] else 0) | (4 if need[4] else 0) | (8 if has_norm else 0)
            n = _linear_workspace(M, N, K, flags, code, wcode, dev.index)
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            p = keep.data_ptr() if keep is not None else 0
            _call(dev, "apa_block_linear_bwd", dy2.data_ptr(), code, _ld(dy2), p + ctx.n_xt if need_in else None,
                  p if ctx.n_xt else None, _lib.ptr(stream), _ld(stream) if has_norm else 0, _lib.ptr(rstd),
                  _lib.ptr(gamma), _REAL[gamma.dtype] if has_norm else 0, _lib.ptr(dr2),
                  _ld(dr2) if dr2 is not None else 0, _lib.ptr(dx), code, K, _lib.ptr(dg), _lib.ptr(dw), wcode, K,
                  _lib.ptr(db), _REAL[bdtype] if db is not None else 0, M, N, K, ws.data_ptr(), n)
        else:
            for t in (dx, dw, db, dg):
                if t is not None:
                    t.zero_()
        if dx is not None and dx.shape != shape:
            dx = dx.view(shape)
        return (dx if need[0] else None, dx if has_res and need[1] else None, dg if need[2] else None, dw, db, None)


_optimizer_steps = 0


def _count_optimizer_step(*_) -> None:
    global _optimizer_steps
    _optimizer_steps += 1


# Fused optimizers change parameters without raising their version counters, so
# a step of any torch.optim optimizer (subclasses too) counts as a change.
register_optimizer_step_post_hook(_count_optimizer_step)


def _capturing(stream) -> bool:
    """Whether a capture is under way on ``stream``: it can be neither waited
    for nor, since a capture begins behind what its stream held, need be."""
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


class _KeptWeight:
    """A layer's cast weight: the block tensor, the parameter that it was cast
    from and that one's state then, an event behind the cast, and the streams
    that are ordered behind it and may read it, by handle."""

    __slots__ = ("block", "weight", "state", "done", "streams")

    def __init__(self, block, weight, state, done, streams):
        self.block, self.weight, self.state, self.done, self.streams = block, weight, state, done, streams


class APABlockLinear(nn.Module):
    """A linear layer whose three products run on block-scaled E4M3 operands.

    ``weight_master`` [out, in] and ``bias_master`` [out] are ordinary
    parameters in ``dtype`` (float32 masters, or bfloat16); their gradients come
    in the same type. Output and input gradient have x's type. In training
    every forward casts the weight anew; without gradients the layer keeps its
    cast weight and renews it when the parameter was replaced, when autograd's
    version counter shows a change in place, after a training forward and after
    any ``torch.optim`` optimizer's step. Call ``refresh_working_copy()`` after
    changes behind all of these: through ``.data``, by a collective or by a
    replayed graph. A weight made under ``torch.inference_mode()`` has no version
    counter and is cast on every call.

    ``forward(x, norm=None, residual=None)``: with ``norm`` (an ``APARMSNorm``)
    the layer is applied to ``norm(x)``, or to the normalised sum x + residual;
    the norm writes the E4M3 operand itself. With a residual the result is
    (y, x + residual)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, dtype: torch.dtype = torch.float32,
                 config: APAConfig = APAConfig()):
        super().__init__()
        if in_features <= 0 or out_features <= 0:
            raise ValueError("APABlockLinear: in_features and out_features must be positive")
        _real(dtype, "APABlockLinear")
        self.in_features = in_features
        self.out_features = out_features
        dev = torch.device(config.device)
        self.weight_master = nn.Parameter(torch.empty(out_features, in_features, dtype=dtype, device=dev))
        nn.init.kaiming_uniform_(self.weight_master, a=math.sqrt(5))
        if bias:
            bound = 1 / math.sqrt(in_features)
            self.bias_master = nn.Parameter(torch.empty(out_features, dtype=dtype, device=dev).uniform_(-bound, bound))
        else:
            self.register_parameter("bias_master", None)
        self._kept: Optional[_KeptWeight] = None
        self._lock = threading.Lock()        # around renewing _kept and adding streams to it

    @property
    def _wq(self) -> Optional[APABlockTensor]:
        kept = self._kept
        return None if kept is None else kept.block

    def refresh_working_copy(self) -> None:
        """Cast the weight for calls without gradients (buffers are kept, so a
        captured graph of such a call sees the new values). Products queued
        before are waited for, on whichever stream the layer was called;
        replays of captured calls are the caller's to order."""
        W = self.weight_master
        _lib.require_cuda(W, "APABlockLinear.refresh_working_copy")
        with self._lock, torch.cuda.device(W.device):
            self._renew(W)

    def _renew(self, W: torch.Tensor) -> Optional[_KeptWeight]:
        """Cast W into the kept buffer. The caller holds the lock and has made
        W's device current."""
        capturing = torch.cuda.is_current_stream_capturing()
        old = self._kept
        if capturing and old is None:
            raise RuntimeError("APABlockLinear.refresh_working_copy: nothing to renew in a captured graph; "
                               "call it once before the capture")
        into = None
        if old is not None and old.block.device == W.device and old.block.shape == W.shape:
            into = old.block
        stream = torch.cuda.current_stream()
        if into is not None and not capturing:
            # products queued on other streams may still read the buffer that is rewritten
            for handle, other in old.streams.items():
                if handle != stream.cuda_stream and not _capturing(other):
                    stream.wait_stream(other)
            into.buffer.record_stream(stream)
        state = self._state(W)               # before the cast: a change during it shows later
        block = self._cast_weight(W, into)
        if capturing:                        # the cast happens when the graph runs
            if into is None:
                self._kept = _KeptWeight(block, None, None, None, {})
            return None
        done = torch.cuda.Event()
        done.record()
        # one store: a reader sees the old event and streams or the new ones
        self._kept = kept = _KeptWeight(block, W, state, done, {stream.cuda_stream: stream})
        return kept

    @staticmethod
    def _cast_weight(W: torch.Tensor, into: Optional[APABlockTensor] = None) -> APABlockTensor:
        # written by the kernel alone: a buffer made in inference mode allows no torch operation in place
        return _cast(_matrix(W.detach(), "APABlockLinear: weight"), True, False, square=True, into=into)[0]

    def _working_copy(self, W: torch.Tensor) -> APABlockTensor:
        """The kept cast of W, renewed where W changed and ordered before the
        current stream's work. A capture that would have to renew it records a
        cast of its own, which nothing outside the graph sees."""
        if W.is_inference():
            # it has no version counter, and inference mode may change it in
            # place: nothing shows whether a cast still holds
            with torch.cuda.device(W.device):
                return self._cast_weight(W)
        handle = _lib.stream_handle(W.device)
        kept = self._kept
        if kept is not None and kept.weight is W and handle in kept.streams and kept.state == self._state(W):
            return kept.block
        with torch.cuda.device(W.device):
            if torch.cuda.is_current_stream_capturing():
                # a capture starts behind what it reads
                return kept.block if self._current(kept, W) else self._cast_weight(W)
            with self._lock:
                kept = self._kept
                if not self._current(kept, W):
                    kept = self._renew(W)
                elif handle not in kept.streams:
                    stream = torch.cuda.current_stream()
                    stream.wait_event(kept.done)
                    kept.block.buffer.record_stream(stream)
                    kept.streams[handle] = stream
                return kept.block

    def _current(self, kept: Optional[_KeptWeight], W: torch.Tensor) -> bool:
        return kept is not None and kept.weight is W and kept.state == self._state(W)

    def __getstate__(self):
        state = self.__dict__.copy()
        state["_kept"] = None                # a copy casts its own weight
        del state["_lock"]
        return state

    def __setstate__(self, state):
        super().__setstate__(state)
        self._kept, self._lock = None, threading.Lock()

    @staticmethod
    def _state(W: torch.Tensor) -> Tuple:
        # a tensor made in inference mode has no version, so its cast is never taken as current
        return (None if W.is_inference() else W._version, W.data_ptr(), W.dtype, _optimizer_steps)

    def forward(self, x: torch.Tensor, norm: Optional[APARMSNorm] = None, residual: Optional[torch.Tensor] = None):
        p = self._parameters           # as in _norm_weight
        try:
            W, b = p["weight_master"], p["bias_master"]
        except KeyError:
            W, b = self.weight_master, self.bias_master
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"APABlockLinear: expected a tensor, got {type(x).__name__}")
        if x.dim() < 1 or x.shape[-1] != self.in_features:
            raise ValueError(f"APABlockLinear: input of shape {list(x.shape)}, expected {self.in_features} features")
        gamma, eps = None, 0.0
        if norm is not None:
            if norm.features != self.in_features:
                raise ValueError(f"APABlockLinear: norm over {norm.features} features, expected {self.in_features}")
            gamma, eps = _norm_weight(norm), norm.eps
            if residual is not None and not isinstance(residual, torch.Tensor):
                raise TypeError(f"APABlockLinear: residual: expected a tensor, got {type(residual).__name__}")
        elif residual is not None:
            raise ValueError("APABlockLinear: residual needs norm")
        _real(x.dtype, "APABlockLinear")
        _lib.require_cuda(x, "APABlockLinear")
        _same_device("APABlockLinear", x.device, W, residual)
        if torch.is_grad_enabled() and (W.requires_grad or x.requires_grad or (b is not None and b.requires_grad)
                                        or (gamma is not None and gamma.requires_grad)
                                        or (residual is not None and residual.requires_grad)):
            kept = self._kept
            if W.requires_grad and kept is not None:
                kept.state = None           # an update follows, by whatever means
            return _BlockLinearFn.apply(x, residual, gamma, W, b, eps)
        wq = self._working_copy(W)
        if norm is None:
            return block_linear(x, wq, b)
        out = rms_norm(x.detach(), gamma.detach(), residual.detach() if residual is not None else None, eps, True)
        q = out if residual is None else out[0]
        y = block_matmul(q, wq, b, x.dtype).view(*x.shape[:-1], self.out_features)
        return y if residual is None else (y, out[1])

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias_master is not None}"
