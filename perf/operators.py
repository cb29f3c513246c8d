"""What the block-scaled FP8 operators of the package ``apa`` are measured on.

Operators (E4M3 values with one power-of-two scale per block of 128):

  linear     y = x W^T + b for serving: x is cast to E4M3 with a scale per row
             and 128 features, W is kept as E4M3 with a scale per 128 x 128
  step       the same layer in training: y, dx, dW and db, the weight cast of
             the step included
  norm       root-mean-square norm with the residual's addition, its output in
             E4M3 with a scale per row and 128 features
  norm_step  the norm in training: y, the residual stream, dx and dgamma
  block      both together in training: residual addition, norm and linear
             layer, forward and backward

``own`` False computes them in their plain form (elementary torch operations
in fp32); True calls the package. ``exact`` is the definition in fp64.
"""
import math
import os
import sys

import torch

own = False

F32, F16, BF16 = "float32", "float16", "bfloat16"
EPS = 1e-6


def listed():
    return [
        # one token of one sequence through a projection of the 4096-wide layer: all latency
        dict(name="linear 1x4096x4096", kind="linear", rows=1, k=4096, n=4096, dtype=BF16, bias=False),
        # a decode batch of 61 sequences through a GPT-2-medium MLP projection, with its bias
        dict(name="linear 61x1024x4096", kind="linear", rows=61, k=1024, n=4096, dtype=BF16, bias=True),
        # the forward of the 4096-wide layer over a full batch: bound by the tensor cores
        dict(name="linear 8192x4096x4096", kind="linear", rows=8192, k=4096, n=4096, dtype=BF16, bias=False),
        # a ragged prompt through a layer whose sizes fit no tile and no block
        dict(name="linear 1037x1000x777", kind="linear", rows=1037, k=1000, n=777, dtype=F16, bias=True),
        # a training step of the 4096-wide layer
        dict(name="step 8192x4096x4096", kind="step", rows=8192, k=4096, n=4096, dtype=BF16, bias=False),
        # the character model's MLP: many tokens, narrow layer
        dict(name="step 16384x384x1536", kind="step", rows=16384, k=384, n=1536, dtype=BF16, bias=True),
        # a small odd layer with fp32 activations
        dict(name="step 1111x520x1000", kind="step", rows=1111, k=520, n=1000, dtype=F32, bias=True),
        # the norm in front of a projection, for a decode batch
        dict(name="norm 7x4096", kind="norm", rows=7, k=4096, dtype=BF16, residual=True),
        # the norm of a full batch
        dict(name="norm 8192x4096", kind="norm", rows=8192, k=4096, dtype=BF16, residual=True),
        # the ViT's tokens in fp32, no residual, trained
        dict(name="norm_step 33280x512", kind="norm_step", rows=33280, k=512, dtype=F32, residual=False),
        # the GPT-2-medium residual stream, trained
        dict(name="norm_step 8192x1024", kind="norm_step", rows=8192, k=1024, dtype=BF16, residual=True),
        # residual, norm and MLP projection of a GPT-2-medium block, trained
        dict(name="block 8192x1024x4096", kind="block", rows=8192, k=1024, n=4096, dtype=BF16, bias=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "step", "step", "norm", "norm_step", "block"])
    dtype = rng.choice([BF16, BF16, F16, F32])
    rows = _spread(rng, 1 if kind in ("linear", "norm") else 16, 16384)
    k = _spread(rng, 64, 4096)
    if rng.random() < 0.5:      # half of the widths are what models use, the others anything
        k = max(64, k // 128 * 128)
    case = dict(kind=kind, rows=rows, k=k, dtype=dtype)
    if kind in ("linear", "step", "block"):
        n = _spread(rng, 64, 4096)
        if rng.random() < 0.5:
            n = max(64, n // 128 * 128)
        case["n"] = n
        case["bias"] = rng.random() < 0.5
        case["rows"] = max(1, min(rows, (8192 * 4096 * 4096) // (k * n)))
    else:
        case["residual"] = rng.random() < 0.7
    return case


def _dt(name):
    return getattr(torch, name)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _activations(g, rows, k, dtype):
    """Tokens of differing size with a few channels that stand out, as behind trained layers."""
    x = torch.randn(rows, k, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g))
    loud = torch.rand(k, device="cuda", generator=g) < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(dtype)


def _leaf(t):
    return t.requires_grad_(True)


def prepare(case, seed):
    g, kind, rows, k = _gen(seed), case["kind"], case["rows"], case["k"]
    dt = _dt(case["dtype"])
    s = {"kind": kind, "x": _activations(g, rows, k, dt)}
    # the block's layer keeps its parameters in bf16, the others fp32 masters
    pdt = torch.bfloat16 if kind == "block" else torch.float32
    if "n" in case:
        n = case["n"]
        s["w"] = (torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k)).to(pdt)
        s["b"] = (0.1 * torch.randn(n, device="cuda", generator=g)).to(pdt) if case["bias"] else None
    if kind in ("norm", "norm_step", "block"):
        s["gamma"] = (1.0 + 0.2 * torch.randn(k, device="cuda", generator=g)).to(pdt)
        res = kind == "block" or case["residual"]
        s["res"] = _activations(g, rows, k, dt) if res else None
    if kind in ("step", "block"):
        s["dy"] = (torch.randn(rows, case["n"], device="cuda", generator=g) * 0.01).to(dt)
    if kind == "norm_step":
        s["dy"] = (torch.randn(rows, k, device="cuda", generator=g) * 0.01).to(dt)
    if kind in ("norm_step", "block") and s["res"] is not None:
        s["dr"] = (torch.randn(rows, k, device="cuda", generator=g) * 0.01).to(dt)
    if own:
        _handles(case, s)
    return s


def _package():
    root = os.path.join(os.getcwd(), "adaptive-precision-ascension_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import apa
    return apa


def _handles(case, s):
    """What a user's program keeps: the package's modules and the cast weight."""
    apa = _package()
    s["apa"] = apa
    kind = case["kind"]
    if kind == "linear":
        s["wq"] = apa.block_cast(s["w"], square=True)
    if kind in ("step", "block"):
        lin = apa.APABlockLinear(case["k"], case["n"], bias=case["bias"], dtype=s["w"].dtype)
        with torch.no_grad():
            lin.weight_master.copy_(s["w"])
            if case["bias"]:
                lin.bias_master.copy_(s["b"])
        s["lin"] = lin
    if kind in ("norm_step", "block"):
        norm = apa.APARMSNorm(case["k"], eps=EPS, dtype=s["gamma"].dtype)
        with torch.no_grad():
            norm.weight.copy_(s["gamma"])
        s["norm"] = norm
    if kind in ("step", "norm_step", "block"):
        _leaf(s["x"])
        if s.get("res") is not None:
            _leaf(s["res"])


def run(s):
    return _own_run(s) if own else _plain_run(s)


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------
def _own_run(s):
    apa, kind = s["apa"], s["kind"]
    if kind == "linear":
        return {"y": apa.block_linear(s["x"], s["wq"], s["b"])}
    if kind == "norm":
        if s["res"] is None:
            q = apa.rms_norm(s["x"], s["gamma"], eps=EPS, quantize=True)
            return {"y": q.dequantize(torch.bfloat16)}
        q, r = apa.rms_norm(s["x"], s["gamma"], residual=s["res"], eps=EPS, quantize=True)
        return {"y": q.dequantize(torch.bfloat16), "r": r}
    if kind == "step":
        lin = s["lin"]
        y = lin(s["x"])
        leaves = [s["x"], lin.weight_master] + ([lin.bias_master] if s["b"] is not None else [])
        grads = torch.autograd.grad(y, leaves, s["dy"])
        return dict(zip(("y", "dx", "dw", "db"), (y,) + grads))
    if kind == "norm_step":
        norm = s["norm"]
        if s["res"] is None:
            y = norm(s["x"])
            grads = torch.autograd.grad(y, [s["x"], norm.weight], s["dy"])
            return dict(zip(("y", "dx", "dgamma"), (y,) + grads))
        y, r = norm(s["x"], s["res"])
        grads = torch.autograd.grad([y, r], [s["x"], norm.weight], [s["dy"], s["dr"]])
        return dict(zip(("y", "r", "dx", "dgamma"), (y, r) + grads))
    lin, norm = s["lin"], s["norm"]
    y, r = lin(s["x"], norm=norm, residual=s["res"])
    leaves = [s["x"], norm.weight, lin.weight_master] + ([lin.bias_master] if s["b"] is not None else [])
    grads = torch.autograd.grad([y, r], leaves, [s["dy"], s["dr"]])
    return dict(zip(("y", "r", "dx", "dgamma", "dw", "db"), (y, r) + grads))


# ---------------------------------------------------------------------------
# the plain forms, in fp32
# ---------------------------------------------------------------------------
def _plain_scale(amax):
    """The smallest power of two s with amax <= 448 s (1 for an empty block)."""
    m, e = torch.frexp(amax)
    p = e - 9 + (m > 0.875).to(e.dtype)
    p = torch.where(amax == 0, torch.zeros_like(p), p.clamp(min=-126))
    return torch.ldexp(torch.ones_like(amax), p)


def _plain_cast(x, square=False):
    """x [R, C] rounded to E4M3 under a scale per row and 128 columns (square: per 128 x 128), as fp32."""
    r, c = x.shape
    rb, cb = (-r % 128 if square else 0), -c % 128
    v = torch.zeros(r + rb, c + cb, device=x.device)
    v[:r, :c] = x
    v = v.view(-1, 128 if square else 1, v.shape[1] // 128, 128)
    sc = _plain_scale(v.abs().amax(dim=(1, 3), keepdim=True))
    q = (v / sc).to(torch.float8_e4m3fn).float() * sc
    return q.reshape(r + rb, c + cb)[:r, :c]


def _plain_norm(s):
    x = s["x"].detach()
    dt = x.dtype
    r = x if s.get("res") is None else (x.float() + s["res"].detach().float()).to(dt)
    rf = r.float()
    rstd = torch.rsqrt(rf.square().mean(dim=1, keepdim=True) + EPS)
    return r, rf, rstd, rf * rstd * s["gamma"].float()


def _plain_norm_backward(s, rf, rstd, dh, extra):
    xhat = rf * rstd
    gd = dh * s["gamma"].float()
    dx = rstd * (gd - xhat * (gd * xhat).mean(dim=1, keepdim=True))
    if extra is not None:
        dx = dx + extra.float()
    return dx, (dh * xhat).sum(dim=0)


def _plain_run(s):
    kind, dt = s["kind"], s["x"].dtype
    if kind == "linear":
        y = _plain_cast(s["x"].float()) @ _plain_cast(s["w"].float(), square=True).t()
        if s["b"] is not None:
            y = y + s["b"]
        return {"y": y.to(dt)}
    if kind == "norm":
        r, _, _, y = _plain_norm(s)
        out = {"y": _plain_cast(y).to(torch.bfloat16)}
        if s["res"] is not None:
            out["r"] = r
        return out
    if kind == "norm_step":
        r, rf, rstd, y = _plain_norm(s)
        dx, dg = _plain_norm_backward(s, rf, rstd, s["dy"].float(), s.get("dr"))
        out = {"y": y.to(dt), "dx": dx.to(dt), "dgamma": dg.to(s["gamma"].dtype)}
        if s["res"] is not None:
            out["r"] = r
        return out
    if kind == "step":
        x = s["x"].float()
    else:
        r, rf, rstd, x = _plain_norm(s)
    dy = s["dy"].float()
    wq = _plain_cast(s["w"].float(), square=True)
    y = _plain_cast(x) @ wq.t()
    if s["b"] is not None:
        y = y + s["b"].float()
    dh = _plain_cast(dy) @ wq
    dw = _plain_cast(dy.t()) @ _plain_cast(x.t()).t()
    out = {"y": y.to(dt), "dw": dw.to(s["w"].dtype)}
    if s["b"] is not None:
        out["db"] = dy.sum(dim=0).to(s["b"].dtype)
    if kind == "step":
        out["dx"] = dh.to(dt)
    else:
        dx, dg = _plain_norm_backward(s, rf, rstd, dh, s["dr"])
        out.update(r=r, dx=dx.to(dt), dgamma=dg.to(s["gamma"].dtype))
    return out


# ---------------------------------------------------------------------------
# the definitions, in fp64
# ---------------------------------------------------------------------------
def _blocks_exact(x, block_rows):
    """fp64 values of x on the E4M3 grid under the scales of its blocks."""
    rows, cols = x.shape
    nr, nc = math.ceil(rows / block_rows), math.ceil(cols / 128)
    pad = torch.nn.functional.pad(x, (0, nc * 128 - cols, 0, nr * block_rows - rows))
    tiles = pad.unflatten(0, (nr, block_rows)).unflatten(2, (nc, 128))
    top = tiles.abs().amax(dim=3).amax(dim=1)
    tiny = 2.0 ** -126
    p = torch.ceil(torch.log2((top / 448.0).clamp(min=tiny)))
    p = torch.where(top > 448.0 * torch.exp2(p), p + 1, p)           # log2's own rounding
    p = torch.where((top <= 448.0 * torch.exp2(p - 1)) & (p > -126), p - 1, p)
    scale = torch.where(top == 0, torch.ones_like(top), torch.exp2(p))[:, None, :, None]
    v = tiles / scale
    mag = v.abs().clamp(min=2.0 ** -9)
    lead = torch.floor(torch.log2(mag))
    lead = torch.where(torch.exp2(lead) > mag, lead - 1, lead)
    lead = torch.where(torch.exp2(lead + 1) <= mag, lead + 1, lead)
    quantum = torch.exp2(lead.clamp(min=-6.0) - 3.0)
    v = torch.round(v / quantum) * quantum
    return (v * scale).flatten(2, 3).flatten(0, 1)[:rows, :cols]


def exact(case, seed):
    s = prepare_inputs_only(case, seed)
    kind = case["kind"]
    d = {n: (t.detach().double() if torch.is_tensor(t) else t) for n, t in s.items()}
    if kind in ("norm", "norm_step", "block"):
        stream = d["x"]
        if d.get("res") is not None:
            stream = (stream + d["res"]).to(s["x"].dtype).double()
        inv = 1.0 / torch.sqrt((stream * stream).sum(dim=1, keepdim=True) / case["k"] + EPS)
        hat = stream * inv
        h = hat * d["gamma"]
    else:
        h = d["x"]
    out = {}
    if kind in ("norm", "norm_step", "block") and d.get("res") is not None:
        out["r"] = stream
    if kind == "norm":
        out["y"] = _blocks_exact(h, 1)
        return out
    if kind == "norm_step":
        out["y"] = h
        dh = d["dy"]
    else:
        wq = _blocks_exact(d["w"], 128)
        out["y"] = torch.einsum("mk,nk->mn", _blocks_exact(h, 1), wq)
        if d["b"] is not None:
            out["y"] = out["y"] + d["b"]
        if kind == "linear":
            return out
        dh = torch.einsum("mn,nk->mk", _blocks_exact(d["dy"], 1), wq)
        out["dw"] = torch.einsum("nm,km->nk", _blocks_exact(d["dy"].t().contiguous(), 1),
                                 _blocks_exact(h.t().contiguous(), 1))
        if d["b"] is not None:
            out["db"] = d["dy"].sum(dim=0)
    if kind == "step":
        out["dx"] = dh
        return out
    out["dgamma"] = torch.einsum("mk,mk->k", dh, hat)
    g = dh * d["gamma"]
    out["dx"] = inv * g - hat * inv * (torch.einsum("mk,mk->m", g, hat) / case["k"])[:, None]
    if d.get("dr") is not None:
        out["dx"] = out["dx"] + d["dr"]
    return out


def prepare_inputs_only(case, seed):
    """The inputs of prepare() without the package's handles."""
    global own
    kept, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = kept


def work(case):
    m, k = case["rows"], case["k"]
    es = 4 if case["dtype"] == F32 else 2
    kind = case["kind"]
    if kind == "norm":
        # x (and the residual) in; the normalised values (and the stream) out
        return {"bytes": m * k * (es + 2 + (2 * es if case["residual"] else 0)) + 4 * k, "flops": 6 * m * k}
    if kind == "norm_step":
        # x, dy in; y, dx out; with a residual also res, dr in and the stream out
        return {"bytes": m * k * es * (7 if case["residual"] else 4) + 8 * k, "flops": 16 * m * k}
    n = case["n"]
    bias = n * (4 if kind != "block" else 2) if case["bias"] else 0
    if kind == "linear":
        # x and the E4M3 weight with its scales in, y out
        return {"bytes": (m * k + m * n) * es + n * k + math.ceil(n / 128) * math.ceil(k / 128) + bias,
                "flops": 2 * m * n * k}
    ws = 4 if kind == "step" else 2
    moved = es * (2 * m * k + 2 * m * n) + ws * 2 * n * k + 2 * bias
    if kind == "block":
        moved += es * 3 * m * k + 4 * k      # the residual and its gradient in, the stream out, gamma and its gradient
    return {"bytes": moved, "flops": 6 * m * n * k}
