"""What the block layer and the norm keep for their backward goes through
autograd's saved tensors: freed with the graph, seen by hooks, recomputed by
checkpointing."""
import gc

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from apa import APABlockLinear, APAConfig, APARMSNorm


def rnd(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


M, K, N = 150, 264, 200
KINDS = ["linear", "norm", "norm+res", "fused", "fused+res"]


def make(kind):
    """(function of the leaves, leaves)"""
    cfg = APAConfig(device="cuda")
    torch.manual_seed(0)
    lin, norm = APABlockLinear(K, N, config=cfg), APARMSNorm(K, config=cfg)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.1 * rnd((K,), 3))
    x, r = (rnd((M, K), s, torch.bfloat16).cuda().requires_grad_(True) for s in (1, 2))

    def both(out):
        return out[0].float().sum() + (out[1].float() ** 2).sum()

    call = {"linear": lambda: (lin(x).float() ** 2).sum(),
            "norm": lambda: (norm(x).float() ** 2).sum(),
            "norm+res": lambda: both(norm(x, r)),
            "fused": lambda: (lin(x, norm=norm).float() ** 2).sum(),
            "fused+res": lambda: both(lin(x, norm=norm, residual=r))}[kind]
    leaves = [x] + ([r] if "res" in kind else [])
    leaves += ([norm.weight] if kind != "linear" else []) + ([] if kind.startswith("norm") else list(lin.parameters()))
    return call, leaves


@pytest.mark.parametrize("kind", KINDS)
def test_hooks_see_what_the_backward_reads(kind):
    call, leaves = make(kind)
    want = torch.autograd.grad(call(), leaves)
    seen = []

    def pack(t):
        seen.append(t)
        return t.cpu()

    with saved_tensors_hooks(pack, lambda t: t.cuda()):
        loss = call()
    if not kind.startswith("norm"):
        # the transposed cast of the weight, and without a norm that of x
        packed = N * K + (0 if kind.startswith("fused") else M * K)
        assert any(t.dtype == torch.uint8 and t.numel() >= packed for t in seen)
    if kind != "linear":
        assert any(t.shape == (M,) and t.dtype == torch.float32 for t in seen)      # the rows' statistics
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, leaves), want))
    with save_on_cpu():
        loss = call()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, leaves), want))


@pytest.mark.parametrize("kind", KINDS)
def test_checkpointing(kind):
    call, leaves = make(kind)
    want = torch.autograd.grad(call(), leaves)
    loss = checkpoint(call, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, leaves), want))


@pytest.mark.parametrize("kind", KINDS)
def test_a_second_backward_needs_the_graph_kept(kind):
    call, leaves = make(kind)
    loss = call()
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, leaves)


@pytest.mark.parametrize("norm", [False, True])
def test_second_backward_of_the_layer_alone(norm):
    """No other operation's saved tensors stand between the caller and the layer's."""
    cfg = APAConfig(device="cuda")
    lin = APABlockLinear(K, N, config=cfg)
    y = lin(rnd((M, K), 1).cuda(), norm=APARMSNorm(K, config=cfg) if norm else None)
    dy = torch.ones_like(y)
    torch.autograd.grad(y, [lin.weight_master], dy)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, [lin.weight_master], dy)


def test_backward_frees_its_operands():
    cfg = APAConfig(device="cuda")
    m = k = n = 1024
    lin = APABlockLinear(k, n, bias=False, config=cfg)
    x = rnd((m, k), 1, torch.bfloat16).cuda()
    lin(x).sum().backward()
    lin.weight_master.grad = None
    gc.collect()
    torch.cuda.synchronize()
    y = lin(x)
    held = torch.cuda.memory_allocated()
    (dw,) = torch.autograd.grad(y, [lin.weight_master], torch.ones_like(y))
    # dw came (4 n k bytes); the transposed cast of x (m k bytes) went, though y still holds the graph
    assert torch.cuda.memory_allocated() <= held + 4 * n * k - m * k
    assert y.grad_fn is not None and dw.shape == (n, k)
