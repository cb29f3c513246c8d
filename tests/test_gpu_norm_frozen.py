"""The norm with parts that want no gradient."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from apa import APABlockLinear, APAConfig, APARMSNorm


def rnd(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("fused", [False, True])
def test_frozen_weight(fused):
    """No gradient for the weight, the others as before."""
    cfg = APAConfig(device="cuda")
    norm, lin = APARMSNorm(256, config=cfg), APABlockLinear(256, 72, config=cfg)
    x, res, dr = rnd((20, 256), 1).requires_grad_(True), rnd((20, 256), 2).requires_grad_(True), rnd((20, 256), 3)
    dy = rnd((20, 72 if fused else 256), 4)

    def run():
        for t in (x, res, norm.weight, lin.weight_master, lin.bias_master):
            t.grad = None
        y, r = lin(x, norm=norm, residual=res) if fused else norm(x, res)
        torch.autograd.backward([y, r], [dy, dr])
        return x.grad, res.grad, lin.weight_master.grad

    want = run()
    assert norm.weight.grad is not None
    norm.weight.requires_grad_(False)
    got = run()
    assert norm.weight.grad is None
    assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(got, want))
    norm.weight.requires_grad_(True)
    x.requires_grad_(False)
    got = run()
    assert x.grad is None and torch.equal(got[1], want[1]) and norm.weight.grad is not None


@pytest.mark.parametrize("fused", [False, True])
def test_only_the_weight_wants_a_gradient(fused):
    cfg = APAConfig(device="cuda")
    norm, lin = APARMSNorm(256, config=cfg), APABlockLinear(256, 72, config=cfg)
    x, dy = rnd((20, 256), 1), rnd((20, 72 if fused else 256), 4)
    for p in lin.parameters():
        p.requires_grad_(False)

    def run():
        norm.weight.grad = None
        (lin(x, norm=norm) if fused else norm(x)).backward(dy)
        return norm.weight.grad

    alone = run()
    x.requires_grad_(True)
    assert torch.equal(run(), alone)
