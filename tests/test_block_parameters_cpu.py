"""Where the block layer and the norm take their parameters from, without a GPU:
the operators themselves are stand-ins."""
import pytest
import torch
from torch.nn.utils import parametrize, prune

from apa import APABlockLinear, APAConfig, APARMSNorm, _lib, blockscale

CPU = APAConfig(device="cpu")


class Doubled(torch.nn.Module):
    def forward(self, w):
        return 2 * w


@pytest.fixture(autouse=True)
def stand_ins(monkeypatch):
    def linear(x, residual, gamma, W, b, eps):
        return (x * gamma if gamma is not None else x) @ W.t() + (0 if b is None else b)

    monkeypatch.setattr(_lib, "require_cuda", lambda t, what: None)
    monkeypatch.setattr(blockscale._BlockLinearFn, "apply", staticmethod(linear))
    monkeypatch.setattr(blockscale._RMSNormFn, "apply", staticmethod(lambda x, w, r, eps: x * w))


def test_parametrized_and_pruned():
    x = torch.randn(3, 8)
    lin, norm = APABlockLinear(8, 4, config=CPU), APARMSNorm(8, config=CPU)
    want = 2 * x @ lin.weight_master.t() + lin.bias_master
    assert torch.equal(lin(2 * x), want)
    parametrize.register_parametrization(norm, "weight", Doubled())
    assert torch.equal(norm(x), 2 * x) and torch.equal(lin(x, norm=norm), want)
    parametrize.register_parametrization(lin, "weight_master", Doubled())
    assert torch.allclose(lin(x), want)
    lin = APABlockLinear(8, 4, config=CPU)
    prune.l1_unstructured(lin, "weight_master", 0.5)
    assert int((lin.weight_master == 0).sum()) == 16
    assert torch.equal(lin(x), x @ lin.weight_master.t() + lin.bias_master)


def test_replicas():
    """As DataParallel makes them: plain tensors in the parameters' place."""
    lin = APABlockLinear(8, 4, config=CPU)
    other = lin._replicate_for_data_parallel()
    other.weight_master, other.bias_master = 2 * lin.weight_master, 2 * lin.bias_master
    x = torch.randn(3, 8)
    assert torch.equal(other(x), x @ other.weight_master.t() + other.bias_master)


def test_functional_call():
    lin = APABlockLinear(8, 4, bias=False, config=CPU)
    x, w = torch.randn(3, 8), torch.randn(4, 8)
    assert torch.allclose(torch.func.functional_call(lin, {"weight_master": w}, (x.requires_grad_(True),)), x @ w.t())
