"""Calls of the block-scaled operators that are refused, without a GPU."""
import pytest
import torch

from apa import APABlockTensor, _lib, block_linear, block_matmul


def block(rows, cols):
    q = torch.randn(rows, cols).to(torch.float8_e4m3fn)
    return APABlockTensor.from_parts(q, torch.zeros(rows, (cols + 127) // 128, dtype=torch.int32))


def test_a_bias_that_wants_a_gradient(monkeypatch):
    """Its gradient would be lost: these operators have none."""
    monkeypatch.setattr(_lib, "require_cuda", lambda t, what: None)
    w, x = block(8, 64), torch.randn(3, 64)
    bias = torch.nn.Parameter(torch.zeros(8))
    for call in (lambda: block_linear(x, w, bias), lambda: block_linear(block(3, 64), w, bias),
                 lambda: block_matmul(block(3, 64), w, bias), lambda: block_linear(x.requires_grad_(True), w)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
