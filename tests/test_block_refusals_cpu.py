"""Calls of the block-scaled operators that are refused, without a GPU."""
import pytest
import torch

from apa import (APABlockLinear, APABlockTensor, APAConfig, APARMSNorm, _lib, block_cast, block_linear, block_matmul,
                 blockscale, rms_norm)


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


def test_out_is_written_in_place(monkeypatch):
    """As torch's own out=: refused where it wants a gradient, and counted as a
    change, so that a backward which would read its old values is refused."""
    monkeypatch.setattr(_lib, "require_cuda", lambda t, what: None)
    monkeypatch.setattr(blockscale, "_matmul", lambda a, b, bias, out, accumulate: None)
    a, w = block(3, 64), block(8, 64)
    leaf = torch.zeros(3, 8, requires_grad=True)
    for out in (leaf, leaf * 1.0):
        with pytest.raises(RuntimeError, match="no gradient"):
            block_matmul(a, w, out=out)
    with torch.no_grad():
        assert block_matmul(a, w, out=leaf) is leaf
    s = torch.ones(3, 8)
    loss = (leaf * s).sum()
    block_matmul(a, w, out=s, accumulate=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        block_matmul(a, w, out=torch.ones(3, 8))


def test_buffers_too_small_for_their_shape():
    """A product reads what the shape says, so the shape has to fit."""
    t = block(5, 200)
    again = APABlockTensor(t.buffer, 5, 200)
    assert torch.equal(again.exponents(), t.exponents())
    longer = APABlockTensor(torch.cat([t.buffer, torch.zeros(64, dtype=torch.uint8)]), 5, 200)
    assert torch.equal(longer.exponents(), t.exponents())
    for args in ((t.buffer, 6, 200), (t.buffer, 5, 209), (t.buffer[:-1], 5, 200), (t.buffer, -1, 200), (t.buffer, 5, 0),
                 (longer.buffer[8:], 5, 200), (torch.zeros(2 * t.buffer.numel(), dtype=torch.uint8)[::2], 5, 200)):
        with pytest.raises(ValueError):
            APABlockTensor(*args)
    for bad in (t.buffer.view(1, -1), t.buffer.float(), t.buffer.numpy()):
        with pytest.raises(TypeError):
            APABlockTensor(bad, 5, 200)


def test_arguments_that_are_no_tensors(monkeypatch):
    monkeypatch.setattr(_lib, "require_cuda", lambda t, what: None)
    cpu = APAConfig(device="cpu")
    x, g, w = torch.randn(3, 64), torch.ones(64), block(8, 64)
    lin, norm = APABlockLinear(64, 8, config=cpu), APARMSNorm(64, config=cpu)
    for call in (lambda: block_linear(x, w, [0.0] * 8), lambda: block_matmul(block(3, 64), w, 1.0),
                 lambda: rms_norm(x, [1.0] * 64, quantize=True), lambda: rms_norm(x, 1.0),
                 lambda: rms_norm(x, g, 2.0), lambda: rms_norm(x, g, 2.0, quantize=True),
                 lambda: rms_norm([1.0], g, quantize=True), lambda: lin(x, norm=norm, residual=1.0)):
        with pytest.raises(TypeError, match="expected a tensor"):
            call()


@pytest.mark.parametrize("shape", [(0,), (3, 0), (2, 3, 0), (0, 4, 0)])
def test_no_columns(shape):
    for call in (lambda x: block_cast(x), lambda x: rms_norm(x, torch.ones(0))):
        with pytest.raises(ValueError, match="has no columns"):
            call(torch.empty(shape))
