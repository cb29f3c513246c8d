"""The block layer's backward for every choice of what wants a gradient, and on
strided inputs: each gradient equals the one of the pass that wants all, bit for
bit."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from apa import APABlockLinear, APAConfig, APARMSNorm

M, K, N = 270, 328, 200


def rnd(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def parts(dtype, norm, residual):
    cfg = APAConfig(device="cuda")
    torch.manual_seed(0)
    lin = APABlockLinear(K, N, config=cfg)
    n = APARMSNorm(K, config=cfg) if norm else None
    leaves = {"x": rnd((M, K), 1, dtype), "w": lin.weight_master, "b": lin.bias_master}
    if norm:
        with torch.no_grad():
            n.weight.copy_(1 + 0.1 * rnd((K,), 3))
        leaves["g"] = n.weight
    if residual:
        leaves["res"] = rnd((M, K), 2, dtype)

    def run(wanted):
        for name, t in leaves.items():
            t.requires_grad_(name in wanted)
        out = lin(leaves["x"], norm=n, residual=leaves.get("res"))
        outs = list(out) if residual else [out]
        seeds = [rnd((M, N), 4, dtype), rnd((M, K), 5, dtype)]
        use = [(o, s) for o, s in zip(outs, seeds) if o.requires_grad]
        grads = torch.autograd.grad([o for o, _ in use], [leaves[w] for w in wanted], [s for _, s in use],
                                    allow_unused=True)
        return dict(zip(wanted, grads)), [o.detach() for o in outs]

    return run, list(leaves)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm,residual", [(False, False), (True, False), (True, True)])
def test_every_subset(dtype, norm, residual):
    run, names = parts(dtype, norm, residual)
    full, outs = run(names)
    # the weight gradient alone is another launch than with the input's; its sum
    # over three slabs of tokens is in one piece in both
    for size in range(1, len(names)):
        for wanted in itertools.combinations(names, size):
            got, again = run(list(wanted))
            assert all(torch.equal(a, b) for a, b in zip(outs, again)), wanted
            for name in wanted:
                assert got[name] is not None and torch.equal(got[name], full[name]), (wanted, name)


@pytest.mark.parametrize("norm", [False, True])
def test_strided_inputs(norm):
    """Views of wider, transposed and repeated storage, and their gradients' layouts."""
    cfg = APAConfig(device="cuda")
    lin, n = APABlockLinear(K, N, config=cfg), APARMSNorm(K, config=cfg) if norm else None
    wide, tall, row = rnd((M, K + 7), 1), rnd((K, M), 2), rnd((1, K), 3)
    dy = rnd((N, M), 4).t()
    for view in (wide[:, 3:3 + K], wide[::2, :K], tall.t(), row.expand(M, K),
                 wide[:, :K].reshape(2, M // 2, K).transpose(0, 1)):
        out = []
        for x in (view, view.clone(memory_format=torch.contiguous_format)):
            x = x.detach().requires_grad_(True)
            y = lin(x, norm=n)
            g = dy[:y.numel() // N].unflatten(0, y.shape[:-1])         # a view, columns apart
            out.append((y.detach(),) + torch.autograd.grad(y, [x, lin.weight_master], g))
        assert all(torch.equal(s, t) for s, t in zip(*out))


def test_one_dimension():
    cfg = APAConfig(device="cuda")
    lin, n = APABlockLinear(K, N, config=cfg), APARMSNorm(K, config=cfg)
    x, r = rnd((K,), 1).requires_grad_(True), rnd((K,), 2).requires_grad_(True)
    y, s = lin(x, norm=n, residual=r)
    y2, s2 = lin(x[None], norm=n, residual=r[None])
    assert y.shape == (N,) and s.shape == (K,) and torch.equal(y[None], y2) and torch.equal(s[None], s2)
    dy, ds = rnd((N,), 3), rnd((K,), 4)
    got = torch.autograd.grad([y, s], [x, r, n.weight, lin.weight_master], [dy, ds])
    want = torch.autograd.grad([y2, s2], [x, r, n.weight, lin.weight_master], [dy[None], ds[None]])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        z, s3 = lin(x, norm=n, residual=r)
        assert torch.equal(z, y) and torch.equal(s3, s) and torch.equal(lin(x), lin(x[None])[0])
