"""APABlockLinear: forward, gradients, the norm in front, and its place beside APALinear."""
import numpy as np
import pytest
import torch
import torch.nn as nn

import blockscale_plain as P

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import apa
    from apa import APABlockLinear, APAConfig, APALinear, APAManager, APARMSNorm, block_cast, block_matmul, rms_norm
    from apa import blockscale

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def f64(t):
    return t.detach().cpu().double().numpy()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def whole(shape, seed, top=8):
    """Whole numbers of at most four bits: exact in E4M3 under any scale."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g).float()


def rnd(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def layer(w, b=None, dtype=torch.float32):
    lin = APABlockLinear(w.shape[1], w.shape[0], bias=b is not None, dtype=dtype, config=APAConfig(device="cuda"))
    with torch.no_grad():
        lin.weight_master.copy_(w)
        if b is not None:
            lin.bias_master.copy_(b)
    return lin


@pytest.mark.parametrize("m,k,n", [(1, 128, 64), (5, 33, 17), (130, 260, 300), (300, 1000, 72), (1024, 384, 1536)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_exact_layer(m, k, n, dtype):
    """Operands of few bits: every product and partial sum is exact, so only the output's rounding is left."""
    x, w, b, dy = whole((m, k), 1), whole((n, k), 2), whole((n,), 3), whole((m, n), 4, 2)
    lin = layer(w, b)
    xd = x.to(dtype).cuda().requires_grad_(True)
    y = lin(xd)
    y.backward(dy.to(dtype).cuda())
    assert y.dtype == dtype and xd.grad.dtype == dtype
    want = (f64(x) @ f64(w).T + f64(b))
    assert torch.equal(y.detach().cpu(), torch.from_numpy(want).to(dtype))
    assert torch.equal(xd.grad.cpu(), torch.from_numpy(f64(dy) @ f64(w)).to(dtype))
    assert np.array_equal(f64(lin.weight_master.grad), f64(dy).T @ f64(x))
    assert np.array_equal(f64(lin.bias_master.grad), f64(dy).sum(0))


@pytest.mark.parametrize("limit", [2, 4, 10])
@pytest.mark.parametrize("m,k,n,dtype", [(700, 600, 300, torch.bfloat16), (2600, 300, 520, torch.float32),
                                         (260, 530, 2050, torch.float16), (9000, 136, 264, torch.bfloat16)])
def test_exact_gradients_in_rounds(m, k, n, dtype, limit):
    """Both gradients' tiles share one launch: on few CTA pairs they take
    several rounds, with the longer product's last round left incomplete, and
    the longer one is split where its tiles outlast an even share. The bias
    gradient's sums come from the same launch or, past few slabs, their own."""
    x, w, dy = whole((m, k), 1, 4), whole((n, k), 2, 4), whole((m, n), 3, 2)
    lin = layer(w, whole((n,), 4))
    runs = []
    for sms in (0, limit):             # workspaces are sized without the limit, as when another part sets it
        xd = x.to(dtype).cuda().requires_grad_(True)
        lin.weight_master.grad = lin.bias_master.grad = None
        blockscale._lib.check(blockscale._lib.lib().apa_set_gemm_sm_limit(sms), "limit")
        try:
            y = lin(xd)
            y.backward(dy.to(dtype).cuda())
        finally:
            blockscale._lib.check(blockscale._lib.lib().apa_set_gemm_sm_limit(0), "limit")
        runs.append((y.detach(), xd.grad, lin.weight_master.grad, lin.bias_master.grad))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert torch.equal(xd.grad.cpu(), torch.from_numpy(f64(dy) @ f64(w)).to(dtype))
    assert np.array_equal(f64(lin.weight_master.grad), f64(dy).T @ f64(x))
    assert np.array_equal(f64(lin.bias_master.grad), f64(dy).sum(0))


def test_gradients_against_differences():
    """On such operands the layer is exactly linear, so differences are exact too."""
    m, k, n = 40, 200, 70
    x, w, dw, dx, dy = whole((m, k), 1, 4), whole((n, k), 2, 4), whole((n, k), 3, 4), whole((m, k), 4, 4), whole((m, n), 5)
    lin = layer(w)
    xd = x.cuda().requires_grad_(True)
    lin(xd).backward(dy.cuda())
    with torch.no_grad():
        y0 = f64(lin(x.cuda()))
        lin.weight_master.add_(dw.cuda())
        y1 = f64(lin(x.cuda()))
        lin.weight_master.sub_(dw.cuda())
        y2 = f64(lin((x + dx).cuda()))
    assert (f64(dy) * (y1 - y0)).sum() == (f64(lin.weight_master.grad) * f64(dw)).sum()
    assert (f64(dy) * (y2 - y0)).sum() == (f64(xd.grad) * f64(dx)).sum()


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,n,dtype", [(64, 130, 200, torch.bfloat16), (700, 520, 260, torch.bfloat16),
                                         (333, 1000, 96, torch.float32), (2100, 96, 140, torch.float16)])
def test_layer_is_its_casts_and_products(m, k, n, dtype, wdtype):
    """Real data: output and gradients equal the plain products of the plainly
    cast operands, up to the accumulation's and the output's rounding."""
    x, w, dy = rnd((m, k), 1, dtype), rnd((n, k), 2).to(wdtype), rnd((m, n), 3, dtype)
    b = rnd((n,), 4).to(wdtype)
    lin = layer(w, b, dtype=wdtype)
    xd = x.cuda().requires_grad_(True)
    y = lin(xd)
    y.backward(dy.cuda())
    xq, wq = P.cast(f64(x))[0], P.cast(f64(w), 128)[0]
    dq, dt, xt = P.cast(f64(dy))[0], P.cast(f64(dy).T)[0], P.cast(f64(x).T)[0]

    def near(got, want, mag, steps):
        tol = (12 + steps) * 2.0 ** -23 * mag + half_step(got.dtype) * (1 + 2.0 ** -9) * np.abs(want)
        assert np.all(np.abs(f64(got) - want) <= tol + 1e-7 * (got.dtype == torch.float16))

    near(y, xq @ wq.T + f64(b), np.abs(xq) @ np.abs(wq).T + np.abs(f64(b)), k / 32)
    near(xd.grad, dq @ wq, np.abs(dq) @ np.abs(wq), n / 32)
    assert lin.weight_master.grad.dtype == wdtype
    near(lin.weight_master.grad, dt @ xt.T, np.abs(dt) @ np.abs(xt).T, m / 32)
    near(lin.bias_master.grad, f64(dy).sum(0), np.abs(f64(dy)).sum(0), m / 32)


@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("lead,k,n,dtype", [((50,), 256, 130, torch.bfloat16), ((3, 70), 520, 96, torch.float32)])
def test_norm_in_front(lead, k, n, dtype, with_res):
    """The fused call is the norm's E4M3 output times the weight, and its
    gradients those of the parts, bit for bit."""
    cfg = APAConfig(device="cuda")
    lin, norm = layer(rnd((n, k), 1), rnd((n,), 2)), APARMSNorm(k, config=cfg)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.1 * rnd((k,), 3))
    x = rnd((*lead, k), 4, dtype).cuda().requires_grad_(True)
    res = rnd((*lead, k), 5, dtype).cuda().requires_grad_(True) if with_res else None
    dy, dr = rnd((*lead, n), 6, dtype).cuda(), rnd((*lead, k), 7, dtype).cuda()
    out = lin(x, norm=norm, residual=res)
    if with_res:
        y, r = out
        torch.autograd.backward([y, r], [dy, dr])
    else:
        y, r = out, x
        y.backward(dy)
    with torch.no_grad():
        plain = rms_norm(x, norm.weight, res, quantize=True)
        q = plain[0] if with_res else plain
        wq, wt = block_cast(lin.weight_master, "both", square=True)
        assert torch.equal(block_matmul(q, wq, lin.bias_master, out_dtype=dtype), y.reshape(-1, n))
        dq, dt = block_cast(dy, "both")
        dh = block_matmul(dq, wt, out_dtype=torch.float32)
        r2 = r.detach().reshape(-1, k)
        _, _, rstd = blockscale._norm_forward(r2, norm.weight, None, norm.eps, True, True)
        dx, dg = blockscale._norm_backward(dh, r2, rstd, norm.weight, dr.view(-1, k) if with_res else None)
        assert torch.equal(x.grad.view(-1, k), dx) and torch.equal(norm.weight.grad, dg)
        _, xt = blockscale._cast(r2, False, True, row_mul=rstd, col_mul=norm.weight)
        assert torch.equal(lin.weight_master.grad, block_matmul(dt, xt, out_dtype=torch.float32))
        if with_res:
            assert torch.equal(res.grad, x.grad)
        # without gradients the layer keeps its cast weight and gives the same
        again = lin(x, norm=norm, residual=res)
        assert torch.equal(again[0] if with_res else again, y)


def test_kept_weight_follows_the_parameter():
    lin = layer(rnd((40, 64), 1))
    x = rnd((3, 64), 2).cuda()
    with torch.no_grad():
        a = lin(x)
        kept = lin._wq.buffer.data_ptr()
        lin.weight_master.mul_(2.0)
        assert torch.equal(lin(x), 2 * a)
        lin.weight_master.data.mul_(2.0)
        lin.refresh_working_copy()
        assert torch.equal(lin(x), 4 * a) and lin._wq.buffer.data_ptr() == kept
    state = lin.state_dict()
    assert set(state) == {"weight_master"}
    other = APABlockLinear(64, 40, bias=False, config=APAConfig(device="cuda"))
    other.load_state_dict(state)
    with torch.no_grad():
        assert torch.equal(other(x), 4 * a)


def test_kept_weight_and_streams():
    """A first call on one stream keeps the weight for the next call on another."""
    x, w = rnd((5, 2048), 1).cuda(), rnd((2048, 2048), 2)
    want = layer(w)(x).detach()
    lin = layer(w)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for turn in range(3):
        outs = []
        with torch.no_grad():
            for s in streams:
                with torch.cuda.stream(s):
                    outs.append(lin(x))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want * 2 ** turn) for o in outs)
        with torch.no_grad():
            lin.weight_master.mul_(2.0)
        torch.cuda.synchronize()


def test_kept_weight_and_captures():
    """A capture that meets a changed weight casts it in the graph, and leaves
    the kept one to calls outside."""
    x, w = rnd((5, 256), 1).cuda(), rnd((192, 256), 2)
    want = layer(w)(x).detach()
    lin = layer(w)
    with torch.no_grad():
        block_cast(lin.weight_master, square=True), layer(w)(x)          # first launches before the capture
        torch.cuda.synchronize()
        fresh = torch.cuda.CUDAGraph()
        with torch.cuda.graph(fresh):
            with pytest.raises(RuntimeError, match="before the capture"):
                lin.refresh_working_copy()
            y = lin(x)
        assert lin._wq is None and torch.equal(lin(x), want)
        fresh.replay()
        assert torch.equal(y, want)
        kept = torch.cuda.CUDAGraph()
        with torch.cuda.graph(kept):
            z = lin(x)
        lin.weight_master.mul_(2.0)
        fresh.replay(), kept.replay()
        assert torch.equal(y, 2 * want) and torch.equal(z, want)         # z reads the kept cast
        assert torch.equal(lin(x), 2 * want)                             # renewed in place
        kept.replay()
        assert torch.equal(z, 2 * want)
        lin.weight_master.mul_(2.0)
        renew = torch.cuda.CUDAGraph()
        with torch.cuda.graph(renew):
            lin.refresh_working_copy()
        kept.replay()
        assert torch.equal(z, 2 * want)
        renew.replay(), kept.replay()
        assert torch.equal(z, 4 * want) and torch.equal(lin(x), 4 * want)


def test_kept_weight_made_in_inference_mode():
    """Kept under inference_mode, renewed outside it."""
    x, w = rnd((5, 256), 1).cuda(), rnd((192, 256), 2)
    lin = layer(w)
    with torch.inference_mode():
        a = lin(x)
    kept = lin._wq.buffer.data_ptr()
    with torch.no_grad():
        lin.weight_master.mul_(2.0)
        b = lin(x)
    assert torch.equal(b, 2 * a) and lin._wq.buffer.data_ptr() == kept
    y = lin(x.clone().requires_grad_(True))
    assert torch.equal(y.detach(), b)


def test_kept_weight_of_another_parameter():
    import copy
    lin = layer(rnd((40, 64), 1))
    x, w = rnd((3, 64), 2).cuda(), rnd((40, 64), 3).cuda()
    with torch.no_grad():
        lin(x)
        want = layer(w)(x)
        v = lin.weight_master._version
        fresh = w.clone()
        for _ in range(v - fresh._version):
            fresh.add_(0.0)
        lin.weight_master = nn.Parameter(fresh)            # as many changes as the one before it
        assert lin.weight_master._version == v and torch.equal(lin(x), want)
        other = copy.deepcopy(lin)
        other.weight_master.mul_(2.0)
        assert torch.equal(other(x), 2 * want) and torch.equal(lin(x), want)
        lin.weight_master.data = 4 * w
        assert torch.equal(lin(x), 4 * want)
        assert torch.equal(lin.to(torch.bfloat16)(x), layer((4 * w).bfloat16().float())(x))
    with torch.inference_mode():
        assert torch.equal(other(x), 2 * want)
        made = layer(w)
        assert torch.equal(made(x), want)


def test_empty_batch_and_frozen_parts():
    lin = layer(rnd((40, 64), 1), rnd((40,), 2))
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    y = lin(x)
    y.sum().backward()
    assert y.shape == (0, 40) and x.grad.shape == (0, 64)
    assert bool((lin.weight_master.grad == 0).all()) and bool((lin.bias_master.grad == 0).all())
    x = rnd((9, 64), 3).cuda()
    lin.zero_grad(set_to_none=True)
    lin(x).sum().backward()                      # no gradient of x wanted
    full = lin.weight_master.grad.clone()
    lin.zero_grad(set_to_none=True)
    lin.weight_master.requires_grad_(False)
    xg = x.clone().requires_grad_(True)
    lin(xg).sum().backward()
    assert lin.weight_master.grad is None and xg.grad is not None and lin.bias_master.grad is not None
    lin.weight_master.requires_grad_(True)
    lin.bias_master.requires_grad_(False)
    lin(x).sum().backward()
    assert torch.equal(lin.weight_master.grad, full)


def test_accumulates_over_passes_and_uses():
    lin = layer(whole((16, 32), 1))
    x, dy = whole((12, 32), 2).cuda(), whole((12, 16), 3).cuda()
    lin(x).backward(dy)
    one = lin.weight_master.grad.clone()
    lin(x).backward(dy)
    assert torch.equal(lin.weight_master.grad, 2 * one)
    lin.weight_master.grad = None
    (lin(x) + lin(x)).backward(dy)
    assert torch.equal(lin.weight_master.grad, 2 * one)


class Net(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.a = APALinear(48, 64, config=cfg)
        self.norm = APARMSNorm(64, config=cfg)
        self.up = APABlockLinear(64, 128, config=cfg)
        self.down = APABlockLinear(128, 64, config=cfg)
        self.out_norm = APARMSNorm(64, config=cfg)
        self.head = APALinear(64, 10, config=cfg)

    def forward(self, x):
        h = self.a(x).float()
        z = torch.nn.functional.gelu(self.up(h, norm=self.norm))
        y, _ = self.out_norm(self.down(z), h)
        return self.head(y)


def test_beside_apalinear_under_a_manager():
    torch.manual_seed(0)
    cfg = APAConfig(device="cuda", check_interval=1)
    net = Net(cfg)
    mgr = APAManager(net, cfg)
    params = mgr.get_trainable_parameters()
    assert len(params) == len(list(net.parameters()))
    opt = torch.optim.AdamW(params, lr=1e-3)
    x = torch.randn(32, 48, device="cuda")
    for bad in (False, True, False):
        mgr.pre_step()
        opt.zero_grad(set_to_none=True)
        y = net(x)
        dy = torch.full_like(y, 0.01)
        loss = (y.float() * 0.01).sum()
        if bad:
            hook = net.down.register_forward_hook(lambda m, i, o: o * torch.tensor(float("inf"), device="cuda"))
            loss = net(x).float().sum()
            hook.remove()
        loss.backward()
        keep = mgr.post_backward_sync_and_eval()
        assert keep is (not bad)
        if keep:
            assert all(bool(torch.isfinite(p.grad).all()) for p in params)
            opt.step()


def test_captured_training_step_matches_eager():
    from apa.graphs import GraphedTrainStep
    torch.manual_seed(1)
    cfg = APAConfig(device="cuda", check_interval=1)
    net = Net(cfg)
    mgr = APAManager(net, cfg)
    x, t = torch.randn(32, 48, device="cuda"), torch.randn(32, 10, device="cuda")
    step = GraphedTrainStep(mgr, lambda a, b: ((net(a).float() - b) ** 2).mean(), (x, t), warmup=2)
    for _ in range(3):
        loss, keep = step(x, t)
    assert keep and step.graph is not None
    got = [net.up.weight_master.grad.clone(), net.down.bias_master.grad.clone(), net.norm.weight.grad.clone()]
    # new weights: the captured step casts them anew
    with torch.no_grad():
        net.up.weight_master.mul_(0.5)
    loss2, _ = step(x, t)
    second = net.up.weight_master.grad.clone()
    torch.cuda.synchronize()
    for p in net.parameters():
        p.grad = None
    mgr.pre_step()
    eager = ((net(x).float() - t) ** 2).mean()
    eager.backward()
    assert torch.equal(eager.detach(), loss2) and torch.equal(net.up.weight_master.grad, second)
    assert not torch.equal(second, got[0])


def test_chain_serving_equals_modules():
    """norm -> product -> norm -> product in E4M3, as a decode step runs it, against the modules without gradients."""
    cfg = APAConfig(device="cuda")
    l1, l2 = layer(rnd((384, 256), 1)), layer(rnd((256, 384), 2))
    n1, n2 = APARMSNorm(256, config=cfg), APARMSNorm(256, config=cfg)
    w1, w2 = block_cast(l1.weight_master, square=True), block_cast(l2.weight_master, square=True)
    for rows in (1, 7, 150):
        x, r = rnd((rows, 256), rows, torch.bfloat16).cuda(), rnd((rows, 256), rows + 1, torch.bfloat16).cuda()
        with torch.no_grad():
            y, r1 = l1(x, norm=n1, residual=r)
            z, r2 = n2(l2(y), r1)
        q, s1 = rms_norm(x, n1.weight.detach(), r, quantize=True)
        u = apa.block_linear(apa.block_linear(q, w1), w2)
        v, s2 = rms_norm(u, n2.weight.detach(), s1)
        assert torch.equal(v, z) and torch.equal(s1, r1) and torch.equal(s2, r2)


def test_second_derivatives_are_refused():
    lin = layer(rnd((40, 64), 1))
    x = rnd((9, 64), 3).cuda().requires_grad_(True)
    norm = APARMSNorm(64, config=APAConfig(device="cuda"))
    for out in (lin(x), norm(x), lin(x, norm=norm)):
        (g,) = torch.autograd.grad(out.sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError):          # no gradient of it, or none a second time
            g.sum().backward()


def test_offsets_past_32_bits():
    """A training step over more than 2^31 activations, on whole numbers: the
    weight gradient's sums stay below 2^24, so all of it is exact."""
    m, k, n = 525_000, 4096, 72
    g = torch.Generator(device="cuda").manual_seed(1)

    def draw(rows, cols, top):
        return torch.randint(-top, top + 1, (rows, cols), generator=g, device="cuda", dtype=torch.int8)

    x, dy, w = draw(m, k, 3).to(torch.bfloat16), draw(m, n, 2).to(torch.bfloat16), draw(n, k, 3).float()
    assert x.numel() > 2 ** 31
    lin = layer(w)
    x.requires_grad_(True)
    y = lin(x)
    y.backward(dy)
    want = torch.zeros(n, k, device="cuda", dtype=torch.float64)
    with torch.no_grad():
        for lo in range(0, m, 75_000):
            want += dy[lo:lo + 75_000].double().T @ x[lo:lo + 75_000].double()
        assert torch.equal(lin.weight_master.grad.double(), want)
        for lo in (0, 262_100, m - 300):
            assert torch.equal(y[lo:lo + 300], (x[lo:lo + 300].double() @ w.double().T).to(torch.bfloat16))
            assert torch.equal(x.grad[lo:lo + 300], (dy[lo:lo + 300].double() @ w.double()).to(torch.bfloat16))


def test_two_steps_at_once():
    """Two layers' training steps on two streams, queued in turn by two threads,
    and then as two captured graphs replayed together: each gives what it gives
    alone, bit for bit."""
    import threading

    parts = []
    for seed, (m, k, n) in enumerate([(2100, 640, 1500), (700, 2048, 520)]):
        lin = layer(rnd((n, k), seed), rnd((n,), seed + 5))
        norm = APARMSNorm(k, config=APAConfig(device="cuda"))
        x = rnd((m, k), seed + 10, torch.bfloat16).cuda().requires_grad_(True)
        parts.append((lin, norm, x, rnd((m, n), seed + 20, torch.bfloat16).cuda(), torch.cuda.Stream()))

    def step(p):
        lin, norm, x, dy, _ = p
        y = lin(x, norm=norm)
        return (y.detach(),) + torch.autograd.grad(y, [x, norm.weight, lin.weight_master, lin.bias_master], dy)

    alone = [step(p) for p in parts]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(parts[i][4]):
            for _ in range(8):
                got[i].append(step(parts[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for want, outs in zip(alone, got):
        assert len(outs) == 8 and all(torch.equal(a, b) for out in outs for a, b in zip(out, want))

    graphs = []
    for p in parts:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=p[4]):
            out = step(p)
        graphs.append((g, out))
    for _ in range(4):
        for p, (g, _) in zip(parts, graphs):
            with torch.cuda.stream(p[4]):
                g.replay()
    torch.cuda.synchronize()
    for want, (_, out) in zip(alone, graphs):
        assert all(torch.equal(a, b) for a, b in zip(out, want))
