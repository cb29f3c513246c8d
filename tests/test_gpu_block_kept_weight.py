"""The cast weight that a block layer keeps for calls without gradients, on the
GPU: every change of the parameter shows in the next call, whatever made it.
Scaling a weight by a power of two scales the layer's output exactly, and whole
numbers of few bits make every product exact, so all comparisons are bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from apa import APABlockLinear, APAConfig


def rnd(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def layer(w, dtype=torch.float32):
    lin = APABlockLinear(w.shape[1], w.shape[0], bias=False, dtype=dtype, config=APAConfig(device="cuda"))
    with torch.no_grad():
        lin.weight_master.copy_(w)
    return lin


def test_weight_changed_in_place_in_inference_mode():
    """A weight made there has no version counter."""
    w, x = rnd((40, 64), 1), rnd((3, 64), 2).cuda()
    with torch.no_grad():
        want = layer(w)(x)
    with torch.inference_mode():
        lin = layer(w)
        assert lin.weight_master.is_inference() and torch.equal(lin(x), want)
        lin.weight_master.mul_(2.0)
        assert torch.equal(lin(x), 2 * want)
        lin.load_state_dict({"weight_master": 4 * w.cuda()})
        assert torch.equal(lin(x), 4 * want)
        lin.refresh_working_copy()
        lin.weight_master.mul_(2.0)
        assert torch.equal(lin(x), 8 * want)
    with torch.no_grad():
        assert torch.equal(lin(x), 8 * want)


@pytest.mark.parametrize("kind", ["fused", "foreach", "apa"])
def test_evaluation_after_an_optimizer_step(kind):
    """Evaluate, train, evaluate: every evaluation uses the stepped weight, also
    when steps follow each other without a forward between them."""
    from apa import APAManager
    from apa.optim import APAAdamW

    w, x = rnd((40, 64), 1), rnd((3, 64), 2).cuda()
    lin = layer(w)
    if kind == "apa":
        opt = APAAdamW(APAManager(torch.nn.Sequential(lin), APAConfig(device="cuda")), lr=0.1)
    else:
        opt = torch.optim.AdamW(lin.parameters(), lr=0.1, **{kind: True})

    def check():
        with torch.no_grad():
            fresh = layer(lin.weight_master)
            assert torch.equal(lin(x), fresh(x))

    check()
    for _ in range(3):
        lin(x).sum().backward()
        opt.step()
        before = lin.weight_master.detach().clone()
        check()
        opt.step()
        assert not torch.equal(lin.weight_master, before)
        check()


def test_first_calls_of_two_threads():
    """A stream and a thread each, released together onto fresh layers."""
    import threading

    w, x = rnd((1024, 1024), 1), rnd((5, 1024), 2).cuda()
    with torch.no_grad():
        want = layer(w)(x)
    streams = [torch.cuda.Stream() for _ in range(4)]
    layers = [layer(w) for _ in range(10)]
    torch.cuda.synchronize()
    gate = threading.Barrier(len(streams))
    outs = [[] for _ in streams]

    def work(i):
        with torch.no_grad(), torch.cuda.stream(streams[i]):
            for lin in layers:
                gate.wait()
                outs[i].append(lin(x))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(streams))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(len(o) == len(layers) and all(torch.equal(y, want) for y in o) for o in outs)


@pytest.mark.parametrize("how", ["replaced", "data"])
def test_replaced_while_another_stream_still_reads(how):
    """A product queued behind other work reads the weight it was called with."""
    w, x = rnd((2048, 2048), 1), rnd((64, 2048), 2).cuda()
    lin = layer(w)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    new = -w.cuda()
    torch.cuda.synchronize()
    with torch.no_grad():
        with torch.cuda.stream(a):
            want = lin(x)
        with torch.cuda.stream(b):
            lin(x)                                    # b is behind the cast
            torch.cuda.synchronize()
            torch.cuda._sleep(100_000_000)            # 50 ms of the GPU's clock
            old = lin(x)
        if how == "replaced":
            lin.weight_master = torch.nn.Parameter(new)
        else:
            lin.weight_master.data = new
        with torch.cuda.stream(a):
            fresh = lin(x)
    torch.cuda.synchronize()
    assert torch.equal(old, want) and torch.equal(fresh, -want)


def test_serving_without_gradients():
    """The layer's parts called one by one, as its parameters are, equal the layer."""
    from apa import APARMSNorm, block_cast, block_linear, block_matmul, rms_norm

    cfg = APAConfig(device="cuda")
    norm, up = APARMSNorm(256, config=cfg), APABlockLinear(256, 384, config=cfg)
    x, h = rnd((7, 256), 1, torch.bfloat16).cuda(), rnd((7, 256), 2, torch.bfloat16).cuda()
    with torch.no_grad():
        w = block_cast(up.weight_master, square=True)
        q, r = rms_norm(x, norm.weight, residual=h, quantize=True)
        y = block_linear(q, w, up.bias_master)
        z = block_matmul(q, w, up.bias_master, out_dtype=torch.bfloat16)
        want, stream = up(x, norm=norm, residual=h)
        assert torch.equal(y, want) and torch.equal(z, want) and torch.equal(r, stream)
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm(x, norm.weight, residual=h, quantize=True)
    for call in (lambda: block_linear(q, w, up.bias_master), lambda: block_linear(x, w, up.bias_master),
                 lambda: block_matmul(q, w, up.bias_master)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
