"""The cast weight that a block layer keeps, without a GPU: streams, events and
the cast are stand-ins that note what happens in which order."""
import contextlib
import threading

import pytest
import torch

from apa import APABlockLinear, APAConfig, _lib, blockscale

W0 = torch.arange(12.0).view(3, 4)


class Stream:
    def __init__(self, handle, log):
        self.cuda_stream, self.log, self.capturing = handle, log, False

    def wait_event(self, event):
        self.log.append(("wait", self.cuda_stream, event.after))

    def wait_stream(self, other):
        self.log.append(("wait", self.cuda_stream, ("stream", other.cuda_stream)))


class Buffer:
    """Stands for the packed cast: holds the values it was cast from."""
    device = torch.device("cpu")

    def __init__(self, shape, log):
        self.shape, self.buffer, self.log, self.values = shape, self, log, None

    def record_stream(self, stream):
        self.log.append(("record", id(self), stream.cuda_stream))

    def data_ptr(self):
        return id(self)


@pytest.fixture
def stage(monkeypatch):
    """A layer whose casts, streams and events are noted in ``stage.log``."""
    class Stage:
        pass
    stage = Stage()
    stage.log, stage.local = [], threading.local()
    stage.streams = {h: Stream(h, stage.log) for h in (1, 2, 3)}
    stage.during_cast = stage.during_record = lambda: None
    here = lambda *a: stage.streams[getattr(stage.local, "handle", 1)]

    class Event:
        after = None

        def record(self, stream=None):
            self.after = ("event", (stream or here()).cuda_stream)
            stage.during_record()

    @contextlib.contextmanager
    def on(stream):
        before = getattr(stage.local, "handle", 1)
        stage.local.handle = stream if isinstance(stream, int) else stream.cuda_stream
        try:
            yield
        finally:
            stage.local.handle = before

    def cast(W, into=None):
        buf = into or Buffer(W.shape, stage.log)
        stage.log.append(("cast", here().cuda_stream, id(buf)))
        stage.during_cast()
        buf.values = W.detach().clone()
        return buf

    stage.on = on
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "current_stream", here)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: here().capturing)
    monkeypatch.setattr(_lib, "stream_handle", lambda d=None: here().cuda_stream)
    monkeypatch.setattr(_lib, "require_cuda", lambda t, what: None)
    monkeypatch.setattr(APABlockLinear, "_cast_weight", staticmethod(cast))

    def make():
        lin = APABlockLinear(4, 3, bias=False, config=APAConfig(device="cpu"))
        with torch.no_grad():
            lin.weight_master.copy_(W0)
        return lin

    stage.make = make
    stage.casts = lambda: [e for e in stage.log if e[0] == "cast"]
    return stage


def served(lin):
    """The values that a call without gradients would use now."""
    return lin._working_copy(lin.weight_master).values


def test_cast_once_while_nothing_changes(stage):
    lin = stage.make()
    for _ in range(3):
        assert torch.equal(served(lin), W0)
    assert len(stage.casts()) == 1
    with torch.no_grad():
        lin.weight_master.mul_(2.0)
    assert torch.equal(served(lin), 2 * W0) and len(stage.casts()) == 2


def test_weight_made_and_changed_in_inference_mode(stage):
    with torch.inference_mode():
        lin = stage.make()
        assert torch.equal(served(lin), W0)
        lin.weight_master.mul_(2.0)
        assert torch.equal(served(lin), 2 * W0)
        lin.refresh_working_copy()
        lin.load_state_dict({"weight_master": W0 + 1})
        assert torch.equal(served(lin), W0 + 1)


@pytest.mark.parametrize("kind", ["fused", "foreach", "own"])
def test_weight_changed_by_an_optimizer(stage, kind):
    """Fused optimizers leave the version counter as it was."""
    lin = stage.make()
    W = lin.weight_master

    class Raw(torch.optim.Optimizer):
        def step(self, closure=None):
            for g in self.param_groups:
                for p in g["params"]:
                    p.data.sub_(p.grad)

    if kind == "own":
        opt = Raw([W], {})
    else:
        opt = torch.optim.SGD([W], lr=1.0, **{kind: True})
    for turn in range(3):
        assert torch.equal(served(lin), W0 - turn)
        W.grad = torch.ones_like(W)
        opt.step()
    assert torch.equal(served(lin), W0 - 3)


def test_weight_changed_between_a_training_forward_and_a_call(stage, monkeypatch):
    """An update that no counter shows: the training forward before it is enough."""
    monkeypatch.setattr(blockscale._BlockLinearFn, "apply", staticmethod(lambda *a: a[0]))
    lin = stage.make()
    assert torch.equal(served(lin), W0)
    lin(torch.ones(2, 4))
    lin.weight_master.data.mul_(2.0)
    assert torch.equal(served(lin), 2 * W0)


def ordered(log, handle, block):
    """Whether work of stream `handle` that reads `block` comes behind its last cast."""
    by = [e[1] for e in log if e[0] == "cast" and e[2] == id(block)][-1]
    return by == handle or ("wait", handle, ("event", by)) in log


def test_first_calls_of_two_threads(stage):
    """Two streams, a thread each. Where both casts can be under way together,
    the second one's buffer is stored before the first call returns."""
    lin = stage.make()
    casting, both, recorded, second = (threading.Event() for _ in range(4))
    got = {}

    def during_cast():
        if threading.current_thread().name == "first":
            casting.set()
            both.wait(0.3)
        else:
            both.set()
            recorded.wait(0.3)

    def during_record():
        if threading.current_thread().name == "first":
            recorded.set()
            second.wait(0.3)

    stage.during_cast, stage.during_record = during_cast, during_record

    def call(handle):
        with stage.on(handle):
            got[handle] = lin._working_copy(lin.weight_master)
        if handle == 2:
            second.set()

    a = threading.Thread(target=call, args=(1,), name="first")
    b = threading.Thread(target=call, args=(2,), name="second")
    a.start()
    casting.wait()
    b.start()
    a.join()
    b.join()
    for handle, block in got.items():
        assert ordered(stage.log, handle, block), (handle, stage.log)
    # and so does the next call of a third stream
    with stage.on(3):
        block = lin._working_copy(lin.weight_master)
    assert ordered(stage.log, 3, block)


def test_copies_and_pickles_have_their_own(stage):
    import copy
    import pickle

    lin = stage.make()
    served(lin)
    for other in (copy.deepcopy(lin), pickle.loads(pickle.dumps(lin))):
        assert other._wq is None and torch.equal(served(other), W0)
        with torch.no_grad():
            other.weight_master.mul_(2.0)
        assert torch.equal(served(other), 2 * W0) and torch.equal(served(lin), W0)


@pytest.mark.parametrize("how", ["replaced", "data", "refresh"])
def test_renewal_waits_for_readers_on_other_streams(stage, how):
    """A replaced weight needs no ordering, so products of the old one may still be queued."""
    lin = stage.make()
    for handle in (1, 2):
        with stage.on(handle):
            served(lin)
    kept = lin._wq
    stage.log.clear()
    if how == "replaced":
        lin.weight_master = torch.nn.Parameter(2 * W0)
    else:
        lin.weight_master.data = 2 * W0
    with stage.on(3):
        if how == "refresh":
            lin.refresh_working_copy()
        assert torch.equal(served(lin), 2 * W0)
    assert lin._wq is kept                       # captured graphs see the new values
    cast = stage.log.index(("cast", 3, id(kept)))
    for entry in (("wait", 3, ("stream", 1)), ("wait", 3, ("stream", 2)), ("record", id(kept), 3)):
        assert stage.log.index(entry) < cast
    assert len(stage.casts()) == 1
    # what comes next waits for the new cast
    with stage.on(1):
        assert torch.equal(served(lin), 2 * W0) and ordered(stage.log, 1, kept)


def test_renewal_beside_a_capture(stage):
    """A stream that is being captured cannot be waited for."""
    lin = stage.make()
    with stage.on(2):
        served(lin)
    stage.streams[2].capturing = True
    with torch.no_grad():
        lin.weight_master.mul_(2.0)
    assert torch.equal(served(lin), 2 * W0)
    assert ("wait", 1, ("stream", 2)) not in stage.log
