"""Every call of a backend is enqueued on torch's current stream of the calling thread, whichever call or thread came before: on a
stand-in for the library that notes the stream the context is bound to during each call."""
import threading

import pytest
import torch

from rtensors_b200 import _lib as L
from rtensors_b200 import backend as B
from rtensors_b200.meta import Meta
from rtensors_b200.tensor import Tensor, cross_entropy_loss, gated_scan_backward


class _Library:
    """Entry points do nothing but note (name, bound stream at entry, bound stream at exit)."""

    def __init__(self):
        self.bound, self.calls, self.pause = None, [], lambda name: None

    def __getattr__(self, name):
        if name == "rtb_ctx_set_stream":
            def bind(ctx, stream):
                self.pause(name)
                self.bound = getattr(stream, "value", stream) or 0
                return 0
            return bind

        def call(*args):
            before = self.bound
            self.pause(name)
            self.calls.append((name, before, self.bound))
            return 0
        return call


@pytest.fixture
def rig(monkeypatch):
    """-> (backend over CPU buffers, the stand-in, a thread-local whose .stream is the current stream)"""
    library, now = _Library(), threading.local()
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: type("S", (), {"cuda_stream": getattr(now, "stream", 0)}))
    monkeypatch.setattr(B, "_current_stream", lambda index: getattr(now, "stream", 0))
    monkeypatch.setattr(B, "lib", lambda: library)
    be = B.CudaB200(0)
    be._torch_device, be._index = torch.device("cpu"), -1
    library.calls.clear()
    return be, library, now


def _ops(be):
    """Calls of each kind, by name: what they enqueue differs, the stream must not."""
    t = lambda *shape: Tensor(be, torch.ones(shape).view(-1), Meta.contiguous(shape))
    x, a, labels = t(2, 3, 4), t(2, 3, 4), Tensor(be, torch.zeros(6, dtype=torch.int32), Meta.contiguous((6,)))
    return {
        "scan": lambda: x.gated_scan_at(1, a), "scan of views": lambda: x.gated_scan_at(1, a, t(2, 1, 8).slice(2, 0, 4)),
        "backward": lambda: gated_scan_backward(x, 1, a, x), "step": lambda: x.gated_step_inplace(a, x),
        "checkpoint": lambda: x.checkpoint8().restore(), "checkpoint of a view": lambda: x.transpose().checkpoint8(),
        "loss": lambda: cross_entropy_loss(t(6, 4), labels, True), "loss of a view": lambda: cross_entropy_loss(t(4, 6).transpose(), labels),
        "add": lambda: x + a, "scalar": lambda: x + 1.0, "in place": lambda: x.relu_inplace(), "fill": lambda: x.fill(2.0), "copy": lambda: x.contiguous(),
        "sum": lambda: be.reduce_view(x.buf, x.meta, 1, L.SUM), "sgd": lambda: be.sgd_update(x.buf, a.buf, 0.1),
        "convert": lambda: be.convert(x.buf, torch.float64), "d2d": lambda: be.copy(x.buf), "read": lambda: be.read(x.buf, 0),
        "l1": lambda: be.l1_loss(x.buf, a.buf),
    }


def test_each_call_goes_to_the_current_stream(rig):
    be, library, now = rig
    ops = _ops(be)
    library.calls.clear()
    for first in ops:
        for second in ops:
            now.stream = 7
            ops[first]()
            now.stream = 9
            n = len(library.calls)
            assert all(c[1] == c[2] == 7 for c in library.calls)
            ops[second]()          # no sync_stream in between
            assert all(c[1] == c[2] == 9 for c in library.calls[n:]), (first, second, library.calls[n:])
            library.calls.clear()


@pytest.mark.parametrize("first", ["scan", "loss", "add", "checkpoint", "sum"])
@pytest.mark.parametrize("second", ["scan", "add", "step"])
def test_two_threads_with_streams_of_their_own(rig, first, second):
    """A thread that is inside a call keeps its stream until the call has returned."""
    be, library, now = rig
    ops = _ops(be)
    library.calls.clear()
    inside, rebound, errors = threading.Event(), threading.Event(), []

    def pause(name):
        if threading.current_thread().name == "one" and name != "rtb_ctx_set_stream":
            inside.set()
            rebound.wait(0.2)       # long enough for the other thread to bind its stream, if it may
        elif threading.current_thread().name == "two" and name != "rtb_ctx_set_stream":
            rebound.set()

    def run(name, op, stream):
        try:
            now.stream = stream
            if name == "two":
                inside.wait(5)
            op()
        except Exception as e:      # a failure in a thread would go unseen
            errors.append(e)
    library.pause = pause
    threads = [threading.Thread(target=run, args=a, name=a[0]) for a in (("one", ops[first], 7), ("two", ops[second], 9))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
    assert not errors and not any(t.is_alive() for t in threads)
    assert {c[1] for c in library.calls} == {7, 9}
    assert all(c[1] == c[2] for c in library.calls), library.calls


def test_waiting_follows_the_current_stream(rig):
    be, library, now = rig
    now.stream = 3
    be.sync()
    now.stream = 4
    be.host_wait()
    assert [c[1] for c in library.calls] == [3, 4]
