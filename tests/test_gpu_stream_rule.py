"""One stream rule for all operations of a shared backend: each call goes to torch's current stream, behind all earlier calls."""
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LONG = 40_000_000   # cycles, some twenty milliseconds


def _b():
    from cuda_engine import backend
    return backend()


def _t(a):
    from rtensors_b200.tensor import Tensor
    return Tensor.from_buf(a, a.shape, a.dtype.type, _b())


def test_ordinary_operations_after_a_sequence_call_on_another_stream():
    rng = np.random.default_rng(1)
    x, a = (rng.uniform(0, 1, (2, 40, 24)).astype(np.float32) for _ in range(2))
    tx, ta = _t(x), _t(a)
    want = (tx.gated_scan_at(1, ta) + 1.0).cpu()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            h = tx.gated_scan_at(1, ta)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.stream(side):
            torch.cuda._sleep(LONG)          # what lands on `side` now is late
        y = h + 1.0                          # the current stream is the default one again
        torch.cuda.current_stream().synchronize()
        assert y.buf.cpu().numpy().tobytes() == want.tobytes()
        y += h
        s = y.sum()
        assert abs(float(s.item()) - float((2 * want.astype(np.float64) - 1).sum())) <= 1e-3 * abs(float(s.item()))
    side.synchronize()


def test_ordinary_operations_after_a_captured_sequence_call():
    from rtensors_b200.tensor import cross_entropy_loss
    rng = np.random.default_rng(2)
    x, t = _t(rng.standard_normal((64, 40)).astype(np.float32)), _t(rng.integers(0, 40, 64))
    want = cross_entropy_loss(x, t).cpu(), (x * x).cpu()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss = cross_entropy_loss(x, t)      # no sync_stream
    y = x * x
    assert y.cpu().tobytes() == want[1].tobytes()
    loss.buf.zero_()
    graph.replay()
    assert loss.cpu().tobytes() == want[0].tobytes()


def test_operands_are_brought_into_form_on_the_current_stream():
    """Labels of another type and views that are copied first: the conversion and the copy come behind what the current stream holds."""
    from rtensors_b200.tensor import cross_entropy_loss
    rng = np.random.default_rng(3)
    x, t = rng.standard_normal((24, 400)).astype(np.float32), rng.integers(0, 24, 400).astype(np.int32)
    tx, tt, zeros = _t(np.zeros_like(x)), _t(np.zeros_like(t)), _t(x)
    want = cross_entropy_loss(_t(x).transpose(), _t(t)).cpu(), zeros.transpose().checkpoint8().codes.cpu()
    src_x, src_t = torch.from_numpy(x).cuda(), torch.from_numpy(t).cuda()
    _b().sync()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
        tx.buf.copy_(src_x.view(-1))
        tt.buf.copy_(src_t)
        loss, codes = cross_entropy_loss(tx.transpose(), tt), tx.transpose().checkpoint8().codes
    side.synchronize()
    assert loss.buf.cpu().numpy().tobytes() == want[0].tobytes() and torch.equal(codes.cpu(), want[1])
    torch.cuda.synchronize()


def test_two_threads_share_a_backend_on_streams_of_their_own():
    from rtensors_b200.tensor import cross_entropy_loss
    rng = np.random.default_rng(4)
    x, a = (rng.uniform(0, 1, (3, 300, 40)).astype(np.float32) for _ in range(2))
    t = rng.integers(0, 40, (3, 300))
    tx, ta, tt = _t(x), _t(a), _t(t)

    def passes():
        out = []
        for _ in range(20):
            h = tx.gated_scan_at(1, ta)
            loss = cross_entropy_loss(h + 1.0, tt)
            out += [h.buf, loss.buf, (h * ta).sum_at(1).buf]
        return out
    want = [v.cpu().numpy().tobytes() for v in passes()]
    torch.cuda.synchronize()
    got, errors = {}, []

    def run(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                outs = passes()
                stream.synchronize()
                got[k] = [v.cpu().numpy().tobytes() for v in outs]
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(120)
    assert not errors and len(got) == 4
    for k in range(4):
        assert got[k] == want
    torch.cuda.synchronize()


def test_calls_keep_their_order_across_a_capture():
    """A stream that is left for a capture is waited for by the next ordinary one."""
    from rtensors_b200.backend import CudaB200
    from rtensors_b200.meta import Meta
    from rtensors_b200.tensor import Tensor
    be = CudaB200(0)
    try:
        buf = torch.zeros(5000, device="cuda")
        x, kept = Tensor(be, buf, Meta.contiguous((5000,))), Tensor(be, torch.ones(64, device="cuda"), Meta.contiguous((64,)))
        streams = [torch.cuda.Stream() for _ in range(3)]
        _ = kept + kept
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            torch.cuda._sleep(LONG)
            x += kept.slice(0, 0, 1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(streams[1]):
            graph.capture_begin(capture_error_mode="relaxed")    # unlike torch.cuda.graph, without a synchronisation
            z = kept * kept
            graph.capture_end()
        with torch.cuda.stream(streams[2]):
            y = x + x                          # behind the addition on the first stream
        streams[2].synchronize()
        assert bool((y.buf == 2.0).all())
        torch.cuda.synchronize()
        del graph, z
    finally:
        torch.cuda.synchronize()
        be.close()
