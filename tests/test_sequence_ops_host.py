"""What the gated recurrence, the 8-bit checkpoints and the cross-entropy refuse before any CUDA call, and their C++ front end."""
import ctypes as C
import os
import subprocess

import pytest

import rtensors_b200 as rt
from rtensors_b200 import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CTX = C.create_string_buffer(64)      # stands for a context: every call below is refused before it is looked at
BUF = C.create_string_buffer(64)
F32, I32 = L.F32, L.I32
SH, ST = L.sizes([2, 3, 4]), L.diffs([12, 4, 1])


def _scan(ctx=CTX, dtype=F32, flags=0, gate=BUF, x=BUF, h=BUF, rank=3, shape=SH, axis=1):
    return rt.lib().rtb_gated_scan(ctx, dtype, flags, gate, ST, 0, x, ST, 0, None, h, rank, shape, axis)


def _back(ctx=CTX, dtype=F32, flags=0, up=BUF, gate=BUF, x=None, h=BUF, codes=None, mags=None, d_gate=BUF, rank=3, shape=SH, axis=1):
    return rt.lib().rtb_gated_scan_backward(ctx, dtype, flags, up, ST, 0, gate, ST, 0, x, ST, 0, h, codes, mags, None, BUF, d_gate, None, rank,
                                            shape, axis)


def _step(ctx=CTX, dtype=F32, flags=0, state=BUF, ss=ST, rank=3, shape=SH):
    return rt.lib().rtb_gated_step(ctx, dtype, flags, state, ss, 0, BUF, ST, 0, BUF, ST, 0, rank, shape)


@pytest.mark.parametrize("call,code", [
    (lambda: _scan(ctx=None), L.ERR_INVALID), (lambda: _scan(dtype=I32), L.ERR_DTYPE), (lambda: _scan(flags=4), L.ERR_INVALID),
    (lambda: _scan(axis=3), L.ERR_DIM), (lambda: _scan(rank=0, axis=0), L.ERR_DIM), (lambda: _scan(rank=129), L.ERR_DIM),
    (lambda: _scan(shape=None), L.ERR_INVALID), (lambda: _scan(gate=None), L.ERR_INVALID), (lambda: _scan(h=None), L.ERR_INVALID),
    (lambda: _scan(shape=L.sizes([1, 1 << 31, 1])), -10),
    (lambda: _back(ctx=None), L.ERR_INVALID), (lambda: _back(dtype=I32), L.ERR_DTYPE), (lambda: _back(up=None), L.ERR_INVALID),
    (lambda: _back(h=None), L.ERR_INVALID), (lambda: _back(h=None, codes=BUF), L.ERR_INVALID),
    (lambda: _back(codes=BUF, mags=BUF), L.ERR_INVALID), (lambda: _back(flags=L.SCAN_COUPLED), L.ERR_INVALID), (lambda: _back(axis=7), L.ERR_DIM),
    (lambda: _step(ctx=None), L.ERR_INVALID), (lambda: _step(dtype=I32), L.ERR_DTYPE), (lambda: _step(flags=L.SCAN_REVERSE), L.ERR_INVALID),
    (lambda: _step(state=None), L.ERR_INVALID), (lambda: _step(ss=L.diffs([0, 4, 1])), L.ERR_SHAPE),
    (lambda: rt.lib().rtb_ckpt8_store(None, F32, BUF, 4, BUF, BUF), L.ERR_INVALID), (lambda: rt.lib().rtb_ckpt8_store(CTX, I32, BUF, 4, BUF, BUF), L.ERR_DTYPE),
    (lambda: rt.lib().rtb_ckpt8_store(CTX, F32, None, 4, BUF, BUF), L.ERR_INVALID),
    (lambda: rt.lib().rtb_ckpt8_store(CTX, F32, BUF, 4, C.addressof(BUF) + 1, BUF), L.ERR_INVALID),
    (lambda: rt.lib().rtb_ckpt8_restore(CTX, F32, BUF, None, 4, BUF), L.ERR_INVALID),
    (lambda: rt.lib().rtb_ckpt8_grad(CTX, F32, 4, BUF, BUF, BUF, 4, BUF), L.ERR_INVALID),
    (lambda: rt.lib().rtb_ckpt8_grad(CTX, F32, -1, BUF, BUF, BUF, 4, BUF), L.ERR_INVALID),
    (lambda: rt.lib().rtb_ckpt8_grad(CTX, F32, 0, BUF, BUF, None, 4, BUF), L.ERR_INVALID),
    (lambda: rt.lib().rtb_cross_entropy(None, F32, BUF, 2, 3, 3, BUF, 0, BUF, None), L.ERR_INVALID),
    (lambda: rt.lib().rtb_cross_entropy(CTX, I32, BUF, 2, 3, 3, BUF, 0, BUF, None), L.ERR_DTYPE),
    (lambda: rt.lib().rtb_cross_entropy(CTX, F32, BUF, 2, 3, 3, None, 0, BUF, None), L.ERR_INVALID),
    (lambda: rt.lib().rtb_cross_entropy(CTX, F32, None, 2, 3, 3, BUF, 0, BUF, None), L.ERR_INVALID),
    (lambda: rt.lib().rtb_cross_entropy(CTX, F32, BUF, 2, 3, 3, BUF, 2, BUF, None), L.ERR_INVALID),
    (lambda: rt.lib().rtb_cross_entropy(CTX, F32, BUF, 2, 3, 3, BUF, 0, None, None), L.ERR_INVALID)])
def test_refusals_before_any_work(call, code):
    assert call() == code
    assert rt.lib().rtb_last_error_string()


def test_nothing_to_do_is_no_error():
    empty = L.sizes([2, 0, 4])
    assert _scan(shape=empty, gate=None, x=None, h=None) == 0 and _step(shape=empty, state=None) == 0
    assert rt.lib().rtb_ckpt8_store(CTX, F32, None, 0, None, None) == 0
    assert rt.lib().rtb_ckpt8_grad(CTX, F32, 0, None, None, None, 0, None) == 0


def _build(tmp_path):
    rt.lib()
    lib = os.path.join(ROOT, "rtensors_b200")
    exe = str(tmp_path / "test_sequence_ops")
    p = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", "test_sequence_ops.cpp"),
                        "-o", exe, "-L", lib, "-lrt_b200", f"-Wl,-rpath,{lib}"], capture_output=True, text=True)
    assert p.returncode == 0, p.stderr
    return exe


def test_cpp_front_end_compiles_and_links(tmp_path):
    _build(tmp_path)


@pytest.mark.gpu
def test_cpp_front_end(tmp_path):
    p = subprocess.run([_build(tmp_path)], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stdout + p.stderr
    assert "ok:" in p.stdout
