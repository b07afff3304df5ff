"""The limit of dynamic shared memory that kernels share over contexts and threads (csrc/rtb_cluster.cuh): two threads whose first calls
need different sizes."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_two_threads_raise_one_limit(tmp_path):
    exe = str(tmp_path / "test_rising_limit")
    cuda = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    p = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-pthread", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "rtensors_b200", "csrc"),
                        "-isystem", cuda, os.path.join(ROOT, "tests", "cpp", "test_rising_limit.cpp"), "-o", exe], capture_output=True, text=True)
    assert p.returncode == 0, p.stderr
    p = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0 and "ok" in p.stdout, p.stdout + p.stderr


_FIRST_CALLS = """
import sys, threading
sys.path.insert(0, sys.argv[1])
import torch
from rtensors_b200.backend import CudaB200
from rtensors_b200.meta import Meta
from rtensors_b200.tensor import Tensor
torch.zeros(1, device="cuda")
start, errors = threading.Barrier(2), []
def run(steps):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            be, shape = CudaB200(0), (1, steps, 64)
            x, a = (Tensor(be, torch.full((steps * 64,), v, device="cuda"), Meta.contiguous(shape)) for v in (1.0, 0.5))
            be.sync()
            start.wait()
            for _ in range(3):
                h = x.gated_scan_at(1, a)     # 1, 1.5, 1.75 ...: 2 to the last bit behind 30 steps
                be.sync()
                assert bool((h.buf.view(steps, 64)[30:] == 2.0).all()) and float(h.buf[64]) == 1.5
            be.close()
    except BaseException as e:
        errors.append(e)
threads = [threading.Thread(target=run, args=(n,)) for n in (60000, 1500)]
for t in threads: t.start()
for t in threads: t.join(60)
sys.exit(repr(errors) if errors or any(t.is_alive() for t in threads) else 0)
"""


@pytest.mark.gpu
def test_first_calls_of_two_threads():
    """In a process of its own, where no size has been asked for: long and short axes need clusters of different sizes."""
    for _ in range(3):
        p = subprocess.run([sys.executable, "-c", _FIRST_CALLS, ROOT], capture_output=True, text=True, timeout=180)
        assert p.returncode == 0, p.stdout + p.stderr
