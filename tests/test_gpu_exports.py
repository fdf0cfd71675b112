"""Tensors of the library used in place by another library of the process
(``__cuda_array_interface__``), with no wait of the caller's.  Each test is a
process of its own, which loads the other library first."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

START = """
import torch                     # before the library: they share one HIP runtime
import numpy as np
import llmrs_hip as hip
hip.init(0)
rng = np.random.default_rng(4)
nkv, nq, hd, rows = 8, 32, 128, 1024
cache = hip.HipPagedCache(nkv, hd, 64, 16, 1, rows)
cache.map(0, range(16))
cache.append(*(hip.Tensor.from_numpy(rng.standard_normal((rows, nkv * hd)).astype(np.float32)) for _ in "kv"), [0], [rows])
q = [hip.Tensor.from_numpy(rng.standard_normal((rows, nq * hd)).astype(np.float32)) for _ in range(2)]
want = [torch.as_tensor(cache.attention(x, [0], [rows]).data()) for x in q]
torch.zeros(1, device="cuda")
torch.cuda.synchronize()
"""


def run(script):
    pytest.importorskip("torch")
    pkg = Path(__file__).resolve().parent.parent / "llm.rs_amd"
    got = subprocess.run([sys.executable, "-c", START + script + "\nprint('done')\n"], capture_output=True, text=True, timeout=100,
                         env=dict(os.environ, PYTHONPATH=str(pkg)))
    assert got.stdout.strip() == "done", got.stderr[-2000:]


def test_values_are_there_when_the_address_is():
    """Rows of attention and of read-back, read on another library's streams as soon
    as the call has returned, behind calls that are still queued."""
    run("""
side = torch.cuda.Stream()
k, v = (torch.as_tensor(x.data()) for x in cache.read([0], [0], [rows]))
for stream in (torch.cuda.default_stream(), side):
    with torch.cuda.stream(stream):
        for i in (0, 1, 0):
            for _ in range(8):
                kept = cache.attention(q[1 - i], [0], [rows])
            out = cache.attention(q[i], [0], [rows])
            view = torch.as_tensor(out, device="cuda")
            got = view.clone()
            assert view.data_ptr() == out.__cuda_array_interface__["data"][0]
            assert torch.equal(got.cpu(), want[i])
            kept = cache.attention(q[i], [0], [rows])
            back = cache.read([0], [0], [rows])
            views = [torch.as_tensor(x, device="cuda") for x in back]
            copies = [x.clone() for x in views]
            assert torch.equal(copies[0].cpu(), k) and torch.equal(copies[1].cpu(), v)
""")


def test_memory_outlives_what_still_reads_it():
    """A view is dropped while work that reads it waits behind other work of its
    stream; calls that follow do not write there."""
    run("""
side = torch.cuda.Stream()
a = torch.zeros(1 << 26, device="cuda")
torch.cuda.synchronize()
for i in (0, 1, 0):
    view = torch.as_tensor(cache.attention(q[i], [0], [rows]), device="cuda")
    with torch.cuda.stream(side):
        for _ in range(40):      # about 4 ms
            a += 1
        got = view.clone()
    del view
    for _ in range(4):
        cache.attention(q[1 - i], [0], [rows])
    side.synchronize()
    assert torch.equal(got.cpu(), want[i])
""")


def test_memory_of_dropped_views_is_used_again():
    """Not for the next tensor, but once the device has been waited for."""
    run("""
def address(t):
    return t.__cuda_array_interface__["data"][0]
seen, last = set(), None
for _ in range(30):
    t = cache.attention(q[0], [0], [rows])
    assert address(t) != last
    last = address(t)
    seen.add(last)
    del t
assert len(seen) <= 4, len(seen)
# (the first round's tensors are free before the second round's: it asks for more)
for wait, n in ((hip.sync, 6), (lambda: hip.Tensor.from_device(torch.zeros(1, device="cuda")), 16)):
    t = cache.attention(q[0], [0], [rows])
    last = address(t)
    del t
    wait()
    kept = [cache.attention(q[0], [0], [rows]) for _ in range(n)]
    assert last in [address(t) for t in kept]
    del kept
""")
