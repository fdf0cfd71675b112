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
