"""The performance cases' calls of the library (perf/operators.py), on the CPU: the
reference cache stands in for the library."""
from __future__ import annotations

import importlib.util
import sys
import types
from pathlib import Path

import numpy as np
import pytest

import paged_ref as ref

torch = pytest.importorskip("torch")
REPO = Path(__file__).resolve().parent.parent


class Handed:
    """A tensor handed over, and how many were."""
    count = 0

    def __init__(self, x):
        self.x = x

    @classmethod
    def from_device(cls, x):
        assert x.is_contiguous() and x.dtype == torch.float32
        cls.count += 1
        return cls(x.numpy().copy())


class Cache:
    raised = 0  # exponents that appended rows raised in blocks with older ones

    def __init__(self, n_kv_heads, head_dim, rope, **_):
        self.ref, self.width = ref.RefCache(n_kv_heads, head_dim, rope), n_kv_heads * head_dim

    def map(self, slot, pages):
        pass

    def truncate(self, slots, lengths):
        assert all(self.ref._slot(s)["len"] >= n >= 0 for s, n in zip(slots, lengths))
        self.ref.truncate(slots, lengths)

    def append(self, k, v, slots, counts, rotate=True):
        assert k.x.shape == v.x.shape == (sum(counts), self.width)
        exps = [(e, dict(e), self.ref._slot(s)["len"]) for s in slots for e in self.ref._slot(s)["exps"]]
        self.ref.append(k.x, v.x, slots, counts, rotate)
        Cache.raised += sum(e[key] > was[key] for e, was, n in exps for key in was if key[0] * ref.BLOCK < n < (key[0] + 1) * ref.BLOCK)

    def read(self, slots, starts, counts):
        return tuple(x.astype(np.float32) for x in self.ref.read(slots, starts, counts))

    def attention(self, q, slots, counts):
        return self.ref.attention(q.x, slots, counts)[0].astype(np.float32)


def verify_drafts(target, ids, counts, accept, draw, draft=None):
    return ref.verify(target.x, ids, counts.tolist(), accept, draw, None if draft is None else draft.x)


@pytest.fixture
def cases(monkeypatch):
    lib = types.ModuleType("llmrs_hip")
    lib.Tensor, lib.HipPagedCache, lib.verify_drafts = Handed, Cache, verify_drafts
    lib.init, lib.sync = lambda device: None, lambda: None
    monkeypatch.setitem(sys.modules, "llmrs_hip", lib)
    monkeypatch.chdir(REPO)
    monkeypatch.setattr(sys, "path", list(sys.path))
    spec = importlib.util.spec_from_file_location("operator_cases", REPO / "perf" / "operators.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.DEV = "cpu"
    return mod


def equal(got, want):
    if isinstance(want, dict):
        assert got.keys() == want.keys()
        for key in want:
            equal(got[key], want[key])
    else:
        torch.testing.assert_close(torch.as_tensor(got), want, rtol=0, atol=0)


@pytest.mark.parametrize("seqs,rows,past,page", [(4, 5, 100, 64), (3, 1, 70, 32), (2, 40, 0, 32)])
def test_append_passes_do_the_same_work(cases, seqs, rows, past, page):
    """Every pass finds the blocks and exponents that the case has, and raises the same."""
    cases.own = True
    s = cases.prepare(cases._cache("append", "", "small", page, seqs, rows, past), 3)
    seen = []
    for _ in range(3):
        Handed.count = Cache.raised = 0
        got = cases.run(s)
        assert Handed.count == 2  # keys and values
        seen.append(Cache.raised)
        cases.own = False
        equal(got, cases.run(s))
        cases.own = True
    assert seen == seen[:1] * 3 and (rows != 5 or seen[0] > 0)


@pytest.mark.parametrize("given", [True, False])
def test_verify_passes_hand_their_tensors_over(cases, given):
    cases.own = True
    s = cases.prepare(cases._verify("", 3, 4, 501, given), 5)
    Handed.count = 0
    got = cases.run(s)
    assert Handed.count == 1 + given
    cases.own = False
    equal(got, cases.run(s))


def test_attention_passes_hand_their_queries_over(cases):
    cases.own = True
    s = cases.prepare(cases._cache("attention", "", "small", 32, 2, 2, 40), 5)
    Handed.count = 0
    got = cases.run(s)
    assert Handed.count == 1
    cases.own = False
    # both round sums of 42 terms and exponentials in f32, of values up to about 4
    torch.testing.assert_close(got, cases.run(s), rtol=0, atol=64 * 2.0 ** -24 * 4)
