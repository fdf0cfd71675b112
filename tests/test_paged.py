"""The paged cache and the verification of drafts without a GPU: the layout of a
block, and every call that is refused before a device is touched."""
from __future__ import annotations

import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import llmrs_hip as lh

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "llm.rs_amd" / "csrc"


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_block_layout(tmp_path):
    exe = tmp_path / "paged_layout"
    subprocess.run(["g++", "-O1", "-std=c++17", f"-I{CSRC}", "-o", str(exe), str(HERE / "native" / "paged_layout.cpp")], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "mismatches 0\n"


def cache(**kw):
    args = dict(n_kv_heads=2, head_dim=64, page_size=32, n_pages=6, max_seqs=3, max_seq=100, rope=None) | kw
    return lh.HipPagedCache(**args)


def refused(code, fn, *args, **kw):
    with pytest.raises(lh.LlmrsError) as e:
        fn(*args, **kw)
    assert e.value.code == code, e.value
    return str(e.value)


@pytest.mark.parametrize("kw", [
    {"head_dim": 96}, {"head_dim": 0}, {"n_kv_heads": 0}, {"n_kv_heads": 257}, {"page_size": 16}, {"page_size": 48},
    {"page_size": 8192}, {"page_size": -32}, {"n_pages": 0}, {"n_pages": -1}, {"page_size": 4096, "n_pages": 1 << 30},
    {"max_seqs": 0}, {"max_seqs": 65537}, {"max_seq": 0}, {"max_seq": (1 << 20) + 1},
    {"max_seqs": 65536, "max_seq": 1 << 20}, {"rope": -1.0}, {"rope": float("nan")}, {"rope": float("inf")},
])
def test_bad_configuration(kw):
    refused(lh.E_INVALID, cache, **kw)


def test_bad_tables():
    c, s = np.zeros((100, 32), np.float32), np.zeros((100, 31), np.float32)
    refused(lh.E_INVALID, cache, rope=(c, s))
    refused(lh.E_INVALID, cache, rope=(c[:50], c[:50]))
    cfg, h = lh.PagedConfig(2, 64, 32, 6, 3, 100, 0.0), C.c_void_p()
    assert lh.lib().llmrs_paged_create(C.byref(cfg), c.ctypes.data_as(C.c_void_p), None, C.byref(h)) == lh.E_INVALID
    assert lh.lib().llmrs_paged_create(None, None, None, C.byref(h)) == lh.E_INVALID
    assert not h.value


def test_mapping_pages():
    c = cache()
    c.map(0, [4, 2])
    assert "in use" in refused(lh.E_INVALID, c.map, 1, [2])
    refused(lh.E_INVALID, c.map, 0, [4])
    refused(lh.E_INVALID, c.map, 1, [3, 3])       # twice in one call
    c.map(1, [3])                                 # which took nothing
    refused(lh.E_RANGE, c.map, 1, [0, 6])
    refused(lh.E_RANGE, c.map, 1, [0, -1])
    refused(lh.E_RANGE, c.map, 0, [0, 1, 5])      # 100 positions are four pages
    refused(lh.E_RANGE, c.map, 3, [0])
    refused(lh.E_RANGE, c.map, -1, [0])
    c.map(0, [0, 1])
    c.map(0, [])
    c.release(0)
    c.map(2, [4, 2, 0, 1])
    assert c.length(2) == 0
    refused(lh.E_RANGE, c.length, 3)
    refused(lh.E_RANGE, c.release, 7)


@pytest.mark.parametrize("bad", [[2 ** 32], np.array([2 ** 32]), np.array([-2 ** 32]), np.array([2 ** 31], np.uint32),
                                 [0.5], np.array([0.0]), np.array([True])])
def test_numbers_that_are_no_slots(bad):
    """Wider numbers are not cut to 32 bits, and fractions not rounded."""
    c = cache()
    c.map(0, [0])
    for slots, counts in ((bad, [0]), ([0], bad)):
        refused(lh.E_INVALID, c.truncate, slots, counts)
        refused(lh.E_INVALID, c.append, None, None, slots, counts)
        refused(lh.E_INVALID, c.attention, None, slots, counts)
        refused(lh.E_INVALID, c.read, slots, [0], counts)
    refused(lh.E_INVALID, c.read, [0], bad, [0])
    refused(lh.E_INVALID, c.map, 1, bad)
    refused(lh.E_INVALID, lh.verify_drafts, None, bad, [1], [0.5], [0.5])
    refused(lh.E_INVALID, lh.verify_drafts, None, [0], bad, [0.5], [0.5])
    for call in (lambda s: c.map(s, [1]), c.release, c.length, lambda n: cache(n_pages=n), lambda n: cache(max_seq=n)):
        refused(lh.E_RANGE, call, 2 ** 32)
        with pytest.raises(TypeError):
            call(0.5)
    assert c.length(0) == 0 and c.length(1) == 0
    c.truncate(np.array([0], np.int64), [0])


def test_lengths_only_shrink():
    c = cache()
    refused(lh.E_RANGE, c.truncate, [0], [1])
    refused(lh.E_RANGE, c.truncate, [0], [-1])
    refused(lh.E_RANGE, c.truncate, [9], [0])
    refused(lh.E_INVALID, c.truncate, [0, 0], [0, 0])
    refused(lh.E_INVALID, c.truncate, [0, 1], [0])
    c.truncate([0, 2], [0, 0])
    c.truncate([], [])


class NoTensor:
    handle = None


def test_append_read_attention_refusals():
    """Slots, counts and positions are looked at before any tensor."""
    c, no = cache(), NoTensor()
    c.map(0, [0, 1, 2, 3])
    c.map(1, [5])
    for call in (c.append, lambda k, v, s, n: c.read(s, n, n), lambda k, v, s, n: c.attention(k, s, n)):
        refused(lh.E_RANGE, call, no, no, [3], [1])
        refused(lh.E_RANGE, call, no, no, [-1], [1])
        refused(lh.E_INVALID, call, no, no, [0, 0], [1, 1])
        refused(lh.E_RANGE, call, no, no, [0], [-1])
        refused(lh.E_RANGE, call, no, no, [0], [101])
        refused(lh.E_INVALID, call, no, no, [0, 1], [1])
    assert "no page" in refused(lh.E_RANGE, c.append, no, no, [0, 1], [100, 33])
    assert "no page" in refused(lh.E_RANGE, c.append, no, no, [2], [1])
    refused(lh.E_INVALID, c.append, no, no, [0], [100])          # fits: now the tensors
    refused(lh.E_RANGE, c.read, [0], [0], [1])                   # nothing there yet
    refused(lh.E_RANGE, c.read, [0], [-1], [0])
    refused(lh.E_RANGE, c.attention, no, [0], [1])
    refused(lh.E_INVALID, c.attention, no, [0], [0])
    assert [c.length(s) for s in range(3)] == [0, 0, 0]


def test_verify_refusals():
    no = NoTensor()
    refused(lh.E_INVALID, lh.verify_drafts, no, [1], [1], [0.5], [0.5])
    refused(lh.E_INVALID, lh.verify_drafts, no, [1], [2], [0.5], [0.5])
    refused(lh.E_INVALID, lh.verify_drafts, no, [1], [1], [0.5, 0.5], [0.5])
    refused(lh.E_INVALID, lh.verify_drafts, no, [], [-1, 1], [], [0.5, 0.5])
    accepted, tokens = lh.verify_drafts(no, [], [], [], [])
    assert accepted.shape == (0,) and tokens.shape == (0, 1)


def test_from_device_takes_device_memory_only():
    refused(lh.E_INVALID, lh.Tensor.from_device, np.zeros(3, np.float32))

    class Fake:
        def __init__(self, **kw):
            self.__cuda_array_interface__ = {"shape": (2, 3), "typestr": "<f4", "data": (0, False), "version": 3} | kw
    refused(lh.E_DTYPE, lh.Tensor.from_device, Fake(typestr="<f2"))
    refused(lh.E_INVALID, lh.Tensor.from_device, Fake(strides=(4, 8)))


def test_more_work_than_a_launch_has_threads():
    """2^32 threads in one dimension are refused, before any tensor is looked at; one
    sequence less is not."""
    c, no = cache(head_dim=128, page_size=4096, n_pages=2 * 65536, max_seqs=65536, max_seq=8192), NoTensor()
    for slot in range(65536):
        c.map(slot, [2 * slot, 2 * slot + 1])
    slots, rows = np.arange(65536, dtype=np.int32), np.full(65536, 8192, np.int32)  # 2^24 blocks of 256 threads
    assert "too much work" in refused(lh.E_INVALID, c.append, no, no, slots, rows)
    assert "null tensor" in refused(lh.E_INVALID, c.append, no, no, slots[:-1], rows[:-1])
    assert c.length(0) == c.length(65535) == 0
    # 2^24 workgroups of attention
    ones = np.ones(65536, np.int32)
    assert "too much work" in refused(lh.E_INVALID, lh.probe_paged_plan, 256, 64, 1, ones, ones)
    assert lh.probe_paged_plan(256, 64, 1, ones[:-1], ones[:-1]) == ([16] * 65535, [1] * 65535)
    # the launch of the second kernel too is looked at before the first is queued
    lengths, counts = np.append(ones, 1 << 20), np.append(ones, 1 << 20)
    assert "too much work" in refused(lh.E_INVALID, lh.probe_paged_plan, 256, 64, 64, lengths[1:], counts[1:])


def test_plan_covers_every_position():
    """Splits of at most 64, none longer than the sequence, and rows without any."""
    for kv, hd, group in ((1, 64, 1), (8, 128, 4), (2, 64, 20), (8, 64, 8), (16, 128, 1)):
        for lengths in ([1], [1, 255, 256, 257], [1 << 20], [4000] * 300, [9000] + [40] * 70, list(range(1, 2000, 37))):
            for rows in (0, 1, 5, 64, 700):
                counts = [min(rows, n) for n in lengths]
                columns, splits = lh.probe_paged_plan(kv, hd, group, lengths, counts)
                for n, r, c, s in zip(lengths, counts, columns, splits):
                    assert (c, s) == (0, 0) if r == 0 else c in (16, 64) and 1 <= s <= min(64, -(-n // (256 if c == 16 else 64)))
    refused(lh.E_RANGE, lh.probe_paged_plan, 1, 64, 1, [3], [4])
    refused(lh.E_INVALID, lh.probe_paged_plan, 0, 64, 1, [3], [3])


def test_plans_of_the_tested_calls():
    """The calls by which test_gpu_paged.py tests the kernel of 64 columns and the
    joining of splits come to it, on 256 CUs."""
    check_tested_plans(256)


def check_tested_plans(cus):
    from test_gpu_paged import MANY
    for nq, kv, hd, _, lens, counts in MANY:
        columns, _ = lh.probe_paged_plan(kv, hd, nq // kv, lens, counts, cus)
        assert columns == [0 if not r else 64 if r * nq // kv >= 64 else 16 for r in counts]
    assert lh.probe_paged_plan(8, 128, 4, [850], [800], cus)[0] == [64]
    assert lh.probe_paged_plan(8, 128, 4, [850, 40], [800, 1], cus)[0] == [64, 16]
    for lens, counts, columns in (([9000] + [40] * 70, [1] * 71, 16), ([9000, 300, 300], [16, 300, 300], 64)):
        c, s = lh.probe_paged_plan(8, 64, 8, lens, counts, cus)
        assert set(c) == {columns} and s[0] > 1 and set(s[1:]) == {1}
    for kv, length, rows in ((2, 5000, 1), (2, 5000, 6), (1, 1300, 2), (1, 1300, 600)):
        assert lh.probe_paged_plan(kv, 128, 4, [length], [rows], cus)[1][0] > 1
    assert lh.probe_paged_plan(8, 128, 4, [999, 500, 1, 64], [3, 2, 1, 1], cus)[1][0] > 1


def test_draws_stay_below_one():
    top = np.float32(1.0 - 2.0 ** -24)
    x = lh._draws([1.0 - 2.0 ** -53, 1.0, 0.25, 1.0 - 2.0 ** -26])
    assert x.dtype == np.float32 and x.tolist() == [top, 1.0, 0.25, top]
    same = np.float32([1.0, 0.5])
    assert lh._draws(same) is same
