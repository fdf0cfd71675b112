"""The paged 8-bit cache, its attention and the verification of drafts on the
GPU, against numpy in 64 bits (paged_ref.py).  Codes are compared exactly;
the attention within the bound that the reference derives."""
from __future__ import annotations

import math
import os
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def within(got, want, tol):
    off = np.where(np.isnan(got), np.inf, np.abs(got - want)) / tol
    i = np.unravel_index(int(np.argmax(off)), off.shape)
    assert off[i] <= 1.0, f"at {i}: {got[i]!r}, in 64 bits {want[i]!r}, {off[i]:.3g} of the bound; {int((off > 1).sum())} like it"


class Both:
    """A cache on the GPU and the reference's, driven alike."""

    def __init__(self, hip, nkv, hd, page=32, pages=None, seqs=8, max_seq=1024, rope="tables", seed=1):
        self.hip, self.nkv, self.hd, self.page, self.max_seq = hip, nkv, hd, page, max_seq
        self.rng = np.random.default_rng(seed)
        tables = ref.rope_tables(max_seq, hd) if rope == "tables" else None
        self.ref = ref.RefCache(nkv, hd, tables)
        n = pages or seqs * -(-max_seq // page)
        self.gpu = hip.HipPagedCache(nkv, hd, page, n, seqs, max_seq, rope=tables)
        self.free = list(self.rng.permutation(n))
        self.mapped = [0] * seqs

    def room(self, slots, counts):
        for s, n in zip(slots, counts):
            want = -(-(self.gpu.length(s) + n) // self.page)
            if want > self.mapped[s]:
                self.gpu.map(s, [self.free.pop() for _ in range(want - self.mapped[s])])
                self.mapped[s] = want

    def rows(self, n, scale=1.0):
        return (self.rng.standard_normal((n, self.nkv * self.hd)) * scale).astype(np.float32)

    def append(self, slots, counts, k=None, v=None, rotate=True):
        n = int(np.sum(counts))
        k = self.rows(n) if k is None else k
        v = self.rows(n) if v is None else v
        self.room(slots, counts)
        self.gpu.append(self.hip.Tensor.from_numpy(k), self.hip.Tensor.from_numpy(v), slots, counts, rotate=rotate)
        self.ref.append(k, v, slots, counts, rotate=rotate)

    def check_rows(self, slots=None):
        slots = sorted(self.ref.slots) if slots is None else slots
        lens = [self.gpu.length(s) for s in slots]
        assert lens == [self.ref.slots[s]["len"] for s in slots]
        got = self.gpu.read(slots, [0] * len(slots), lens)
        for g, want in zip(got, self.ref.read(slots, [0] * len(slots), lens)):
            np.testing.assert_array_equal(g.data(), want.astype(np.float32))

    def check_attention(self, nq, slots, counts, scale=1.0):
        q = (self.rng.standard_normal((int(np.sum(counts)), nq * self.hd)) * scale).astype(np.float32)
        got = self.gpu.attention(self.hip.Tensor.from_numpy(q), slots, counts).data()
        want, tol = self.ref.attention(q, slots, counts)
        within(got, want, tol)
        return got


SHAPES = [(1, 64), (2, 64), (8, 64), (1, 128), (3, 128), (8, 128)]


@pytest.mark.parametrize("nkv,hd", SHAPES)
@pytest.mark.parametrize("page", [32, 64, 256])
def test_append_by_pieces(hip, nkv, hd, page):
    """Rows that come one by one, in pieces and as prompts, in slots of any order;
    later rows larger, so that blocks raise their exponents."""
    b = Both(hip, nkv, hd, page, seqs=5, max_seq=300)
    for step, (slots, counts) in enumerate([([3, 0], [1, 40]), ([0, 4, 3], [1, 100, 2]), ([1], [1]), ([3, 1, 0], [31, 0, 5]),
                                            ([0], [1]), ([4, 2], [64, 33]), ([4], [1]), ([2, 3], [0, 7])]):
        n = sum(counts)
        grow = np.float32(1.7 ** step)
        b.append(slots, counts, b.rows(n, grow), b.rows(n, grow * 0.3))
        b.check_rows()


@pytest.mark.parametrize("hd", [64, 128])
def test_append_one_by_one_growing(hip, hd):
    """Every row of a block raises the exponent, by 0 to 9 steps."""
    b = Both(hip, 2, hd, max_seq=96)
    for i in range(70):
        b.append([0], [1], b.rows(1, 2.0 ** (i % 32 * 1.3)), b.rows(1, 2.0 ** ((i * 7) % 40 - 20)))
    b.check_rows()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rope", ["tables", None])
def test_append_without_rotation(hip, hd, rope):
    b = Both(hip, 2, hd, rope=rope)
    b.append([0, 1], [45, 3], rotate=False)
    b.append([0], [7])
    b.check_rows()


def test_append_reads_back_what_it_holds(hip):
    """Values of the cache, appended unrotated to another slot, are held as they are."""
    b = Both(hip, 2, 128)
    b.append([0], [77])
    k, v = b.gpu.read([0], [0], [77])
    b.room([1], [77])
    b.gpu.append(k, v, [1], [77], rotate=False)
    for x, y in zip((k, v), b.gpu.read([1], [0], [77])):
        np.testing.assert_array_equal(x.data(), y.data())


@pytest.mark.parametrize("hd", [64, 128])
def test_append_special_values(hip, hd):
    """Zeros, borders of a step and of an exponent, the smallest and largest
    magnitudes, NaN and infinities."""
    b = Both(hip, 2, hd, max_seq=400)
    nan, inf = np.nan, np.inf
    border = np.array([0.5, 1.5, 2.5, -0.5, -1.5, 126.5, 127.0, 63.5, 0.49999997, 3.4999998], np.float32)
    sets = [np.zeros(1), border, border * 2.0 ** -30, border * 2.0 ** 100, [127.0], [127.00001], [2.0 ** -101, 2.0 ** -149],
            [2.0 ** -94], [3.4028235e38, 1.0], [inf, 1.0, -inf, nan], [nan], [1.0, nan, -3.0], [-0.0, 1e-3]]
    for rows, part in enumerate(sets):
        x = np.resize(np.asarray(part, np.float32), (3 + rows % 4, 2 * hd)).astype(np.float32)
        b.append([0], [x.shape[0]], x, x[::-1].copy())
        b.append([1], [x.shape[0]], x, -x, rotate=False)
        b.check_rows()


def test_zero_counts_and_empty_calls(hip):
    b = Both(hip, 2, 64)
    b.append([0, 1], [0, 0], b.rows(0), b.rows(0))
    assert [b.gpu.length(s) for s in (0, 1)] == [0, 0]
    b.append([2, 0, 1], [0, 5, 0])
    k, v = b.gpu.read([0, 2], [2, 0], [0, 0])
    assert k.shape == v.shape == (0, 128)
    out = b.gpu.attention(b.hip.Tensor.from_numpy(np.zeros((0, 4 * 64), np.float32)), [0, 1], [0, 0])
    assert out.shape == (0, 256) and out.data().size == 0
    b.check_attention(4, [1, 0, 2], [0, 3, 0])


def test_read_ranges(hip):
    b = Both(hip, 3, 64, page=64)
    b.append([0, 1], [100, 65])
    for starts, counts in [([0, 0], [1, 65]), ([31, 64], [2, 1]), ([99, 10], [1, 0]), ([33, 1], [64, 63])]:
        for g, want in zip(b.gpu.read([0, 1], starts, counts), b.ref.read([0, 1], starts, counts)):
            np.testing.assert_array_equal(g.data(), want.astype(np.float32))


def test_truncate_and_append_again(hip):
    """Refused drafts are cut off and overwritten; a block begun again starts
    with a scale of its own, one that is not keeps what it had."""
    b = Both(hip, 2, 128)
    b.append([0, 1], [40, 32])
    b.append([0, 1], [6, 1], b.rows(7, 50.0), b.rows(7, 50.0))
    b.gpu.truncate([1, 0], [32, 41])
    b.ref.truncate([1, 0], [32, 41])
    b.append([0, 1], [3, 2], b.rows(5, 0.1), b.rows(5, 0.1))
    b.check_rows()
    b.check_attention(4, [0, 1], [3, 2])


def test_released_pages_serve_another_sequence(hip):
    b = Both(hip, 1, 64, pages=4, seqs=3, max_seq=128)
    b.append([0], [100])
    b.gpu.release(0)
    del b.ref.slots[0]
    assert b.gpu.length(0) == 0
    b.free, b.mapped[0] = [0, 1, 2, 3], 0
    b.append([2, 0], [70, 20])
    b.check_rows()
    b.check_attention(2, [0, 2], [1, 1])


@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 64), (8, 8, 64), (32, 8, 64), (16, 1, 64), (3, 3, 128), (8, 2, 128),
                                       (64, 8, 128), (20, 1, 128), (40, 1, 64)])
@pytest.mark.parametrize("lens", [[1], [2, 33], [64, 31, 65], [257, 1, 128, 700]])
def test_attention_single_tokens(hip, nq, nkv, hd, lens):
    b = Both(hip, nkv, hd, seqs=len(lens), max_seq=701, seed=len(lens))
    b.append(list(range(len(lens))), lens)
    b.check_attention(nq, list(range(len(lens)))[::-1], [1] * len(lens))


@pytest.mark.parametrize("nq,nkv,hd,page", [(4, 2, 64, 32), (32, 8, 64, 64), (5, 1, 64, 32), (2, 2, 128, 128), (8, 1, 128, 32),
                                            (12, 2, 128, 64)])
@pytest.mark.parametrize("lens,counts", [([5], [5]), ([40, 9], [3, 9]), ([33, 64, 70], [32, 1, 17]), ([300], [7]),
                                         ([130, 200], [130, 60])])
def test_attention_several_rows(hip, nq, nkv, hd, page, lens, counts):
    """Drafts and prompts: rows see the positions up to their own."""
    b = Both(hip, nkv, hd, page, seqs=len(lens), max_seq=320, seed=sum(counts))
    b.append(list(range(len(lens))), lens)
    b.check_attention(nq, list(range(len(lens))), counts)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [96, 97, 130, 300])
def test_attention_mixed_batch(hip, hd, n):
    """A prompt, drafts and single tokens in one call, over many sequences: as many
    as a launch's own arguments hold (96), and more."""
    b = Both(hip, 2, hd, seqs=n, max_seq=200, seed=3)
    lens = [1 + (37 * i) % 90 for i in range(n)]
    lens[7], lens[60] = 150, 120
    b.append(list(range(n)), lens)
    counts = [1 + i % 3 if lens[i] >= 3 else 1 for i in range(n)]
    counts[7], counts[60], counts[5] = 80, 1, 0
    b.check_attention(4, list(range(n)), counts)
    b.check_rows()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_scores_of_any_size(hip, hd):
    """Peaked softmaxes, equal scores, and a query of zeros."""
    b = Both(hip, 1, hd, max_seq=400)
    b.append([0], [333])
    for scale in (0.0, 1e-6, 1.0, 30.0, 1e4):
        b.check_attention(2, [0], [2], scale)


@pytest.mark.parametrize("scale", [1e6, 1e8, 1e9, 1e20, 1e33, -1e9, -1e20, -1e33])
@pytest.mark.parametrize("n", [2, 600])
def test_attention_scores_past_f32s_steps(hip, n, scale):
    """Scores whose last place in f32 is a factor of e and more, all of one sign:
    which of the nearly greatest win is open, but the result is a weighted mean of
    the values that a row sees (off by the roundings of the bound), never NaN."""
    b = Both(hip, 1, 128, max_seq=1300, rope=None)
    b.append([0], [1300], np.abs(b.rows(1300)), None)
    q = np.abs(b.rng.standard_normal((n, 4 * 128))).astype(np.float32) * np.float32(scale)
    got = b.gpu.attention(hip.Tensor.from_numpy(q), [0], [n]).data().reshape(n, 4, 128)
    v = b.ref.values(0)[1][:, 0]
    room = (1300 + 64) * 2.0 ** -24 * np.abs(v).max()
    assert (got <= v.max(0) + room).all() and (got >= v.min(0) - room).all()
    # one position far above the others: its value alone
    k = np.full((65, 128), 1.0, np.float32)
    k[40] = 2.0 if scale > 0 else 0.5
    b.append([1], [65], k, b.rows(65))
    got = b.gpu.attention(hip.Tensor.from_numpy(q[:2]), [1], [2]).data().reshape(2, 4, 128)
    v = b.ref.values(1)[1][40, 0]
    np.testing.assert_allclose(got, np.broadcast_to(v, got.shape), rtol=64 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("big,small", [(2.0 ** 60, 2.0 ** -60), (2.0 ** 15, 2.0 ** -15)])
def test_attention_values_of_any_size(hip, hd, big, small):
    """Blocks whose values differ by up to 2^120: those that the softmax leaves
    out must not drown the others."""
    b = Both(hip, 1, hd, max_seq=400, rope=None)
    k, v = b.rows(256), b.rows(256)
    # the first and third 64 positions score far below the others and hold huge values
    q = b.rng.standard_normal((1, hd)).astype(np.float32)
    k += np.where((np.arange(256) // 64 % 2 == 0)[:, None], -40.0, 0.0).astype(np.float32) * q / np.abs(q).max()
    v *= np.where((np.arange(256) // 64 % 2 == 0)[:, None], big, small).astype(np.float32)
    b.append([0], [256], k, v)
    for scale in (1.0, 8.0):
        x = (q * scale).astype(np.float32)
        got = b.gpu.attention(hip.Tensor.from_numpy(x), [0], [1]).data()
        within(got, *b.ref.attention(x, [0], [1]))


def test_attention_rows_that_are_not_finite(hip):
    """A query row with a NaN or an infinity gives NaN in its own head only; the
    others are as without it."""
    b = Both(hip, 2, 128)
    b.append([0, 1], [90, 40])
    q = b.rng.standard_normal((4, 4 * 128)).astype(np.float32)
    clean = b.gpu.attention(hip.Tensor.from_numpy(q), [0, 1], [3, 1]).data()
    q[1, 130], q[3, 511] = np.nan, np.inf
    got = b.gpu.attention(hip.Tensor.from_numpy(q), [0, 1], [3, 1]).data()
    bad = np.zeros((4, 4, 128), bool)
    bad[1, 1] = bad[3, 3] = True
    bad = bad.reshape(4, 512)
    assert np.isnan(got[bad]).all()
    np.testing.assert_array_equal(got[~bad], clean[~bad])


def test_stale_rows_are_not_seen(hip):
    """What an earlier sequence left behind the length, NaN-free or not, does not
    reach the result."""
    b = Both(hip, 1, 64, pages=2, seqs=2, max_seq=64)
    b.append([0], [64], b.rows(64, 1e30), b.rows(64, 1e30))
    b.gpu.release(0)
    b.ref.slots.clear()
    b.free, b.mapped = [1, 0], [0, 0]
    b.append([1], [33])
    b.check_rows([1])
    b.check_attention(2, [1], [1])


def test_offsets_past_32_bits(hip):
    """Pages more than 4 GiB into the pool."""
    pages = 40000  # 8 heads x 2 x 64 positions x 128 dims: 128 KiB each
    c = Both(hip, 8, 128, page=64, pages=pages, seqs=2, max_seq=512)
    c.free = [p for i in range(8) for p in (i, pages - 1 - i)]  # taken from the back
    c.append([0, 1], [300, 70])
    c.append([1, 0], [1, 2])
    c.check_rows()
    c.check_attention(16, [0, 1], [2, 1])


@pytest.mark.parametrize("length,counts", [(5000, [1]), (5000, [6]), (3000, [1000])])
def test_attention_long(hip, length, counts):
    """A long sequence, its splits and tiles, against a sample of the rows in 64 bits."""
    nq, nkv, hd = 8, 2, 128
    b = Both(hip, nkv, hd, page=128, seqs=1, max_seq=5120)
    b.append([0], [length])
    q = b.rng.standard_normal((counts[0], nq * hd)).astype(np.float32)
    got = b.gpu.attention(hip.Tensor.from_numpy(q), [0], counts).data()
    # the reference's rows one at a time: it takes the sequence as ending there
    for i in sorted({0, counts[0] // 2, counts[0] - 1}):
        b.ref.truncate([0], [length - counts[0] + i + 1])
        within(got[i:i + 1], *b.ref.attention(q[i:i + 1], [0], [1]))


def check_sample(b, nq, slots, counts, scale=1.0):
    """Attention of many rows, a few of each sequence against the reference."""
    q = (b.rng.standard_normal((int(np.sum(counts)), nq * b.hd)) * scale).astype(np.float32)
    got = b.gpu.attention(b.hip.Tensor.from_numpy(q), slots, counts).data()
    assert np.isfinite(got).all()
    row = 0
    for s, n in zip(slots, counts):
        length = b.gpu.length(s)
        # the reference's rows one at a time: it takes the sequence as ending there
        for i in sorted({0, n // 3, n - 1} & set(range(n))):
            b.ref.truncate([s], [length - n + i + 1])
            within(got[row + i:row + i + 1], *b.ref.attention(q[row + i:row + i + 1], [s], [1]))
        b.ref.truncate([s], [length])
        row += n
    return q, got


# (query heads, KV heads, head_dim, page, lengths, rows): enough columns for the kernel
# of 64 of them, 96 for each of 256 CUs, in whole tiles and with a rest, behind earlier
# positions and from the first on
MANY = [(32, 8, 128, 64, [1000], [800]), (32, 8, 128, 32, [777], [777]), (16, 16, 64, 128, [1601], [1600]),
        (64, 2, 128, 256, [451], [387]), (32, 8, 64, 32, [500, 1, 400, 333], [500, 1, 400, 16]),
        (32, 8, 128, 64, [300, 700, 65, 63, 1025], [300, 500, 65, 0, 1])]


@pytest.mark.parametrize("nq,nkv,hd,page,lens,counts", MANY)
def test_attention_many_columns(hip, nq, nkv, hd, page, lens, counts):
    b = Both(hip, nkv, hd, page=page, max_seq=2048)
    slots = list(range(len(lens)))[::-1]
    b.append(slots, lens)
    check_sample(b, nq, slots, counts)


def test_tested_calls_take_their_kernels(hip):
    """On this device's CUs, whose number the plan goes by."""
    from test_paged import check_tested_plans
    check_tested_plans(hip.num_cus())


def test_attention_many_columns_scores_of_any_size(hip):
    """As for few columns: zeros, peaked softmaxes, one sign past f32's steps."""
    b = Both(hip, 8, 128, max_seq=1024, rope=None)
    b.append([0], [850], np.abs(b.rows(850)), None)
    for scale in (0.0, 30.0, 1e4):
        check_sample(b, 32, [0], [800], scale)
    v = b.ref.values(0)[1]
    room = (1024 + 64) * 2.0 ** -24 * np.abs(v).max()
    for scale in (1e6, 1e9, 1e33, -1e9, -1e33):
        q = np.abs(b.rng.standard_normal((800, 32 * 128))).astype(np.float32) * np.float32(scale)
        got = b.gpu.attention(hip.Tensor.from_numpy(q), [0], [800]).data().reshape(800, 8, 4, 128)
        assert (got <= v.max(0)[None, :, None] + room).all() and (got >= v.min(0)[None, :, None] - room).all()


def test_attention_many_columns_not_finite_and_same_bits(hip):
    b = Both(hip, 8, 128, max_seq=1024)
    b.append([0, 1], [850, 40])
    q, clean = check_sample(b, 32, [0, 1], [800, 1])
    np.testing.assert_array_equal(b.gpu.attention(hip.Tensor.from_numpy(q), [0, 1], [800, 1]).data(), clean)
    bad = np.zeros((801, 32, 128), bool)
    for row, head, x in ((0, 3, np.nan), (517, 31, np.inf), (799, 0, -np.inf), (800, 7, np.nan)):
        q[row, 128 * head + 5] = x
        bad[row, head] = True
    bad = bad.reshape(801, -1)
    got = b.gpu.attention(hip.Tensor.from_numpy(q), [0, 1], [800, 1]).data()
    assert np.isnan(got[bad]).all()
    np.testing.assert_array_equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("lens,counts", [([9000] + [40] * 70, [1] * 71), ([9000, 300, 300], [16, 300, 300])])
def test_attention_one_sequence_outlasts_the_others(hip, lens, counts):
    """A batch that fills the chip, with one long sequence whose tiles are split."""
    b = Both(hip, 8, 64, seqs=len(lens), max_seq=9216)
    slots = list(range(len(lens)))
    b.append(slots, lens)
    check_sample(b, 64, slots, counts)


def test_same_call_same_bits(hip):
    """No result depends on the order workgroups end in."""
    b = Both(hip, 8, 128, seqs=4, max_seq=1000)
    b.append([0, 1, 2, 3], [999, 500, 1, 64])
    q = hip.Tensor.from_numpy(b.rng.standard_normal((7, 32 * 128)).astype(np.float32))
    first = b.gpu.attention(q, [0, 1, 2, 3], [3, 2, 1, 1]).data()
    for _ in range(5):
        np.testing.assert_array_equal(b.gpu.attention(q, [0, 1, 2, 3], [3, 2, 1, 1]).data(), first)


def test_two_caches_from_two_threads(hip):
    """Calls of several host threads are taken one after the other."""
    caches = [Both(hip, 2, 64, max_seq=256, seed=i) for i in range(2)]
    failed = []

    def work(c):
        try:
            for _ in range(20):
                c.append([0, 1], [3, 1])
            c.check_rows()
            c.check_attention(4, [0, 1], [2, 1])
        except BaseException as e:  # noqa: BLE001 - reported by the main thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=(c,)) for c in caches]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]


def test_tensor_shapes_refused(hip):
    b = Both(hip, 2, 64)
    b.append([0], [10])
    T = hip.Tensor.from_numpy
    ok = np.zeros((2, 128), np.float32)
    for k, v in [(ok[:1], ok), (ok, ok[:1]), (np.zeros((2, 64), np.float32), ok), (np.zeros(256, np.float32), ok)]:
        with pytest.raises(hip.LlmrsError) as e:
            b.gpu.append(T(k), T(v), [0], [2])
        assert e.value.code == hip.E_INVALID
    for q in (np.zeros((2, 64), np.float32), np.zeros((1, 128), np.float32), np.zeros((2, 192), np.float32), np.zeros(256, np.float32)):
        with pytest.raises(hip.LlmrsError) as e:
            b.gpu.attention(T(q), [0], [2])
        assert e.value.code == hip.E_INVALID
    codes = hip.Tensor.from_q8_0(np.zeros((2, 128), np.int8), np.zeros((2, 4), np.float32), 2, 128)
    for call in (lambda: b.gpu.append(codes, codes, [0], [2]), lambda: b.gpu.attention(codes, [0], [2])):
        with pytest.raises(hip.LlmrsError) as e:
            call()
        assert e.value.code == hip.E_DTYPE
    assert b.gpu.length(0) == 10
    b.check_rows()


# ---- verification of drafts ----------------------------------------------------
def probabilities(rng, rows, vocab, temperature=2.0):
    x = rng.standard_normal((rows, vocab)) * temperature
    p = np.exp(x - x.max(1, keepdims=True))
    return (p / p.sum(1, keepdims=True)).astype(np.float32)


def check_verify(hip, target, ids, counts, accept, draw, draft=None):
    T = hip.Tensor.from_numpy
    got = hip.verify_drafts(T(target), ids, counts, accept, draw, draft=None if draft is None else T(draft))
    want = ref.verify(target, ids, counts, accept, draw, draft)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    return got


def uniform(rng, n):
    return (rng.integers(0, 1 << 24, n) / np.float32(1 << 24)).astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 7, 255, 2047, 2048, 2049, 32003, 128256])
@pytest.mark.parametrize("given", [True, False])
@pytest.mark.parametrize("counts", [[0], [1], [3, 0, 5, 1], [64, 2]])
def test_verify(hip, vocab, given, counts):
    rng = np.random.default_rng(vocab + len(counts))
    n = sum(counts)
    target = probabilities(rng, n + len(counts), vocab)
    rows = [j for i, g in enumerate(counts) for j in range(sum(counts[:i]) + i, sum(counts[:i]) + i + g)]
    draft = None
    if given:
        noisy = target[rows] * np.exp(0.3 * rng.standard_normal((n, vocab)))
        draft = (noisy / noisy.sum(1, keepdims=True)).astype(np.float32) if n else np.zeros((0, vocab), np.float32)
    source = draft if given else target[rows]
    ids = [int(rng.choice(vocab, p=r.astype(np.float64) / r.sum(dtype=np.float64))) for r in source]
    check_verify(hip, target, ids, counts, uniform(rng, n), uniform(rng, len(counts)), draft)


@pytest.mark.parametrize("given", [True, False])
def test_verify_vocabularies_past_a_wave_of_sums(hip, given):
    """More than 512 slices of 512 ids; draws in each part."""
    rng = np.random.default_rng(8)
    V, counts = 512 * 1024 + 77, [1, 0, 2]
    target = probabilities(rng, 6, V)
    draft = probabilities(rng, 3, V) if given else None
    ids = rng.integers(0, V, 3)
    for x in (0.0, 0.2, 0.51, 0.75, 0.999, 1.0 - 2.0 ** -24):
        check_verify(hip, target, ids, counts, uniform(rng, 3), np.full(3, x, np.float32), draft)
        check_verify(hip, target, ids, counts, np.zeros(3, np.float32), np.full(3, x, np.float32), draft)


def test_verify_answers_past_the_host_buffer(hip):
    """So many sequences that the answer comes through device memory."""
    rng = np.random.default_rng(9)
    n, V = 44000, 5
    counts = rng.integers(0, 2, n).astype(np.int32)
    rows = int(counts.sum())
    target = probabilities(rng, rows + n, V, 1.0)
    check_verify(hip, target, rng.integers(0, V, rows), counts, uniform(rng, rows), uniform(rng, n))


def test_verify_many_sequences(hip):
    rng = np.random.default_rng(5)
    counts = [int(c) for c in rng.integers(0, 7, 300)]
    n, V = sum(counts), 1009
    target, draft = probabilities(rng, n + 300, V, 1.0), probabilities(rng, n, V, 1.0)
    accepted, _ = check_verify(hip, target, rng.integers(0, V, n), counts, uniform(rng, n), uniform(rng, 300), draft)
    assert accepted.max() > 1


def test_verify_borders(hip):
    """Equal rows leave nothing to draw from but the target; an id without draft
    probability is taken if the target has it; running sums that meet the draw exactly go
    on to the next id; the draws 0 and the largest below 1."""
    V = 8
    p = np.array([0.25, 0.0, 0.125, 0.125, 0.5, 0.0, 0.0, 0.0], np.float32)
    q = np.array([0.5, 0.0, 0.0, 0.0, 0.25, 0.25, 0.0, 0.0], np.float32)
    top = np.float32(1.0 - 2.0 ** -24)
    for draw in (0.0, 0.125, 0.25, 0.375, 0.5, 0.9, top):
        for ids, accept in [([0], 0.5), ([0], 0.49), ([0], 1.0), ([2], 0.0), ([2], 1.0), ([1], 0.0), ([4], 1.0), ([5], 0.0)]:
            for d in (q, p, None):
                check_verify(hip, np.stack([p, q]), ids, [1], np.float32([accept]), np.float32([draw]),
                             None if d is None else d[None])


def lanes_scanned(v):
    """Running sums of 64 numbers in 64 bits, in the order in which a wave forms them:
    by steps of 1, 2, 4 and 8 within each 16, then the 16s' totals."""
    v = np.asarray(v, np.float64).reshape(4, 16)
    for step in (1, 2, 4, 8):
        v = v + np.concatenate((np.zeros((4, step)), v[:, :-step]), 1)
    v = v + np.array([0.0, v[0, 15], 0.0, v[2, 15]])[:, None]
    return (v + np.array([0.0, 0.0, v[1, 15], v[1, 15]])[:, None]).reshape(64)


def test_verify_draws_nothing_from_empty_slices(hip):
    """Rows with an id in few of the sums' slices, as top-k leaves them.  The running sum
    over the slices is formed as a tree, so behind an empty one it may be a last place
    larger than before it; a draw that meets the sum there takes an id that has something.
    64 numbers of one sign in whatever order are off by up to 63 roundings of their sum, on
    either side of the comparison: the ids whose exact running sum reaches half of the total
    less that, while the one before them does not exceed half and that."""
    rng = np.random.default_rng(17)
    rows, at = [], []
    while len(rows) < 12:
        n = int(rng.integers(3, 12))
        slices = np.sort(rng.choice(30, n, replace=False))
        w = np.zeros(32, np.float32)
        w[slices] = (10.0 ** rng.uniform(-16, 0, n)).astype(np.float32)
        sums = np.concatenate((w, w)).astype(np.float64)  # both halves alike: half of the total ends the first
        running = lanes_scanned(sums)
        if sums[np.nonzero(running > 0.5 * running[63])[0][0]] > 0:
            continue
        row, ids = np.zeros(64 * 512, np.float32), rng.integers(0, 512, 64) + 512 * np.arange(64)
        row[ids] = sums
        rows.append(row)
        exact = [math.fsum(sums[:i]) for i in range(65)]
        room = 2 * 64 * 2.0 ** -53 * exact[64]
        at.append({int(ids[i]) for i in range(64) if sums[i] > 0 and exact[i + 1] >= exact[64] / 2 - room and exact[i] <= exact[64] / 2 + room})
        assert {int(ids[slices[-1]]), int(ids[32 + slices[0]])} <= at[-1]
    target = np.stack(rows)
    # after other slices as well, past the sums that a wave holds at once
    for before in (0, 512 * 512, 512 * 512 * 3):
        wide = np.concatenate((np.zeros((len(rows), before), np.float32), target), 1)
        _, tokens = hip.verify_drafts(hip.Tensor.from_numpy(wide), [], [0] * len(rows), [], [0.5] * len(rows))
        for i, ids in enumerate(at):
            assert tokens[i, 0] - before in ids, (i, before, tokens[i, 0], ids)


def test_verify_odd_rows(hip):
    """Rows of zeros, negative entries and NaN: nothing negative or NaN is drawn."""
    V = 4099
    p = np.zeros((2, V), np.float32)
    _, tokens = check_verify(hip, p, [3], [1], np.float32([0.5]), np.float32([0.5]), np.ones((1, V), np.float32))
    assert tokens[0, 0] == V - 1
    p[:, 4000], p[:, 7], p[:, 9] = 0.25, np.nan, -3.0
    for draw in (0.0, 0.99):
        accepted, tokens = check_verify(hip, p, [7], [1], np.float32([0.0]), np.float32([draw]))
        assert accepted[0] == 0 and tokens[0].tolist() == [4000, -1]


def test_verify_draws_of_64_bits(hip):
    """A number below 1 that f32 has no nearer neighbour for than 1 is a draw all the same."""
    p = hip.Tensor.from_numpy(np.full((2, 6), 1 / 6, np.float32))
    top = 1.0 - 2.0 ** -53
    for draw in ([top, 0.5], np.array([top, 0.5]), np.array([[top], [0.5]])):
        accepted, tokens = hip.verify_drafts(p, [], [0, 0], [], draw)
        assert accepted.tolist() == [0, 0] and tokens[:, 0].tolist() == [5, 3]
    for draw in ([1.0, 0.5], np.array([1.0, 0.5]), np.float32([1.0, 0.5]), [np.nan, 0.5], [1.0 + 2.0 ** -30, 0.5]):
        with pytest.raises(hip.LlmrsError) as e:
            hip.verify_drafts(p, [], [0, 0], [], draw)
        assert e.value.code == hip.E_INVALID


def test_verify_refusals(hip):
    T = hip.Tensor.from_numpy
    p, q = np.full((3, 5), 0.2, np.float32), np.full((2, 5), 0.2, np.float32)
    good = dict(target=p, ids=[1, 2], counts=[2], accept=[0.5, 0.5], draw=[0.5], draft=q)
    for code, kw in [(hip.E_RANGE, {"ids": [1, 5]}), (hip.E_RANGE, {"ids": [-1, 2]}), (hip.E_INVALID, {"accept": [0.5, 1.5]}),
                     (hip.E_INVALID, {"accept": [np.nan, 0.5]}), (hip.E_INVALID, {"draw": [1.0]}), (hip.E_INVALID, {"draw": [-0.1]}),
                     (hip.E_INVALID, {"target": p[:2]}), (hip.E_INVALID, {"draft": q[:1]}), (hip.E_INVALID, {"draft": q[:, :4].copy()}),
                     (hip.E_RANGE, {"ids": [1] * 65, "accept": [0.5] * 65, "counts": [65]})]:
        a = good | kw
        with pytest.raises(hip.LlmrsError) as e:
            hip.verify_drafts(T(a["target"]), a["ids"], a["counts"], a["accept"], a["draw"], draft=T(a["draft"]))
        assert e.value.code == code, (kw, e.value)


# ---- the operators together ------------------------------------------------------
def test_drafted_decoding(hip):
    """A one-layer model served with drafts looked up in its own text: each round
    appends the drafts' keys and values, attends, verifies and cuts the refused ones off.
    The text is that of decoding token by token with the same target rows' draws."""
    rng = np.random.default_rng(11)
    V, nq, nkv, hd = 96, 4, 2, 64
    H = nq * hd
    be = hip.HipBackend()
    T = hip.Tensor.from_numpy
    W = {n: (rng.standard_normal((o, H)) / 16).astype(np.float32) for n, o in
         (("q", H), ("k", nkv * hd), ("v", nkv * hd), ("o", H), ("head", V))}
    W["head"] *= 24
    D = {n: T(w) for n, w in W.items()}
    emb = rng.standard_normal((V, H)).astype(np.float32)
    both = Both(hip, nkv, hd, seqs=2, max_seq=256)
    c = both.gpu
    text = [[int(t) for t in rng.integers(0, V, 20)] * 2 for _ in range(2)]

    def forward(slots, tokens):
        """Probabilities after each token, on the GPU, and in 64 bits."""
        flat = [t for ts in tokens for t in ts]
        counts = [len(ts) for ts in tokens]
        x = T(emb[flat])
        k, v, q = (be.matmul_transposed(x, D[n]) for n in "kvq")
        both.room(slots, counts)
        c.append(k, v, slots, counts)
        both.ref.append(k.data(), v.data(), slots, counts)
        ctx = c.attention(q, slots, counts)
        within(ctx.data(), *both.ref.attention(q.data(), slots, counts))
        h = be.matmul_transposed(ctx, D["o"])
        be.add_assign(h, x)
        return be.softmax(be.matmul_transposed(h, D["head"]))

    slots = [1, 0]
    forward(slots, [text[s][:-1] for s in slots])
    taken = 0
    for _ in range(12):
        drafts = []
        for s in slots:  # what followed the last token before, up to four ids
            at = [i for i in range(len(text[s]) - 1) if text[s][i] == text[s][-1]]
            drafts.append(text[s][at[-1] + 1:at[-1] + 5] if at else [])
        p = forward(slots, [[text[s][-1]] + d for s, d in zip(slots, drafts)])
        ids = [t for d in drafts for t in d]
        counts = [len(d) for d in drafts]
        accept, draw = uniform(rng, len(ids)), uniform(rng, 2)
        accepted, tokens = hip.verify_drafts(p, ids, counts, accept, draw)
        want = ref.verify(p.data(), ids, counts, accept, draw)
        np.testing.assert_array_equal(accepted, want[0])
        np.testing.assert_array_equal(tokens, want[1])
        for i, s in enumerate(slots):
            text[s] += [int(t) for t in tokens[i, :accepted[i] + 1]]
        lengths = [len(text[s]) - 1 for s in slots]
        c.truncate(slots, lengths)
        both.ref.truncate(slots, lengths)
        taken += int(accepted.sum())
    assert [c.length(s) for s in slots] == [len(text[s]) - 1 for s in slots]
    assert taken > 0
    both.check_rows()


DEVICE_ARRAYS = """
import torch                     # before the library: they share one HIP runtime
import numpy as np
import llmrs_hip as hip
hip.init(0)
x = torch.arange(24, dtype=torch.float32, device="cuda").reshape(2, 3, 4)
t = hip.Tensor.from_device(x)
x.zero_()
assert t.shape == (2, 3, 4)
np.testing.assert_array_equal(t.data().ravel(), np.arange(24, dtype=np.float32))
hip.HipBackend().add_assign(t, t)
hip.sync()
y = torch.as_tensor(t, device="cuda")
assert y.data_ptr() == t.__cuda_array_interface__["data"][0]
np.testing.assert_array_equal(y.cpu().numpy().ravel(), 2 * np.arange(24, dtype=np.float32))
# written on a stream of its own and not waited for
side = torch.cuda.Stream()
with torch.cuda.stream(side):
    z = torch.zeros(1 << 24, device="cuda")
    for _ in range(20):
        z += 1
np.testing.assert_array_equal(hip.Tensor.from_device(z).data()[::1 << 16], 20.0)
for bad in (x.permute(2, 0, 1), x.double(), x.cpu()):
    try:
        hip.Tensor.from_device(bad)
    except hip.LlmrsError as e:
        assert e.code in (hip.E_INVALID, hip.E_DTYPE)
    else:
        raise AssertionError("not refused")
assert hip.Tensor.from_device(torch.zeros(0, 4, device="cuda")).shape == (0, 4)
assert tuple(torch.as_tensor(hip.Tensor.zeros((0, 3)), device="cuda").shape) == (0, 3)
torch.cuda.synchronize()
print("arrays ok")
"""


def test_device_arrays():
    """Tensors from and to another library's device memory, in a process that
    loads that library first."""
    pytest.importorskip("torch")
    pkg = Path(__file__).resolve().parent.parent / "llm.rs_amd"
    got = subprocess.run([sys.executable, "-c", DEVICE_ARRAYS], capture_output=True, text=True, timeout=100,
                         env=dict(os.environ, PYTHONPATH=str(pkg)))
    assert got.stdout.strip() == "arrays ok", got.stderr[-2000:]
