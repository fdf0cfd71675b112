"""The paged cache, its attention and the verification of drafts in plain numpy,
64 bits, from their definitions."""
from __future__ import annotations

import math

import numpy as np

BLOCK = 32
E_MIN, E_MAX = -100, 121
TOP = np.ldexp(127.0, E_MAX)


def needed(top):
    """The smallest exponent in range with top <= 127 * 2^e."""
    for e in range(E_MIN, E_MAX + 1):
        if top <= math.ldexp(127.0, e):
            return e
    return E_MAX


def turned(x, cos, sin, start):
    """Rows [rows][heads][hd] rotated to positions start.."""
    h = x.shape[-1] // 2
    c, s = (t[start:start + x.shape[0], None].astype(np.float64) for t in (cos, sin))
    return np.concatenate((x[..., :h] * c - x[..., h:] * s, x[..., :h] * s + x[..., h:] * c), -1)


class RefCache:
    """Each slot's codes and exponents, [K, V][positions][heads][hd] and [block][heads]."""

    def __init__(self, nkv, hd, rope=None):
        self.nkv, self.hd, self.rope = nkv, hd, rope
        self.slots = {}

    def _slot(self, s):
        empty = [np.zeros((0, self.nkv, self.hd)) for _ in "kv"]
        return self.slots.setdefault(s, {"codes": empty, "exps": [{}, {}], "len": 0})

    def append(self, k, v, slots, counts, rotate=True):
        row = 0
        for s, n in zip(slots, counts):
            st = self._slot(s)
            p = st["len"]
            for which, x in enumerate((k, v)):
                x = x[row:row + n].astype(np.float64).reshape(n, self.nkv, self.hd)
                with np.errstate(invalid="ignore"):
                    if which == 0 and rotate and self.rope is not None:
                        x = turned(x, *self.rope, p)
                x = np.clip(np.where(np.isnan(x), 0.0, x), -TOP, TOP)
                codes = np.concatenate((st["codes"][which][:p], np.zeros_like(x)))
                for b in range(p // BLOCK, (p + n - 1) // BLOCK + 1 if n else 0):
                    lo, hi = max(p, b * BLOCK), min(p + n, (b + 1) * BLOCK)
                    for h in range(self.nkv):
                        new = x[lo - p:hi - p, h]
                        e = needed(np.abs(new).max())
                        if lo > b * BLOCK:
                            was = st["exps"][which][b, h]
                            e = max(e, was)
                            old = slice(b * BLOCK, lo)
                            codes[old, h] = np.rint(np.ldexp(codes[old, h], was - e))
                        st["exps"][which][b, h] = e
                        codes[lo:hi, h] = np.rint(np.ldexp(new, -e))
                st["codes"][which] = codes
            st["len"] = p + n
            row += n

    def truncate(self, slots, lengths):
        for s, n in zip(slots, lengths):
            self._slot(s)["len"] = n

    def values(self, s):
        """K and V of a slot, [positions][heads][hd]."""
        st = self._slot(s)
        out = []
        for which in range(2):
            x = st["codes"][which][:st["len"]].copy()
            for b in range(-(-st["len"] // BLOCK)):
                for h in range(self.nkv):
                    rows = slice(b * BLOCK, (b + 1) * BLOCK)
                    x[rows, h] = np.ldexp(x[rows, h], st["exps"][which][b, h])
            out.append(x)
        return out

    def read(self, slots, starts, counts):
        got = [[], []]
        for s, a, n in zip(slots, starts, counts):
            for which, x in enumerate(self.values(s)):
                got[which].append(x[a:a + n].reshape(n, self.nkv * self.hd))
        return tuple(np.concatenate(g) for g in got)

    def attention(self, q, slots, counts):
        """The attention, and a bound on how far a computation in f32 may be off.

        delta bounds the relative error of an unnormalised weight: q rotated in
        f32 (3 roundings) and rounded to 22 bits below its row's largest value, the
        score's f32 sum, product and scale (8 roundings of its size), log2(e) and exp2
        (4 roundings).  The sum of the lowest of q's three bytes times the codes counts in
        whole steps of 2^8: q's integer is at most 2^22, so a step is 2^8 / 2^21 = 2^-13 of
        q's largest value (an integer in (2^21, 2^22]) times one step of K.  A sum of n weighted values in f32, in whatever order, adds n
        roundings of sum p |v|; the weights are split in 22 bits, and joining and dividing
        add a few.  A weight p * 2^e is held as f16 hi + lo with the largest at 2^14: where
        lo has f16's smallest step, 2^-24, it is off by up to half of that, 2^-25 / 2^14 =
        2^-39 of the largest weight, times the code."""
        nq = q.shape[1] // self.hd
        rep, u = nq // self.nkv, 2.0 ** -24
        out, tol, row = [], [], 0
        for s, n in zip(slots, counts):
            k, v = self.values(s)
            length, (kexps, exps) = k.shape[0], self._slot(s)["exps"]
            x = q[row:row + n].astype(np.float64).reshape(n, nq, self.hd)
            row += n
            if self.rope is not None:
                x = turned(x, *self.rope, length - n)
            o, t = np.empty((n, nq, self.hd)), np.empty((n, nq, self.hd))
            for i in range(n):
                seen = length - n + i + 1
                for h in range(nq):
                    kk, vv = k[:seen, h // rep], v[:seen, h // rep]
                    sc = kk @ x[i, h] / math.sqrt(self.hd)
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    o[i, h] = p @ vv
                    size = np.abs(kk) @ np.abs(x[i, h]) / math.sqrt(self.hd)
                    kstep = np.ldexp(1.0, [kexps[j // BLOCK, h // rep] for j in range(seen)])
                    fixed = np.abs(x[i, h]).max() * (2.0 ** -23 * np.abs(kk).sum(1) + 2.0 ** -13 * kstep) / math.sqrt(self.hd)
                    delta = float(np.max(6 * u * size + 8 * u * np.abs(sc) + 8 * u * np.abs(sc - sc.max()) + fixed)) + 8 * u
                    step = np.ldexp(1.0, [exps[j // BLOCK, h // rep] for j in range(seen)])
                    floor = 2.0 ** -39 * np.max(p * step) * (np.abs(vv) / step[:, None]).sum(0)
                    t[i, h] = (2 * delta + (seen + 32) * u) * (p @ np.abs(vv)) + floor + 1e-37
            out.append(o.reshape(n, nq * self.hd))
            tol.append(t.reshape(n, nq * self.hd))
        return np.concatenate(out), np.concatenate(tol)


def rope_tables(rows, hd, theta=500000.0):
    a = np.arange(rows)[:, None] * theta ** (-2.0 * np.arange(hd // 2) / hd)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def verify(target, ids, counts, accept, draw, draft=None):
    """(accepted, tokens) of drafts against the target."""
    t0 = d0 = 0
    accepted, tokens = [], []
    width = max(counts) + 1
    for i, g in enumerate(counts):
        k = 0
        while k < g:
            q = 1.0 if draft is None else float(draft[d0 + k, ids[d0 + k]])
            if not float(accept[d0 + k]) * q < float(target[t0 + k, ids[d0 + k]]):
                break
            k += 1
        w = target[t0 + k].astype(np.float64)
        if k < g:
            q = draft[d0 + k].astype(np.float64) if draft is not None else (np.arange(w.size) == ids[d0 + k]) * 1.0
            left = w - q
        else:
            left = w
        left, w = (np.where(x > 0, x, 0.0) for x in (left, w))
        if not left.sum() > 0:
            left = w
        c = np.cumsum(left)
        over = np.nonzero(c > float(draw[i]) * c[-1])[0]
        accepted.append(k)
        tokens.append([*ids[d0:d0 + k], over[0] if over.size else w.size - 1] + [-1] * (width - 1 - k))
        t0, d0 = t0 + g + 1, d0 + g
    return np.array(accepted, np.int32), np.array(tokens, np.int32)
