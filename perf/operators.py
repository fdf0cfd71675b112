"""The operators of serving from a paged 8-bit key/value cache, as cases that can be timed.

``append``     new keys and values into the cache, keys rotated to their positions on
               the way (``HipPagedCache.append``), and what the touched blocks then hold
``attention``  new rows of several sequences over their cached positions
               (``HipPagedCache.attention``)
``verify``     drafted tokens against the target's probabilities, from given random
               numbers (``verify_drafts``)

``own`` selects the framework's operators; otherwise ``run`` computes them in
elementary torch operations.

The cache holds 8-bit codes with a power-of-two scale for each head and block of
32 positions: a value is code * 2^e, where e is the smallest exponent for which
the largest magnitude among the block's rows is at most 127 * 2^e.  Rows that
join a block may raise its exponent; the codes already there are then rounded to
the new step.
"""
from __future__ import annotations

import importlib
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False
DEV = "cuda" if torch.cuda.is_available() else "cpu"
BLOCK = 32                  # positions that share a scale
E_MIN, E_MAX = -100, 121    # range of the exponents
THETA = 500000.0

# name: (query heads, KV heads, head_dim)
HEADS = {
    "small": (4, 2, 64),
    "1b": (32, 8, 64),
    "8b": (32, 8, 128),
    "70b": (64, 8, 128),
    "one_kv": (16, 1, 64),
    "own_kv": (12, 12, 64),
}


def _cache(op, name, heads, page, seqs, rows, past):
    """`seqs` sequences, the first with `rows` new rows after `past` positions and the others with fewer."""
    return {"op": op, "name": name, "heads": heads, "page": page, "seqs": seqs, "rows": rows, "past": past}


def _verify(name, seqs, drafts, vocab, given):
    return {"op": "verify", "name": name, "seqs": seqs, "drafts": drafts, "vocab": vocab, "given": given}


def listed():
    return [
        # the smallest: one layer's new token of a single chat
        _cache("append", "append_1", "1b", 32, 1, 1, 700),
        # a decode step of a server's batch, contexts of different lengths
        _cache("append", "append_64", "8b", 64, 64, 1, 2049),
        # drafted tokens of sixteen requests, up to five each
        _cache("append", "append_draft_16", "8b", 32, 16, 5, 1000),
        # four long prompts admitted together
        _cache("append", "append_prompt_4", "8b", 128, 4, 2048, 0),
        # a decode step of a single chat on the small shape
        _cache("attention", "attend_1", "1b", 32, 1, 1, 512),
        # one question about a long document, the widest shape
        _cache("attention", "attend_1_long", "70b", 256, 1, 1, 32767),
        # a decode step of a server's batch
        _cache("attention", "attend_64", "8b", 64, 64, 1, 4000),
        # drafted tokens of sixteen requests looked at in one pass
        _cache("attention", "attend_draft_16", "70b", 32, 16, 5, 2100),
        # the largest: a prompt's second chunk
        _cache("attention", "attend_prompt", "8b", 128, 1, 2048, 2048),
        # one chat's drafts
        _verify("verify_1", 1, 4, 32000, True),
        # a batch's drafts over the full vocabulary
        _verify("verify_32", 32, 5, 128256, True),
        # drafts looked up in the text, which come without probabilities; an odd vocabulary
        _verify("verify_lookup_16", 16, 8, 32003, False),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "attention", "attention", "verify"])
    if op == "verify":
        c = _verify("", log_int(1, 48), rng.randint(1, 8), log_int(500, 128256), rng.random() < 0.7)
    else:
        heads, page = rng.choice(sorted(HEADS)), rng.choice([32, 64, 128, 256])
        kind = rng.choice(["decode", "draft", "prompt"])
        if kind == "prompt":
            seqs = rng.randint(1, 4)
            c = _cache(op, "", heads, page, seqs, log_int(16, 2048 if op == "append" else 1024 // seqs),
                       rng.choice([0, log_int(1, 2048)]))
        else:
            past = log_int(1, 8192)
            c = _cache(op, "", heads, page, log_int(1, max(1, min(96, 200000 // past))),
                       1 if kind == "decode" else rng.randint(2, 8), past)
    return {k: v for k, v in c.items() if k != "name"}


# ---- what a case says ----------------------------------------------------------
def _counts(case):
    """New rows of each sequence, and the positions before them."""
    n, r, p = case["seqs"], case["rows"], case["past"]
    rows = [r - r * i // (2 * n) for i in range(n)]
    past = [max(0, p - 3 * p * i // (4 * n) - 13 * i % 31) for i in range(n)]
    return rows, past


def _drafts(case):
    """Drafted tokens of each sequence: from `drafts` down to none."""
    g, n = case["drafts"], case["seqs"]
    return [g - (i * (g + 1) // n) for i in range(n)]


def work(case):
    if case["op"] == "verify":
        V, n = case["vocab"], case["seqs"]
        return {"bytes": n * V * (8 if case["given"] else 4) + 16 * sum(_drafts(case)) + 8 * n, "flops": 3 * n * V}
    nq, nkv, hd = HEADS[case["heads"]]
    rows, past = _counts(case)
    if case["op"] == "append":
        new, back = sum(rows), sum(r + p % BLOCK for r, p in zip(rows, past))
        # f32 rows in, codes out; the touched blocks' codes in, f32 rows out
        return {"bytes": nkv * hd * (new * (8 + 2) + back * (2 + 8)) + 4 * hd * new, "flops": nkv * hd * (new * 7 + back * 2)}
    pairs = sum(r * p + r * (r + 1) // 2 for r, p in zip(rows, past))
    return {"bytes": 2 * nkv * hd * sum(r + p for r, p in zip(rows, past)) + 8 * nq * hd * sum(rows),
            "flops": 4 * nq * hd * pairs}


# ---- inputs --------------------------------------------------------------------
def _gen(seed, tag):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + 7919 * tag + 17) & 0x7FFFFFFFFFFFFFFF)
    return g


def _normal(seed, tag, *shape):
    return torch.randn(*shape, generator=_gen(seed, tag), device=DEV)


def _uniform(seed, tag, *shape):
    """Uniform multiples of 2^-24 in [0, 1)."""
    return torch.randint(0, 1 << 24, shape, generator=_gen(seed, tag), device=DEV).float() / 16777216.0


def _two_to(e):
    """2^e in 64 bits, by the exponent field."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _needed(amax):
    """The smallest exponent with amax <= 127 * 2^e (127/128 * 2^7 = 127)."""
    f, x = torch.frexp(amax)
    e = x.long() - 7 + (f > 127.0 / 128.0)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _ints(values):
    return torch.tensor(values, dtype=torch.int64, device=DEV)


def _cache_inputs(case, seed):
    """A filled cache and the new rows. Keys and values have channels of different sizes, as a model's have."""
    nq, nkv, hd = HEADS[case["heads"]]
    rows, past = _counts(case)
    held = past if case["op"] == "append" else [p + r for p, r in zip(past, rows)]
    n, per = case["seqs"], case["page"] // BLOCK
    pages = [-(-(p + r) // case["page"]) for p, r in zip(past, rows)]
    order = torch.randperm(sum(pages) + 3, generator=torch.Generator().manual_seed(int(seed) & 0x7FFFFFFF)).tolist()
    table = [[order.pop() for _ in range(k)] for k in pages]
    most = max(pages)
    blocks = _ints([t + [0] * (most - len(t)) for t in table])
    blocks = (blocks[..., None] * per + torch.arange(per, device=DEV)).reshape(n, most * per)
    # rows held by each block of the pool
    starts = BLOCK * torch.arange(most * per, device=DEV)
    fill = torch.zeros((sum(pages) + 3) * per, dtype=torch.int64, device=DEV)
    real = starts[None] < _ints([k * case["page"] for k in pages])[:, None]
    fill[blocks[real]] = (_ints(held)[:, None] - starts).clamp(0, BLOCK)[real]
    valid = torch.arange(BLOCK, device=DEV) < fill[:, None]
    s = {"case": case, "rows": rows, "past": past, "held": held, "table": table, "blocks": blocks, "pages": len(fill) // per}
    for k, name in enumerate("kv"):
        size = torch.exp(0.4 * _normal(seed, 10 + k, nkv, hd))
        x = _normal(seed, 20 + k, len(fill), BLOCK, nkv, hd) * size * valid[..., None, None]
        e = _needed(x.abs().amax((1, 3)))
        s[name + "_exp"] = e.to(torch.int8)
        s[name + "_codes"] = torch.round(x * _two_to(-e).float()[:, None, :, None]).to(torch.int8)
        del x
        s["new_" + name] = _normal(seed, 30 + k, sum(rows), nkv * hd) * size.reshape(-1)
    s["q"] = _normal(seed, 40, sum(rows), nq * hd)
    angle = torch.arange(max(p + r for p, r in zip(past, rows)), dtype=torch.float64, device=DEV)[:, None] * (
        THETA ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=DEV) / hd))
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    # the batch as the scheduler knows it: sequence and place of each packed row
    s["row_seq"] = _ints([i for i, r in enumerate(rows) for _ in range(r)])
    s["row_at"] = _ints([t for r in rows for t in range(r)])
    s["first"] = _ints([sum(rows[:i]) for i in range(n)])
    s["n_rows"], s["n_past"], s["n_held"] = _ints(rows), _ints(past), _ints(held)
    return s


def _verify_inputs(case, seed):
    """A target that mostly agrees with its draft, whose tokens the draft's probabilities gave, or that were found
    in the text and have about even odds."""
    g, V = _drafts(case), case["vocab"]
    first = [sum(g[:i]) + i for i in range(len(g))]
    at = [f + j for f, k in zip(first, g) for j in range(k)]  # the target's rows that have a draft
    logits = 2.5 * _normal(seed, 1, sum(g) + len(g), V)
    s = {"case": case, "drafts": g, "draft": None}
    if case["given"]:
        below = logits[at] + 0.7 * _normal(seed, 2, len(at), V)
        s["draft"] = torch.softmax(below, -1)
        s["ids"] = (below - torch.log(-torch.log(_uniform(seed, 3, len(at), V) + 2.0 ** -26))).argmax(-1).int()
    else:
        s["ids"] = torch.randint(0, V, (len(at),), generator=_gen(seed, 3), device=DEV, dtype=torch.int32)
        logits[at, s["ids"].long()] += math.log(V) + 3.0
    s["target"] = torch.softmax(logits, -1)
    s["accept"], s["draw"] = _uniform(seed, 4, len(at)), _uniform(seed, 5, len(g))
    s["first"], s["first_draft"], s["n_drafts"] = _ints(first), _ints([f - i for i, f in enumerate(first)]), _ints(g)
    return s


def prepare(case, seed):
    s = _verify_inputs(case, seed) if case["op"] == "verify" else _cache_inputs(case, seed)
    if own:
        # the handles that a program on this framework holds: the library, the batch's slots and
        # lengths, the cache with what it holds (tensors and numbers are handed over in the pass)
        sys.path.insert(0, str(Path.cwd() / "llm.rs_amd"))
        lh = s["lh"] = importlib.import_module("llmrs_hip")
        lh.init(0)
        if case["op"] == "verify":
            s["own"] = {"counts": np.array(s["drafts"], np.int32)}
            return s
        nq, nkv, hd = HEADS[case["heads"]]
        n = case["seqs"]
        cache = lh.HipPagedCache(n_kv_heads=nkv, head_dim=hd, page_size=case["page"], n_pages=s["pages"], max_seqs=n,
                                 max_seq=len(s["cos"]), rope=(s["cos"].cpu().numpy(), s["sin"].cpu().numpy()))
        for i, pages in enumerate(s["table"]):
            cache.map(i, pages)
        slots, held = np.arange(n, dtype=np.int32), np.array(s["held"], np.int32)
        past, rows = np.array(s["past"], np.int32), np.array(s["rows"], np.int32)

        def cached(starts, ends):  # what the cache holds of these positions
            at = torch.arange(s["blocks"].shape[1] * BLOCK, device=DEV)
            kept = (at >= _ints(starts)[:, None]) & (at < _ints(ends)[:, None])
            return [lh.Tensor.from_device(_values(s, x).reshape(n, -1, nkv * hd)[kept].contiguous()) for x in "kv"]

        if held.sum():
            cache.append(*cached([0] * n, s["held"]), slots, held, rotate=False)
        s["own"] = {"cache": cache, "slots": slots, "rows": rows, "past": past, "from": past // BLOCK * BLOCK,
                    "older": past % BLOCK, "back": past % BLOCK + rows}
        if case["op"] == "append":
            s["own"]["begun"] = cached((past // BLOCK * BLOCK).tolist(), s["past"])
    return s


# ---- one pass ------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return {"append": _own_append, "attention": _own_attention, "verify": _own_verify}[op](s, s["own"], s["lh"])
    return {"append": _append, "attention": _attention, "verify": _verified}[op](s)


def _own_append(s, o, lh):
    c = o["cache"]
    # the state as it was: truncating leaves the exponents that the new rows raised, so the blocks
    # that they joined begin again with the rows and exponents that they had
    c.truncate(o["slots"], o["from"])
    c.append(*o["begun"], o["slots"], o["older"], rotate=False)
    k, v = (lh.Tensor.from_device(s["new_" + x]) for x in "kv")
    c.append(k, v, o["slots"], o["rows"])
    k, v = c.read(o["slots"], o["from"], o["back"])
    lh.sync()  # the results are there before another stream reads them
    return {"k": torch.as_tensor(k, device=DEV), "v": torch.as_tensor(v, device=DEV)}


def _own_attention(s, o, lh):
    out = o["cache"].attention(lh.Tensor.from_device(s["q"]), o["slots"], o["rows"])
    lh.sync()
    return torch.as_tensor(out, device=DEV)


def _own_verify(s, o, lh):
    target, draft = (None if s[x] is None else lh.Tensor.from_device(s[x]) for x in ("target", "draft"))
    ids, accept, draw = (s[x].cpu().numpy() for x in ("ids", "accept", "draw"))
    accepted, tokens = lh.verify_drafts(target, ids, o["counts"], accept, draw, draft=draft)
    return {"accepted": accepted, "tokens": tokens}


def _values(s, name):
    """The cache's values in f32 by sequence, [sequences][positions][KV heads][head_dim]."""
    b = s["blocks"]
    x = s[name + "_codes"][b].float() * _two_to(s[name + "_exp"][b]).float()[:, :, None, :, None]
    return x.reshape(b.shape[0], -1, *x.shape[3:])


def _rotated(x, c, t):
    """Halves of x turned by the angles of c + i t."""
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * t, a * t + b * c), -1)


def _append(s):
    nq, nkv, hd = HEADS[s["case"]["heads"]]
    rows, past = s["n_rows"], s["n_past"]
    # every sequence's touched blocks, as many as the widest has
    head = past // BLOCK
    span = max(((p % BLOCK) + r + BLOCK - 1) // BLOCK for p, r in zip(s["past"], s["rows"]))
    nth = head[:, None] + torch.arange(span, device=DEV)
    block = torch.gather(s["blocks"], 1, nth.clamp(max=s["blocks"].shape[1] - 1))
    pos = nth[..., None] * BLOCK + torch.arange(BLOCK, device=DEV)
    end = (past + rows)[:, None, None]
    old = pos < past[:, None, None]
    new = ~old & (pos < end)
    src = (s["first"] - past)[:, None, None] + pos
    src = torch.where(new, src, torch.zeros_like(src))
    out = {}
    for name in "kv":
        x = s["new_" + name].double().reshape(-1, nkv, hd)
        if name == "k":
            at = past[s["row_seq"]] + s["row_at"]
            x = _rotated(x, s["cos"].double()[at][:, None], s["sin"].double()[at][:, None])
        x = x[src] * new[..., None, None]
        e_old = s[name + "_exp"][block].long()
        need = _needed(x.abs().amax((2, 4)))
        e = torch.where(old.any(2)[..., None], torch.maximum(e_old, need), need)
        codes = torch.round(x * _two_to(-e)[:, :, None, :, None])
        kept = s[name + "_codes"][block].double() * _two_to(e_old - e)[:, :, None, :, None]
        codes = torch.where(old[..., None, None], torch.round(kept), codes)
        value = (codes * _two_to(e)[:, :, None, :, None]).float()
        out[name] = value[pos < end].reshape(-1, nkv * hd)
    return out


def _attention(s):
    nq, nkv, hd = HEADS[s["case"]["heads"]]
    n, c = s["case"]["seqs"], max(s["rows"])
    k, v = _values(s, "k").permute(0, 2, 3, 1).contiguous(), _values(s, "v").permute(0, 2, 1, 3).contiguous()
    t = torch.arange(c, device=DEV)
    at = s["n_past"][:, None] + t.clamp(max=c - 1)                       # [n][c] positions
    row = s["first"][:, None] + torch.minimum(t[None], s["n_rows"][:, None] - 1)
    at = torch.minimum(at, (s["n_past"] + s["n_rows"] - 1)[:, None])
    q = s["q"].reshape(-1, nq, hd)[row]                                 # [n][c][nq][hd]
    q = _rotated(q, s["cos"][at][:, :, None], s["sin"][at][:, :, None])
    q = q.reshape(n, c, nkv, nq // nkv, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, hd)
    p = torch.matmul(q, k).reshape(n, nkv, nq // nkv, c, -1) / math.sqrt(hd)
    p.masked_fill_((torch.arange(p.shape[-1], device=DEV) > at[..., None])[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(n, nkv, -1, p.shape[-1]), v).reshape(n, nkv, nq // nkv, c, hd) / total
    return out.permute(0, 3, 1, 2, 4).reshape(n, c, nq * hd)[s["row_seq"], s["row_at"]]


def _verified(s):
    n, g, V = s["case"]["seqs"], s["n_drafts"], s["case"]["vocab"]
    most = max(s["drafts"])
    j = torch.arange(most, device=DEV)
    has = j < g[:, None]
    if s["ids"].numel():
        d = torch.where(has, s["first_draft"][:, None] + j, torch.zeros_like(has, dtype=torch.int64))
        ids, u = s["ids"].long()[d], s["accept"].double()[d]
        p = s["target"][s["first"][:, None] + torch.where(has, j, torch.zeros_like(j)), ids].double()
        q = s["draft"][d, ids].double() if s["draft"] is not None else torch.ones_like(p)
        accepted = ((u * q < p) & has).long().cumprod(1).sum(1)
    else:
        accepted, ids = torch.zeros_like(g), torch.zeros(n, most, dtype=torch.int64, device=DEV)
    # the row drawn from: what the target has over the draft, or the target after the last draft
    w = s["target"][s["first"] + accepted].double()
    rest = (accepted < g)[:, None]
    if s["ids"].numel():
        at = torch.minimum(accepted, g - 1).clamp(min=0)
        if s["draft"] is not None:
            less = s["draft"][torch.where(rest[:, 0], s["first_draft"] + at, torch.zeros_like(at))].double()
        else:
            less = torch.zeros_like(w).scatter_(1, torch.gather(ids, 1, at[:, None]), 1.0)
        left = (w - less).clamp(min=0.0)
        w = torch.where(rest & (left.sum(1, keepdim=True) > 0), left, w)
    c = w.cumsum(1)
    drawn = (c <= s["draw"].double()[:, None] * c[:, -1:]).sum(1).clamp(max=V - 1)
    place = torch.arange(most + 1, device=DEV)
    padded = torch.cat((ids, torch.zeros_like(ids[:, :1])), 1) if most else torch.zeros(n, 1, dtype=torch.int64, device=DEV)
    tokens = torch.where(place < accepted[:, None], padded, torch.where(place == accepted[:, None], drawn[:, None], torch.full_like(padded, -1)))
    return {"accepted": accepted.int(), "tokens": tokens.int()}


# ---- the same in 64 bits ---------------------------------------------------------
def exact(case, seed):
    if case["op"] == "verify":
        return _exact_verify(_verify_inputs(case, seed))
    s = _cache_inputs(case, seed)
    return (_exact_append if case["op"] == "append" else _exact_attention)(s)


def _turn(x, cos, sin, start):
    """Rows [rows][heads][hd] at positions start.. as complex numbers turned by their angles, in 64 bits."""
    h = x.shape[-1] // 2
    c, t = (a[start:start + len(x), None].astype(np.float64) for a in (cos, sin))
    return np.concatenate((x[..., :h] * c - x[..., h:] * t, x[..., :h] * t + x[..., h:] * c), -1)


def _exact_append(s):
    nq, nkv, hd = HEADS[s["case"]["heads"]]
    cos, sin = s["cos"].cpu().numpy(), s["sin"].cpu().numpy()
    blocks = s["blocks"].cpu().numpy()
    out = {}
    for name in "kv":
        codes, exps = s[name + "_codes"].cpu().numpy(), s[name + "_exp"].cpu().numpy().astype(np.int64)
        fresh = s["new_" + name].cpu().numpy().astype(np.float64).reshape(-1, nkv, hd)
        got, row = [], 0
        for i, (r, p) in enumerate(zip(s["rows"], s["past"])):
            x = fresh[row:row + r]
            x = _turn(x, cos, sin, p) if name == "k" else x
            row += r
            for b in range(p // BLOCK, (p + r - 1) // BLOCK + 1):
                part = x[max(0, b * BLOCK - p):max(0, (b + 1) * BLOCK - p)]
                kept = max(0, p - b * BLOCK)
                top = np.abs(part).max((0, 2))
                e = np.where(top > 0, np.frexp(top)[1] - 7, E_MIN)
                e = np.clip(np.where(top > np.ldexp(127.0, e), e + 1, e), E_MIN, E_MAX)
                if kept:
                    was = exps[blocks[i, b]]
                    e = np.maximum(e, was)
                    before = np.rint(np.ldexp(codes[blocks[i, b], :kept].astype(np.float64), (was - e)[:, None]))
                    got.append(np.ldexp(before, e[:, None]))
                got.append(np.ldexp(np.rint(np.ldexp(part, -e[:, None])), e[:, None]))
        out[name] = np.concatenate(got).reshape(-1, nkv * hd)
    return out


def _exact_attention(s):
    nq, nkv, hd = HEADS[s["case"]["heads"]]
    cos, sin = s["cos"].cpu().numpy(), s["sin"].cpu().numpy()
    q = s["q"].cpu().numpy().astype(np.float64).reshape(-1, nq, hd)
    out, row = [], 0
    for i, (r, p) in enumerate(zip(s["rows"], s["past"])):
        b = s["blocks"][i, : -(-(p + r) // BLOCK)]
        k, v = ((s[x + "_codes"][b].double() * torch.pow(2.0, s[x + "_exp"][b].double())[:, None, :, None]).reshape(-1, nkv, hd)[: p + r]
                for x in "kv")
        turned = torch.from_numpy(_turn(q[row:row + r], cos, sin, p)).to(DEV)
        row += r
        seen = torch.arange(p + r, device=DEV) <= torch.arange(p, p + r, device=DEV)[:, None]
        heads = []
        for h in range(nq):
            score = (turned[:, h] @ k[:, h // (nq // nkv)].T.contiguous() / math.sqrt(hd)).masked_fill(~seen, -math.inf)
            heads.append(score.softmax(-1) @ v[:, h // (nq // nkv)])
        out.append(torch.stack(heads, 1).reshape(r, nq * hd))
    return torch.cat(out)


def _exact_verify(s):
    target, ids = s["target"].cpu().numpy(), s["ids"].cpu().numpy()
    draft = None if s["draft"] is None else s["draft"].cpu().numpy()
    u, draws = s["accept"].cpu().numpy().astype(np.float64), s["draw"].cpu().numpy().astype(np.float64)
    accepted, tokens, at, d0 = [], [], 0, 0
    for i, g in enumerate(s["drafts"]):
        k = 0
        while k < g:
            x = ids[d0 + k]
            if not u[d0 + k] * (1.0 if draft is None else float(draft[d0 + k, x])) < float(target[at + k, x]):
                break
            k += 1
        w = target[at + k].astype(np.float64)
        if k < g:
            less = draft[d0 + k].astype(np.float64) if draft is not None else (np.arange(len(w)) == ids[d0 + k]).astype(np.float64)
            left = np.maximum(w - less, 0.0)
            w = left if left.sum() > 0 else w
        c = np.cumsum(w)
        got = min(int(np.searchsorted(c, draws[i] * c[-1], side="right")), len(w) - 1)
        accepted.append(k)
        tokens.append(list(ids[d0:d0 + k]) + [got] + [-1] * (max(s["drafts"]) - k))
        at, d0 = at + g + 1, d0 + g
    return {"accepted": np.array(accepted, np.int32), "tokens": np.array(tokens, np.int32)}
