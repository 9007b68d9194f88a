"""Pages for the next step, attention over shared prefixes and the verification of drafted tokens, against plain restatements.

Tolerances.  Pages, places and tokens are whole numbers and have to be equal.  A draft is judged by a sum of f32 exponentials: each has an
argument rounded to 2^-24 of itself and is off by 2 half steps, so that a probability is within 2^-20 of itself for arguments up to some ten; drafts
nearer to the border than that are left out of a comparison (tests assert that hardly any is).  Weights that tokens are drawn from have 64 bits:
a draw nearer to a border than 2^-40 of the whole is left out.
"""
import ctypes
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from conftest import ROOT, cg
from test_paged import BF16, F32, Host, attention, back, net, plain_logits, put, rounded
from test_paged import PARTS, off_from_rounded, relative

gpu = pytest.mark.gpu
INDEX = 6


def raises_index(B):
    with pytest.raises(cg.BackendPanic) as e:
        B.sync()
    assert e.value.status == INDEX


# ---------------------------------------------------------------- pages for the next step


def plain_assign(lens, new, done, first, held, table, free, n_free, page, budget):
    """Row by row; (starts, lens, held, n_free, positions, slots), table and free in place, and whether something cannot be."""
    rows, cols = table.shape
    bad = n_free > len(free)
    ask = []
    for r in range(rows):
        l, w, h, f = int(lens[r]), int(new[r]), int(held[r]), int(first[r])
        ends = bool(done[r])
        ok = h <= cols and f <= h and (ends or (l <= h * page and (w == 0 or -(-(l + w) // page) <= cols)))
        bad = bad or not ok
        ask.append((ok, ends, l, w, h, f))
    give = [(r, c) for r, (ok, ends, l, w, h, f) in enumerate(ask) if ok and ends for c in range(f, h)]
    valid = n_free + len(give) <= len(free) and n_free <= len(free)
    bad = bad or not valid
    count = n_free
    if valid:
        for r, c in give:
            free[count] = table[r, c]
            count += 1
    sums = {}
    needs = {r: max(-(-(l + w) // page) - h, 0) if w else 0 for r, (ok, ends, l, w, h, f) in enumerate(ask) if ok and valid and not ends}
    pages = tokens = 0
    for runs in (True, False):
        for r, need in needs.items():
            ok, ends, l, w, h, f = ask[r]
            if (l > f * page) == runs:
                sums[r] = (pages, need, w, w > 0 and (need == 0 or pages + need <= count) and tokens + w <= budget)
                pages += need
                tokens += w
    starts, lens_out, held_out, positions, slots = [0], [], [], [], []
    top = count
    for r, (ok, ends, l, w, h, f) in enumerate(ask):
        before, need, w, fits = sums.get(r, (0, 0, 0, False))
        if ok and valid and ends:
            lens_out.append(0)
            held_out.append(f)
            starts.append(starts[-1])
            continue
        n = w if fits else 0
        if fits:
            for j in range(need):
                table[r, h + j] = free[top - 1 - before - j]
            count -= need
        starts.append(starts[-1] + n)
        lens_out.append(l + n)
        held_out.append(h + (need if fits else 0))
        for p in range(l, l + n):
            positions.append(p)
            slots.append((int(table[r, p // page]) * page + p % page) & 0xFFFFFFFF)
    return starts, lens_out, held_out, count, positions, slots, bad


def requests(rng, rows, page, cached=300, prompt=200, drafts=4, spare=3, tight=0.6):
    """Requests in the middle of their lives, and more pages asked for than there are."""
    cols = -(-(max(cached, prompt) + drafts + 2) // page) + spare
    kind = rng.random(rows)
    lens = np.where(kind < 0.6, rng.integers(1, cached + 1, rows), 0)
    new = np.where(kind < 0.6, rng.integers(0, drafts + 2, rows), rng.integers(0, prompt + 1, rows))
    done = (rng.random(rows) < 0.15).astype(np.int64) * rng.integers(1, 9, rows)
    held = np.minimum(-(-lens // page) + rng.integers(0, 2, rows), cols)
    first = np.where(rng.random(rows) < 0.3, lens // page // 2, 0)
    prefix = rng.random(rows) < 0.2     # rows that begin behind a prefix of others
    first = np.where(prefix, np.minimum(2, cols - 1), first)
    lens = np.where(prefix, first * page, lens)
    held = np.where(prefix, first, held)
    new = np.where(prefix, rng.integers(0, 20, rows), new)
    table = rng.integers(0, 1 << 20, (rows, cols))
    need = int(np.maximum(-(-(lens + new) // page) - held, 0).sum())
    n_free = int(need * tight) + int(rng.integers(0, 3))
    free = rng.integers(0, 1 << 20, n_free + int(held.sum()) + int(rng.integers(0, 5)))
    return dict(lens=lens, new=new, done=done, first=first, held=held, table=table, free=free, n_free=n_free)


def check_assign(B, s, page, budget, places=None, in_place=False, outputs=("positions", "slots"), optional=("done", "first"), raises=None):
    rows = len(s["lens"])
    places = budget if places is None else places
    zero = np.zeros(rows, np.int64)
    want_table, want_free = s["table"].copy(), s["free"].copy()
    want = plain_assign(s["lens"], s["new"], s["done"] if "done" in optional else zero, s["first"] if "first" in optional else zero, s["held"], want_table, want_free,
                        s["n_free"], page, min(budget or 1 << 40, places if outputs else 1 << 40))
    up = {n: put(B, np.asarray(s[n], np.uint32)) for n in ("lens", "new", "done", "first", "held", "table", "free")}
    up["n_free"] = put(B, np.uint32([s["n_free"]]))
    old = np.arange(7, 7 + places).astype(np.uint32)
    more = {n: put(B, old) for n in outputs}
    starts = put(B, np.full(rows + 1, 99, np.uint32))
    outs = {n: up[n[:-4]] if in_place else put(B, np.full(1 if n == "n_free_out" else rows, 98, np.uint32)) for n in ("lens_out", "held_out", "n_free_out")}
    B.paged_assign(up["lens"][0], up["new"][0], page, up["held"][0], up["table"][0], up["free"][0], up["n_free"][0], starts[0],
                   done=up["done"][0] if "done" in optional else None, first=up["first"][0] if "first" in optional else None, max_tokens=budget,
                   **{n: t[0] for n, t in more.items()}, **({} if in_place else {n: t[0] for n, t in outs.items()}))
    if want[6] if raises is None else raises:
        raises_index(B)
    get = lambda t: back(B, t[1]).astype(np.int64) & 0xFFFFFFFF
    assert get(starts).tolist() == want[0]
    assert get(outs["lens_out"]).tolist() == want[1] and get(outs["held_out"]).tolist() == want[2] and get(outs["n_free_out"]).tolist() == [want[3]]
    assert np.array_equal(get(up["table"]), want_table)
    # what is above the stack is nobody's
    assert np.array_equal(get(up["free"])[:want[3]], want_free[:want[3]])
    n = len(want[4])
    for name, values in (("positions", want[4]), ("slots", want[5])):
        if name in outputs:
            got = get(more[name])
            assert got[:n].tolist() == values and np.array_equal(got[n:], old[n:])
    return want


@gpu
@pytest.mark.parametrize("rows", [1, 2, 8, 31, 33, 127, 128, 129, 300, 512, 513])
@pytest.mark.parametrize("page", [8, 16, 256])
def test_assign(cuda, rows, page):
    rng = np.random.default_rng(rows + page)
    fits = 0
    for i in range(4):
        s = requests(rng, rows, page, cached=int(rng.integers(1, 400)), prompt=int(rng.integers(1, 300)), tight=(0.0, 0.5, 0.9, 1.0)[i])
        want = check_assign(cuda, s, page, int(s["new"].sum() * (0.7 if i == 2 else 1)) + i, in_place=i % 2 == 0)
        fits += want[0][-1]
    assert fits > 0


@gpu
@pytest.mark.parametrize("rows", [1024, 1025, 2100, 4096])
def test_assign_many_rows(cuda, rows):
    rng = np.random.default_rng(rows)
    for tight in (0.4, 1.0):
        s = requests(rng, rows, 16, cached=90, prompt=60, tight=tight)
        check_assign(cuda, s, 16, int(s["new"].sum()), in_place=tight == 1.0)


@gpu
def test_assign_of_one_long_prompt_and_most_rows(cuda):
    rng = np.random.default_rng(0)
    s = requests(rng, 3, 16)
    s.update(lens=np.int64([0, 5, 0]), new=np.int64([1, 1, 70001]), done=np.int64([0, 0, 0]), first=np.int64([0, 0, 0]), held=np.int64([0, 1, 0]),
             table=rng.integers(0, 9, (3, 4400)), free=rng.permutation(6000), n_free=5000)
    assert check_assign(cuda, s, 16, 80000)[0][-1] == 70003
    rows = 65535
    s = dict(lens=np.zeros(rows, np.int64), new=np.ones(rows, np.int64), done=np.zeros(rows, np.int64), first=np.zeros(rows, np.int64), held=np.zeros(rows, np.int64),
             table=np.zeros((rows, 1), np.int64), free=rng.permutation(rows), n_free=rows - 5)
    assert check_assign(cuda, s, 8, rows)[0][-1] == rows - 5


@gpu
@pytest.mark.parametrize("outputs", [(), ("positions",), ("slots",)])
@pytest.mark.parametrize("optional", [(), ("done",), ("first",)])
def test_assign_without_some_of_its_tensors(cuda, outputs, optional):
    rng = np.random.default_rng(len(outputs) + 2 * len(optional))
    s = requests(rng, 40, 16)
    if "first" not in optional:
        s["lens"] = np.minimum(s["lens"], s["held"] * 16)
    check_assign(cuda, s, 16, 0 if not outputs else 5000, places=5000, outputs=outputs, optional=optional)
    check_assign(cuda, s, 16, 300, places=5000, outputs=outputs, optional=optional, in_place=True)


@gpu
def test_assign_rows_that_cannot_be(cuda):
    """They get nothing and raise; the others are served as if they were not there."""
    rng = np.random.default_rng(5)
    for i in range(12):
        s = requests(rng, 20, 16, tight=2.0)
        r = int(rng.integers(0, 20))
        cols = s["table"].shape[1]
        for name, value in [(("held", cols + 1),), (("first", s["held"][r] + 1),), (("lens", s["held"][r] * 16 + 1), ("done", 0)), (("new", cols * 16 + 1), ("done", 0)),
                            (("new", 0xFFFFFFFF), ("done", 0)), (("lens", 0xFFFFFFFF), ("done", 0))][i % 6]:
            s[name] = s[name].copy()
            s[name][r] = value
        assert check_assign(cuda, s, 16, 9000)[6]
    s = requests(rng, 20, 16)
    s["n_free"] = len(s["free"]) + 1
    assert check_assign(cuda, s, 16, 9000)[0][-1] == 0
    s = requests(rng, 20, 16)
    s["done"][:] = 1
    s["free"] = s["free"][:s["n_free"]]
    want = check_assign(cuda, s, 16, 9000)
    assert want[6] and want[1] == s["lens"].tolist()


@gpu
def test_assign_slots_beyond_32_bits(cuda):
    s = dict(lens=np.int64([0, 0]), new=np.int64([2, 2]), done=np.int64([0, 0]), first=np.int64([0, 0]), held=np.int64([0, 0]), table=np.zeros((2, 2), np.int64),
             free=np.int64([(1 << 28) - 1, 1 << 28]), n_free=2)
    table, free = s["table"].copy(), s["free"].copy()
    up = {n: put(cuda, np.asarray(s[n], np.uint32)) for n in ("lens", "new", "held", "table", "free")}
    n_free, starts, slots = (put(cuda, np.zeros(n, np.uint32) + f) for n, f in ((1, 2), (3, 0), (4, 0)))
    cuda.paged_assign(up["lens"][0], up["new"][0], 16, up["held"][0], up["table"][0], up["free"][0], n_free[0], starts[0], slots=slots[0])
    raises_index(cuda)
    assert (back(cuda, slots[1]).astype(np.int64) & 0xFFFFFFFF).tolist() == [0xFFFFFFFF] * 2 + [0xFFFFFFF0, 0xFFFFFFF1]


# ---------------------------------------------------------------- drafted tokens


def plain_verify(logits, probs, tokens, starts, uniform, heat, lens, judged=2.0 ** -20, drawn=2.0 ** -40):
    """Row by row in 64 bits: (accepted, next, lens), and the rows that a border is too near for."""
    out, near = [], set()
    for r in range(len(starts) - 1):
        a, b = int(starts[r]), int(starts[r + 1])
        if a == b:
            out.append(None)
            continue
        T = float(heat[r])
        for m in range(a, b):
            x = logits[m].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            top = x.max()
            last = m == b - 1
            if not np.isfinite(top):
                w = None
                break
            if not T > 0:
                p = np.zeros_like(x)
                p[int(np.argmax(x))] = 1.0
            else:
                p = np.exp((x - top) / min(max(T, 2.0 ** -100), 2.0 ** 100))
                p /= p.sum()
            if last:
                w = p
                break
            d = int(tokens[m + 1])
            q = np.zeros_like(x) if probs is None else probs[m].astype(np.float64)
            q = np.where(q > 0, q, 0.0)
            if probs is None:
                q[d] = 1.0
            if T > 0:
                u = np.float64(uniform[m])
                stands = u * q[d] < p[d]
                if abs(u * q[d] - p[d]) <= judged * p[d]:
                    near.add(r)
            else:
                stands = p[d] == 1.0
            if not stands:
                w = np.maximum(p - q, 0.0) if T > 0 else p
                if T > 0 and probs is None:
                    w = p.copy()
                    w[d] = 0.0
                if not w.sum() > 0:
                    w = p
                break
        if w is None:
            token = 0xFFFFFFFF
        else:
            c = np.cumsum(w)
            t = np.float64(uniform[b - 1]) * c[-1]
            if not T > 0:
                token = int(np.argmax(w))
            else:
                above = np.nonzero((c > t) & (w > 0))[0]
                token = int(above[0]) if len(above) else int(np.nonzero(w)[0][-1])
                if len(w) > 1 and np.abs(c[:-1] - t).min() <= drawn * c[-1] and 0 < t < c[-1]:
                    near.add(r)
        out.append((m - a, token, int(lens[r]) - (b - 1 - m)))
    return out, near


class Drafts:
    """Rows of counts[r] tokens; the drafter's logits are much like the target's."""

    def __init__(self, counts, V, seed=0, store="f32", probs="f32", heat=1.0, peak=True, spread=2.5, spare=1):
        rng = self.rng = np.random.default_rng(seed)
        self.counts, self.V, self.store, self.kind = counts, V, store, probs
        self.starts = np.concatenate([[0], np.cumsum(counts)])
        M = self.M = int(self.starts[-1]) + spare
        x = rng.standard_normal((M, V)) * spread
        if peak:
            x[np.arange(M), rng.integers(0, V, M)] = math.log(V) + 3.0
        self.logits = rounded(x, store)
        d = x + rng.standard_normal((M, V)) * 0.7
        q = np.exp(d - d.max(1, keepdims=True))
        q /= q.sum(1, keepdims=True)
        self.probs = None if probs == "none" else rounded(q, probs)
        self.tokens = rng.integers(0, V, M)
        for m in range(M - 1):
            self.tokens[m + 1] = int(np.argmax(d[m])) if probs == "none" else int(np.argmax(q[m] / rng.exponential(size=V)))
        self.uniform = rng.random(M).astype(np.float32)
        self.uniform = np.minimum(self.uniform, np.float32(1 - 2.0 ** -24))
        rows = len(counts)
        self.heat = np.full(rows, heat, np.float32) if np.ndim(heat) == 0 else np.resize(np.asarray(heat, np.float32), rows)
        self.lens = np.array([40 + 3 * r + n for r, n in enumerate(counts)])


def device_rows(B, a, store, offset, pad):
    """Rows `pad` values apart that begin `offset` values into their memory; what is between is NaN."""
    import torch
    M, V = a.shape
    flat = torch.full((offset + M * (V + pad) + 8,), float("nan"), device="cuda").to({"f32": torch.float32, "bf16": torch.bfloat16}[store])
    x = flat[offset:offset + M * (V + pad)].reshape(M, V + pad)[:, :V]
    x.copy_(torch.from_numpy(np.ascontiguousarray(a)))
    torch.cuda.synchronize()
    return B.from_device(x), flat


def check_verify(B, d, offset=0, pad=0, max_new=None, in_place=False, with_heat=True, limit=0.02):
    logits = device_rows(B, d.logits, d.store, offset, pad)
    probs = None if d.probs is None else device_rows(B, d.probs, d.kind, offset and 8 - offset, pad // 2)
    tokens, starts, lens = (put(B, np.asarray(x, np.uint32)) for x in (d.tokens, d.starts, d.lens))
    uniform, heat = put(B, d.uniform), put(B, d.heat)
    rows = len(d.counts)
    out = [put(B, np.full(rows, 77, np.uint32)) for _ in range(3)]
    if in_place:
        out[2] = lens
    B.verify_drafts(logits[0], tokens[0], starts[0], uniform[0], probs=probs and probs[0], temperature=heat[0] if with_heat else None, lens=lens[0],
                    max_new=max(d.counts) if max_new is None else max_new, out=[x[0] for x in out])
    got = np.stack([back(B, x[1]).astype(np.int64) & 0xFFFFFFFF for x in out], 1)
    want, near = plain_verify(d.logits, d.probs, d.tokens, d.starts, d.uniform, d.heat if with_heat else np.ones(rows), d.lens)
    assert len(near) <= limit * rows + 1, near
    for r, w in enumerate(want):
        if w is None:
            assert got[r].tolist() == [77, 77, int(d.lens[r]) if in_place else 77]
        elif r not in near:
            assert got[r].tolist() == list(w), (r, got[r], w)
    return got


COUNTS = [[1], [5], [1, 2, 0, 4, 9], [3] * 20, [0, 0, 1], [6] * 70]


@gpu
@pytest.mark.parametrize("store,probs", [("f32", "f32"), ("f32", "none"), ("bf16", "bf16"), ("bf16", "none"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("V", [1, 2, 3, 7, 31, 64, 257, 1000, 4099])
@pytest.mark.parametrize("heat", [1.0, 0.0, [0.6, 0.0, 1.7]])
def test_verify(cuda, store, probs, V, heat):
    for i, counts in enumerate(COUNTS):
        check_verify(cuda, Drafts(counts, V, seed=i + V, store=store, probs=probs, heat=heat), in_place=i % 2 == 0, with_heat=heat != 1.0 or i % 3 > 0)


@gpu
@pytest.mark.parametrize("store,probs,V,counts", [("f32", "f32", 50257, [4, 2, 5]), ("bf16", "bf16", 151936, [3, 5]), ("bf16", "none", 256000, [8]), ("f32", "none", 128256, [1, 3, 2]),
                                                  ("f32", "f32", 1 << 19, [2]), ("bf16", "bf16", (1 << 19) - 3, [2, 2]), ("bf16", "f32", 32000, [4] * 40)])
def test_verify_whole_vocabularies(cuda, store, probs, V, counts):
    check_verify(cuda, Drafts(counts, V, seed=V, store=store, probs=probs))


@gpu
@pytest.mark.parametrize("store,probs,V,counts,offset,pad", [("f32", "f32", 131077, [2] * 19, 0, 0), ("bf16", "bf16", 140001, [2, 1] * 13, 3, 5), ("bf16", "none", 131072, [1, 3] * 10, 0, 0),
                                                             ("f32", "bf16", 20001, [3] * 20, 1, 2), ("f32", "none", 9001, [2] * 50, 0, 3)])
def test_verify_rows_that_fill_the_device(cuda, store, probs, V, counts, offset, pad):
    """Rows and vocabularies at which other numbers of threads and blocks are taken."""
    check_verify(cuda, Drafts(counts, V, seed=V, store=store, probs=probs, heat=[1.0, 0.7, 0.0]), offset=offset, pad=pad)


@gpu
@pytest.mark.parametrize("store,probs", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "none")])
@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (3, 5), (2, 64), (7, 3)])
def test_verify_rows_that_begin_anywhere(cuda, store, probs, offset, pad):
    for V in (1, 9, 515, 3001):
        check_verify(cuda, Drafts([3, 1, 6, 2], V, seed=V, store=store, probs=probs), offset=offset, pad=pad, max_new=0)


@gpu
@pytest.mark.parametrize("store,probs", [("f32", "f32"), ("bf16", "none")])
@pytest.mark.parametrize("heat", [1.0, 0.0])
def test_verify_long_rows(cuda, store, probs, heat):
    """More positions than are held at a time; drafts that nearly all stand."""
    d = Drafts([40, 9, 17, 33, 1], 600, seed=3, store=store, probs=probs, heat=heat, spread=0.2)
    d.uniform[:] = d.uniform * 0.2
    if heat == 0.0:
        d.tokens[1:] = d.logits.argmax(1)[:-1]
    got = check_verify(cuda, d)
    assert got[0, 0] > 8


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("probs", ["f32", "none"])
@pytest.mark.parametrize("heat", [1.0, 0.0, 0.3])
def test_verify_masked_logits(cuda, store, probs, heat):
    """-inf, the lowest value of the type, and NaN in masked places; all masked; an infinity."""
    lowest = float(np.float32(-3.0e38))
    for fill in (-np.inf, lowest, np.nan):
        d = Drafts([4] * 30, 700, seed=11, store=store, probs=probs, heat=heat)
        mask = d.rng.random(d.logits.shape) < 0.9
        mask[np.arange(d.M), d.rng.integers(0, 700, d.M)] = False
        d.logits[mask] = rounded(np.float32([fill]), store)[0] if np.isfinite(fill) else fill
        check_verify(cuda, d)
        d.logits[::5] = fill if not np.isfinite(fill) else -np.inf   # nothing is left of these
        got = check_verify(cuda, d)
        assert (got[:, 1] == 0xFFFFFFFF).any()
        d.logits[1::5, 3] = np.inf
        check_verify(cuda, d)


@gpu
def test_verify_numbers_at_the_ends(cuda):
    """u of 0 takes the first token with a weight, of 1 (or none) the last; the drafter's probabilities above the target's, negative and NaN."""
    for store in ("f32", "bf16"):
        d = Drafts([1] * 6 + [2] * 6, 900, seed=2, store=store)
        for u in (0.0, 1.0, 2.0 ** -30, 1 - 2.0 ** -24):
            d.uniform[:] = u
            check_verify(cuda, d, limit=1.0 if 0 < u < 1 else 0.02)
        d.logits[:, 0] = -np.inf
        d.logits[:, -5:] = -np.inf
        for u in (0.0, 1.0):
            d.uniform[:] = u
            got = check_verify(cuda, d)
            assert (got[:6, 1] == (1 if u == 0 else 894)).all()
        d = Drafts([2] * 12, 900, seed=2, store=store)
        d.probs[:] = 2.0
        d.uniform[::2] = 0.999
        check_verify(cuda, d)
        d.probs[:, ::3] = np.nan
        d.probs[:, 1::3] = -1.0
        check_verify(cuda, d)


@gpu
@pytest.mark.parametrize("heat", [1e-30, 2.0 ** -120, 1e-3, 50.0, 1e30, np.inf, np.nan, -1.0])
def test_verify_temperatures(cuda, heat):
    for store in ("f32", "bf16"):
        d = Drafts([3] * 10, 300, seed=9, store=store, heat=heat)
        check_verify(cuda, d, limit=0.2)


@gpu
def test_verify_equal_logits_go_to_the_first(cuda):
    for store in ("f32", "bf16"):
        d = Drafts([3] * 8, 2000, seed=4, store=store, probs="none", heat=0.0)
        d.logits[:, [17, 900, 1999]] = 30.0
        d.logits[::2, 5] = 0.0
        d.tokens[:] = 17
        got = check_verify(cuda, d)
        assert (got[:, 0] == 2).all() and (got[:, 1] == 17).all()
        d.logits[:] = -0.0
        d.logits[:, 7] = 0.0
        assert (check_verify(cuda, d)[:, 1] == 0).all()


@gpu
def test_verify_tokens_are_distributed_as_the_targets(cuda):
    """The first token put out, over many rows of the same logits: within 5 standard deviations of the target's probability, whatever the drafter's."""
    rows, V = 20000, 7
    rng = np.random.default_rng(0)
    logits = np.resize(rng.standard_normal(V) * 1.5, (2 * rows, V)).astype(np.float32)
    q = rng.random(V)
    q = (q / q.sum()).astype(np.float32)
    drafts = rng.choice(V, rows, p=q.astype(np.float64) / q.astype(np.float64).sum())
    tokens = np.zeros(2 * rows, np.uint32)
    tokens[1::2] = drafts
    B = cuda
    for probs in (np.resize(q, (2 * rows, V)), None):
        if probs is None:
            tokens[1::2] = 3
        out = [put(B, np.zeros(rows, np.uint32)) for _ in range(2)]
        B.verify_drafts(put(B, logits)[0], put(B, tokens)[0], put(B, np.arange(0, 2 * rows + 1, 2).astype(np.uint32))[0],
                        put(B, rng.random(2 * rows).astype(np.float32))[0], probs=None if probs is None else put(B, probs)[0], max_new=2,
                        out=(out[0][0], out[1][0], None))
        accepted, following = (back(B, x[1]) for x in out)
        first = np.where(accepted == 1, tokens[1::2], following)
        p = np.exp(logits[0].astype(np.float64))
        p /= p.sum()
        seen = np.bincount(first, minlength=V) / rows
        assert (np.abs(seen - p) <= 5 * np.sqrt(p * (1 - p) / rows)).all()
        # a draft stands with probability min(1, p / q): over all drafts sum min(p, q), and p of the one token that has no probabilities
        stands = p[3] if probs is None else np.minimum(p, q).sum()
        assert abs(accepted.mean() - stands) <= 5 * math.sqrt(stands * (1 - stands) / rows)


@gpu
def test_verify_rows_that_cannot_be(cuda):
    import torch
    B = cuda
    d = Drafts([3, 4, 2, 3], 100, seed=1)
    for what in ("draft", "starts", "most", "lens"):
        tokens, starts, lens = d.tokens.copy(), d.starts.copy(), d.lens.copy()
        most = 4
        if what == "draft":
            tokens[d.starts[1] + 3] = 100
        elif what == "starts":
            starts[1] = d.M + 5
        elif what == "most":
            most = 3
        else:
            lens[1] = 2
        out = [put(B, np.full(4, 77, np.uint32)) for _ in range(3)]
        B.verify_drafts(put(B, d.logits)[0], put(B, tokens.astype(np.uint32))[0], put(B, starts.astype(np.uint32))[0], put(B, d.uniform)[0], probs=put(B, d.probs)[0],
                        lens=put(B, lens.astype(np.uint32))[0], max_new=most, out=[x[0] for x in out])
        raises_index(B)
        got = [back(B, x[1]) for x in out]
        assert all(g[1] == 77 and g[3] != 77 for g in got), what
        assert what == "starts" or all(g[0] != 77 for g in got)


@gpu
@pytest.mark.parametrize("lazy", [0, 1])
def test_verify_lengths_of_rows_without_tokens(lazy):
    """Without an output of its own the call returns all rows' lengths: those of rows that had no tokens are what they were."""
    B = cg.CudaBackend(0, cg.PREC_F32)
    B.set_option("lazy", lazy)
    d = Drafts([2, 0, 3, 0, 1], 300, seed=1)
    t = [B.from_numpy(np.asarray(x, np.uint32)) for x in (d.tokens, d.starts, d.lens)]
    lens = B.cast(B.add(B.from_numpy(d.lens.astype(np.float32)), B.from_numpy(np.zeros(5, np.float32))), cg.U32) if lazy else t[2]
    accepted, following, left = B.verify_drafts(B.from_numpy(d.logits), t[0], t[1], B.from_numpy(d.uniform), probs=B.from_numpy(d.probs), lens=lens)
    want, near = plain_verify(d.logits, d.probs, d.tokens, d.starts, d.uniform, d.heat, d.lens)
    assert not near
    got = [B.to_numpy(x).astype(np.int64) for x in (accepted, following, left)]
    assert [g[r] for r, w in enumerate(want) if w for g in got] == [x for w in want if w for x in w]
    assert [got[2][r] for r in (1, 3)] == [d.lens[r] for r in (1, 3)]
    assert B.to_numpy(lens).tolist() == d.lens.tolist()   # (which stay as they are)
    # a step in which no row has any
    none = B.verify_drafts(B.zeros((0, 300), cg.F32), B.zeros((0,), cg.U32), B.zeros((6,), cg.U32), B.zeros((0,), cg.F32), lens=lens)
    assert B.to_numpy(none[2]).tolist() == d.lens.tolist()
    B.close()


@gpu
@pytest.mark.parametrize("V", [700, 20001])
@pytest.mark.parametrize("store", ["f32", "bf16"])
def test_verify_drafters_that_agree_with_the_target(cuda, V, store):
    """The drafter's probabilities are the target's, rounded to f32, but for the draft's, which are twice that: what is left of the target are roundings of some 2^-26 of it.
    The kernel's weights are within 2^-46 of themselves, so what is left of the sums within 2^-44 / 2^-28 of that, and draws nearer to a border are left out."""
    rows = 60
    d = Drafts([2] * rows, V, seed=V, store=store, probs="f32", spread=1.0, peak=False)
    x = d.logits.astype(np.float64)
    p = np.exp(x - x.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    d.probs = p.astype(np.float32)
    at = np.arange(0, 2 * rows, 2)
    d.probs[at, d.tokens[at + 1]] *= 2
    d.uniform[at] = 0.9
    rest = np.maximum(p - d.probs, 0.0)[at].sum(1)
    assert (rest > 2.0 ** -28).all() and (rest < 2.0 ** -20).all()
    out = [put(cuda, np.zeros(rows, np.uint32)) for _ in range(2)]
    u32 = lambda a: put(cuda, np.asarray(a, np.uint32))[0]
    cuda.verify_drafts(put(cuda, d.logits, store)[0], u32(d.tokens), u32(d.starts), put(cuda, d.uniform)[0], probs=put(cuda, d.probs)[0], max_new=2, out=(out[0][0], out[1][0], None))
    want, near = plain_verify(d.logits, d.probs, d.tokens, d.starts, d.uniform, d.heat, d.lens, drawn=2.0 ** -16)
    assert len(near) < rows / 3
    for r in set(range(rows)) - near:
        assert (back(cuda, out[0][1])[r], back(cuda, out[1][1])[r]) == want[r][:2], r


# ---------------------------------------------------------------- attention over shared prefixes


@pytest.fixture
def always(cuda):
    """Prefixes are read once however little that saves."""
    cuda.set_option("shared_prefix", 2)
    yield cuda
    cuda.set_option("shared_prefix", 1)


class Shared:
    """Groups (rows, shared tokens), between them rows of none (shared None); new[r] tokens of row r, `own[r]` cached ones behind the prefix with them.  Full pages of a prefix
    are one for all rows, its begun page is copied."""

    def __init__(self, groups, new, own, page, seed=0, spare=0, extra=1):
        rng = self.rng = np.random.default_rng(seed)
        self.page, self.new = page, new
        first, shared, prefix = [], [], []
        r = 0
        for n, s in groups:
            if s is not None:
                if first and first[-1] != r:   # rows of none in between: a group that shares nothing
                    shared.append(0)
                    first.append(r)
                elif not first:
                    first.append(r)
                shared.append(s)
                first.append(r + n)
            prefix += [s or 0] * n
            r += n
        self.groups, self.shared = first or [0], shared
        self.total = [p + o for p, o in zip(prefix, own)]
        self.prefix = prefix
        rows = len(new)
        self.starts = np.concatenate([[0], np.cumsum(new)])
        self.M = int(self.starts[-1]) + spare
        self.cols = max(-(-t // page) for t in self.total) + extra
        self.n_pages = rows * self.cols + 3
        self.table = rng.permutation(self.n_pages)[:rows * self.cols].reshape(rows, self.cols)
        r = 0
        for n, s in groups:
            if s:
                self.table[r:r + n, :s // page] = self.table[r, :s // page]
            r += n

    def pool(self, nkv, d, store, stale):
        """Pages whose places that are nobody's hold `stale`."""
        x = rounded(self.rng.standard_normal((self.n_pages, nkv, self.page, d)), store)
        used = np.zeros((self.n_pages, self.page), bool)
        begin = 0
        for r, t in enumerate(self.total):
            s = self.prefix[r]
            if not (r and s == self.prefix[r - 1] and (self.table[r, :s // self.page] == self.table[r - 1, :s // self.page]).all() and self.same_group(r)):
                begin = r
            c, k = divmod(s, self.page)
            if k:
                x[self.table[r, c], :, :k] = x[self.table[begin, c], :, :k]
            at = np.arange(t)
            used[self.table[r, at // self.page], at % self.page] = True
        if stale is not None:
            x.transpose(0, 2, 1, 3)[~used] = stale
        return x

    def same_group(self, r):
        return any(a < r < b for a, b in zip(self.groups, self.groups[1:]))

    def gather(self, pages, r):
        at = np.arange(self.total[r])
        return pages[self.table[r, at // self.page], :, at % self.page]


def check_shared(B, b, store, nh, nkv, d, window=0, cap=0.0, scale=0.0, spread=1.5, stale=np.nan, strided=False, offset=None, max_new=None, max_shared=None, repeat=1):
    import torch
    rng = b.rng
    k, v = (b.pool(nkv, d, store, stale) for _ in range(2))
    q = rounded(rng.standard_normal((b.M, nh, d)) * spread, store)
    old = rounded(rng.standard_normal((b.M, nh, d)), store)
    out, kd, vd = put(B, old, store), put(B, k, store), put(B, v, store)
    if strided or offset is not None:
        flat = torch.zeros(b.M * (nh + 3) * (d + 8) + (offset or 0), device="cuda").to(kd[1].dtype)
        wide = flat[offset or 0:].reshape(b.M, nh + 3, d + 8)[:, :nh, :d] if strided else flat[offset:offset + q.size].reshape(q.shape)
        wide.copy_(torch.from_numpy(q))
        torch.cuda.synchronize()
        qd = (B.from_device(wide), flat)
    else:
        qd = put(B, q, store)
    table, starts, lens, groups, shared = (put(B, np.asarray(x, np.uint32)) for x in (b.table, b.starts, b.total, b.groups, b.shared))
    most, longest = max(b.new) if max_new is None else max_new, max(b.shared + [1]) if max_shared is None else max_shared
    work = B.paged_shared_work(qd[0], kd[0], table[0], groups[0], max_new=most, max_shared=longest)
    for _ in range(repeat):
        B.paged_shared_attention(qd[0], kd[0], vd[0], table[0], starts[0], lens[0], groups[0], shared[0], work, max_new=most, max_shared=longest, scale=scale,
                                 window=window, softcap=cap, out=out[0])
    got = back(B, out[1])
    want, lim = old.astype(np.float64), np.zeros((b.M, nh, d))
    f = scale or 1.0 / math.sqrt(d)
    for r, (n, t) in enumerate(zip(b.new, b.total)):
        kk, vv = (b.gather(x, r).astype(np.float64) for x in (k, v))
        for i in range(n):
            m, pos = int(b.starts[r]) + i, t - n + i
            lo = max(0, pos - window + 1) if window else 0
            want[m], mass, size = attention(q[m].astype(np.float64), kk[lo:pos + 1], vv[lo:pos + 1], pos - lo, f, 0, cap)
            off = 2 * (d + 6) * F32 * size[:, None] + (pos - lo + 24) * F32
            lim[m] = off * np.abs(vv[lo:pos + 1]).max() + (BF16 * (np.abs(want[m]) + 2 * mass) * (1 + 2.0 ** -7) if store == "bf16" else 0)
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4], np.abs(got - want).max())
    return work.shape[0]


# (rows, shared tokens) of the groups, new tokens, own cached tokens with them
GROUPS = [([(1, 1)], [1], [1]), ([(3, 40)], [1, 1, 1], [1, 9, 30]), ([(2, 129), (3, 64)], [1, 2, 3, 1, 0], [5, 2, 40, 1, 0]),
          ([(2, None), (4, 300), (1, None), (2, 77)], [1, 1, 4, 1, 2, 1, 3, 1, 1], [100, 3, 4, 70, 20, 1, 33, 200, 1]),
          ([(9, 513)], [1] * 9, [1 + 11 * r for r in range(9)]), ([(40, 200), (1, 5), (3, 0)], [1] * 44, [1 + r for r in range(44)]),
          ([(3, 640)], [5, 8, 2], [8, 64, 65]), ([(2, None)], [1, 2], [30, 40])]


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (8, 1, 128), (2, 2, 256), (3, 3, 24), (6, 2, 96), (32, 4, 128), (8, 2, 40), (5, 1, 64)])
@pytest.mark.parametrize("window,cap", [(0, 0.0), (70, 0.0), (0, 3.0), (33, 20.0)])
def test_shared_attention(always, store, nh, nkv, d, window, cap):
    for i, (groups, new, own) in enumerate(GROUPS):
        check_shared(always, Shared(groups, new, own, (8, 16, 64, 256)[i % 4], seed=i, spare=i % 3), store, nh, nkv, d, window, cap, scale=0.0 if i % 3 else 0.3, strided=i % 2 == 1)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (8, 2, 128), (2, 1, 256)])
@pytest.mark.parametrize("page", [8, 32, 1024])
def test_shared_attention_many_chunks(always, store, nh, nkv, d, page):
    """Prefixes of many chunks and of hardly more than some, that end anywhere."""
    for i, shared in enumerate((127, 128, 129, 256, 1000, 3001)):
        b = Shared([(3, shared), (2, shared // 2)], [1, 2, 1, 1, 3], [1, 5, 70, 33, 3], page, seed=i)
        floats = check_shared(always, b, store, nh, nkv, d, repeat=2)
        assert shared < 1000 or floats > 2 * b.M * nh * (d + 2)   # (several chunks)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(4, 1, 64), (16, 2, 128), (4, 2, 256)])
def test_shared_attention_many_queries(always, store, nh, nkv, d):
    """Groups whose queries fill more than a tile, and rows that fill one by themselves."""
    check_shared(always, Shared([(70, 300), (20, 129)], [1 + r % 4 for r in range(90)], [4 + r for r in range(90)], 16, seed=1), store, nh, nkv, d)
    check_shared(always, Shared([(3, 500)], [150, 3, 40], [150, 60, 41], 16, seed=2), store, nh, nkv, d)
    check_shared(always, Shared([(1, 200)] * 50, [1] * 50, [2] * 50, 16, seed=3), store, nh, nkv, d)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 150])
def test_shared_attention_many_rows(always, store, window):
    """More rows than are looked up at a time, many of them without tokens; many groups, and more than share."""
    rng = np.random.default_rng(window)
    new = [int(x) for x in rng.integers(0, 3, 1500)]
    check_shared(always, Shared([(1500, 140)], new, [n + 2 for n in new], 32, seed=1), store, 2, 1, 64, window)
    new = [int(x) for x in rng.integers(0, 2, 150)]
    floats = check_shared(always, Shared([(2, 64 + g) for g in range(75)], new, [n + 2 for n in new], 32, seed=2), store, 4, 2, 64, window)
    assert floats > 1
    assert check_shared(always, Shared([(1, 40)] * 300, [1] * 300, [3] * 300, 8, seed=3), store, 4, 2, 64, window) == 1


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 5, 64, 150])
def test_shared_attention_tokens_inside_the_prefix(always, store, window):
    """New tokens that stand before the prefix's end, rows that end there, and rows shorter than that."""
    b = Shared([(4, 200)], [3, 5, 1, 8], [2, 0, 30, 4], 16, seed=4)
    assert [t - n for n, t in zip(b.new, b.total)][1] < 200
    for d in (64, 128):
        check_shared(always, b, store, 4, 2, d, window)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("offset", [1, 2, 8])
def test_shared_attention_of_unaligned_queries(always, store, offset):
    for d in (64, 128, 40):
        check_shared(always, Shared([(4, 200), (2, 70)], [1, 2, 3, 1, 1, 1], [3, 9, 30, 1, 5, 6], 16, seed=offset), store, 4, 2, d, offset=offset)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
def test_shared_attention_without_its_numbers(always, store):
    """max_new and max_shared not known: the packed tokens and the table's width stand for them."""
    for new in ([1, 2, 3, 1, 1, 1], [1, 20, 3, 1, 1, 1]):
        b = Shared([(4, 200), (2, 70)], new, [3, 29, 30, 1, 5, 6], 16, seed=6, extra=40)
        check_shared(always, b, store, 4, 2, 64, max_new=0, max_shared=0)
        check_shared(always, b, store, 4, 2, 128, max_new=0, max_shared=200)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
def test_shared_attention_groups_that_cannot_be(always, store):
    """Such a group's rows are left as they were, and the others are not."""
    B = always
    nh, nkv, d = 4, 2, 64
    for what in ("order", "rows", "shared", "starts"):
        b = Shared([(2, 100), (2, 150)], [1, 1, 1, 2], [5, 6, 7, 8], 16, seed=7)
        k, v = (put(B, b.pool(nkv, d, store, None), store) for _ in range(2))
        groups, shared, starts = list(b.groups), list(b.shared), b.starts.copy()
        if what == "order":
            groups = [0, 4, 2]
        elif what == "rows":
            groups = [0, 2, 5]
        elif what == "shared":
            shared[1] = 151
        else:
            starts[4] = 99
        q, out = put(B, rounded(b.rng.standard_normal((b.M, nh, d)), store), store), put(B, np.full((b.M, nh, d), 7.0, np.float32), store)
        up = [put(B, np.asarray(x, np.uint32))[0] for x in (b.table, starts, b.total, groups, shared)]
        work = B.paged_shared_work(q[0], k[0], up[0], up[3], max_new=2, max_shared=150)
        B.paged_shared_attention(q[0], k[0], v[0], *up, work, max_new=2, max_shared=150, out=out[0])
        raises_index(B)
        got = back(B, out[1])
        assert np.isfinite(got).all()
        if what != "order":
            assert (got[:2] != 7.0).all()
        if what in ("rows", "shared"):
            assert (got[2:] == 7.0).all()
    # pages that do not exist count as zeros, and are not read
    b = Shared([(2, 100)], [1, 1], [5, 6], 16, seed=7)
    k, v = (put(B, b.pool(nkv, d, store, None), store) for _ in range(2))
    b.table[0, 2] = b.n_pages + 4
    q, out = put(B, rounded(b.rng.standard_normal((b.M, nh, d)), store), store), put(B, np.full((b.M, nh, d), 7.0, np.float32), store)
    up = [put(B, np.asarray(x, np.uint32))[0] for x in (b.table, b.starts, b.total, b.groups, b.shared)]
    work = B.paged_shared_work(q[0], k[0], up[0], up[3], max_new=1, max_shared=100)
    B.paged_shared_attention(q[0], k[0], v[0], *up, work, max_new=1, max_shared=100, out=out[0])
    raises_index(B)
    assert np.isfinite(back(B, out[1])).all()


@gpu
@pytest.mark.parametrize("store,nh,nkv,d,rows,shared", [("bf16", 8, 8, 128, 12, 800), ("f32", 4, 2, 64, 24, 1500), ("bf16", 4, 4, 256, 10, 1000)])
def test_shared_attention_where_it_saves_enough(cuda, store, nh, nkv, d, rows, shared):
    """Without the option: prefixes that are read once, and the same ones row by row."""
    b = Shared([(rows, shared)], [1 + r % 2 for r in range(rows)], [2 + 5 * r for r in range(rows)], 32, seed=rows)
    assert check_shared(cuda, b, store, nh, nkv, d) > 1
    try:
        cuda.set_option("shared_prefix", 0)
        assert check_shared(cuda, b, store, nh, nkv, d) == 1
    finally:
        cuda.set_option("shared_prefix", 1)
    assert check_shared(cuda, Shared([(2, shared)], [1, 1], [2, 5], 32), store, nh, nkv, d) == 1


def sees(b, where, keep=None):
    """Packed tokens that see cached position `where` of row `keep` (of every row of its group, where that is shared)."""
    rows = [r for r in range(len(b.new)) if r == keep or (where < min(b.prefix[keep], b.prefix[r]) and group_of(b, r) == group_of(b, keep))]
    return [int(b.starts[r]) + i for r in rows for i in range(b.new[r]) if b.total[r] - b.new[r] + i >= where]


def group_of(b, r):
    return sum(g <= r for g in b.groups)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("new", [[1] * 7, [3, 1, 2, 4, 3, 1, 2]])
def test_shared_attention_of_what_is_no_number(always, store, nh, nkv, d, new):
    """NaN and infinities in a query, in a shared key and value, and in a key of the row's own: who sees them gets NaN where cg_paged_attention gives it, and
    nobody else does.  The others' outputs are within the bound of check_shared of the formula's with and without, so within twice that of each other."""
    B, rep = always, nh // nkv
    b = Shared([(4, 700), (3, 300)], new, [5 + 9 * r for r in range(7)], 16, seed=d)
    k, v = (b.pool(nkv, d, store, None) for _ in range(2))
    q = rounded(b.rng.standard_normal((b.M, nh, d)) * 1.5, store)
    table, starts, lens, groups, shared = (put(B, np.asarray(x, np.uint32))[0] for x in (b.table, b.starts, b.total, b.groups, b.shared))
    most = max(new)

    def outputs(q, k, v):
        both = []
        for option in (2, 0):
            B.set_option("shared_prefix", option)
            Q, K, V, out = (put(B, x, store) for x in (q, k, v, np.zeros_like(q)))
            work = B.paged_shared_work(Q[0], K[0], table, groups, max_new=most, max_shared=700)
            assert (work.shape[0] > 1) == (option == 2)
            B.paged_shared_attention(Q[0], K[0], V[0], table, starts, lens, groups, shared, work, max_new=most, max_shared=700, out=out[0])
            both.append(back(B, out[1]))
        B.set_option("shared_prefix", 2)
        return both

    clean = outputs(q, k, v)[0]
    assert np.isfinite(clean).all()
    size = np.abs(q.astype(np.float64)).sum(2).max() * np.abs(k).max() / math.sqrt(d)
    near = 2 * np.abs(v).max() * (2 * (d + 6) * F32 * size + 1000 * F32 + (4 * BF16 if store == "bf16" else 0))
    place = lambda r, p: (b.table[r, p // b.page], slice(None), p % b.page)
    for what, bad in [("query", np.nan), ("query", np.inf), ("key", np.nan), ("key", np.inf), ("own", np.nan), ("value", np.nan), ("value", np.inf)]:
        Q, K, V = q.copy(), k.copy(), v.copy()
        touched = np.zeros((b.M, nh, d), bool)
        m = int(b.starts[2]) + new[2] - 1
        if what == "query":
            Q[m, 1, 7] = bad
            touched[m, 1] = True
        elif what == "own":
            at = b.total[1] - new[1]
            K[place(1, at)][0, 3] = bad
            touched[sees(b, at, 1), :rep] = True
        elif what == "key":
            K[place(4, 150)][1, 3] = bad
            touched[sees(b, 150, 4), rep:] = True
            if bad == np.inf:   # (no number where the query's component is above 0; below it nothing is left of that key)
                Q[..., 3] = np.abs(Q[..., 3]) + 0.5
        else:
            for r in range(4):   # (every row has its own copy of the prefix's begun page)
                V[place(r, 699)][0, 5] = bad
            touched[sees(b, 699, 0), :rep, 5] = True
        assert touched.any() and not touched.all()
        got, row_by_row = outputs(Q, K, V)
        # (of infinite values there are infinities or, where a probability has two parts, NaN)
        none, same = (~np.isfinite(x) if what == "value" else np.isnan(x) for x in (got, row_by_row))
        assert np.array_equal(none, touched), (what, bad, np.argwhere(none != touched)[:4])
        assert np.array_equal(none, same), (what, bad)
        if (what, bad) != ("key", np.inf):
            assert (np.abs(got - clean)[~touched] <= near).all(), (what, bad)


@gpu
@pytest.mark.parametrize("store,offset,rows,nh,nkv,shared", [("f32", None, 8, 32, 8, 2500), ("f32", None, 8, 32, 8, 5000), ("f32", None, 16, 4, 2, 10000), ("bf16", 1, 8, 32, 8, 4000),
                                                            ("bf16", 1, 8, 32, 8, 8000)])
@pytest.mark.parametrize("window", [0, 3000])
def test_shared_attention_chunks_that_begin_inside_a_tile(cuda, store, offset, rows, nh, nkv, shared, window):
    """Chunks of 192 and 320 keys of heads of 64, of which few queries take 128 at a time: every other one begins in the middle of a tile."""
    cuda.set_option("shared_prefix", 1 if window == 0 and store == "f32" else 2)
    try:
        b = Shared([(rows, shared)], [1] * rows, [2 + r for r in range(rows)], 64, seed=shared)
        assert check_shared(cuda, b, store, nh, nkv, 64, window=window, offset=offset) > 2 * b.M * nh * 66
    finally:
        cuda.set_option("shared_prefix", 1)


@gpu
@pytest.mark.parametrize("store,nh,nkv,d", [("f32", 32, 8, 64), ("bf16", 32, 8, 64), ("bf16", 16, 4, 256)])
def test_one_workspace_for_all_smaller_steps(always, store, nh, nkv, d):
    """Made for a step in which rows have drafts, used by steps with a token each, with rows that have none, and with shorter prefixes; against the same rows read for
    themselves.  Both are within the bound of check_shared, which is less than (2 (d + 6) size + t + 24) 2^-24 (and 4 2^-8 in bf16) of the largest value."""
    import torch
    B, rows, page, T = always, 40, 64, 3200
    gen = torch.Generator(device="cuda").manual_seed(d)
    dtype = torch.float32 if store == "f32" else torch.bfloat16
    cols = T // page + 1
    n = T // page + rows
    pages = [torch.randn(n, nkv, page, d, generator=gen, device="cuda").to(dtype) for _ in range(2)]
    ids = torch.randperm(n, generator=gen, device="cuda").int()
    table = torch.cat([ids[:T // page].repeat(rows, 1), ids[T // page:, None]], 1).contiguous()
    torch.cuda.synchronize()
    k, v, tab = (B.from_device(x) for x in (*pages, table))
    u32 = lambda a: put(B, np.asarray(a, np.uint32))[0]
    q_of = lambda M: torch.randn(M, nh, d, generator=gen, device="cuda").to(dtype)
    steps = [(4, 40, T), (4, 17, T), (1, 40, T), (4, 40, 1900), (1, 33, T), (1, 32, T), (2, 16, T), (1, 31, T), (1, 9, T), (1, 1, T), (1, 32, 1900), (1, 33, 130)]
    rooms = [B.paged_shared_work(B.from_device(q_of(each * count)), k, tab, u32([0, rows]), max_new=each, max_shared=T) for each, count in ((4, 40), (1, 33))]
    for (each, count, shared), room in [(x, rooms[0]) for x in steps] + [(x, rooms[1]) for x in steps[4:]]:
        new = [each if r < count else 0 for r in range(rows)]
        M = sum(new)
        Q = q_of(M)
        starts, lens = np.concatenate([[0], np.cumsum(new)]), [T + 10 if x else 0 for x in new]
        outs = [torch.zeros(M, nh, d, device="cuda", dtype=dtype) for _ in range(2)]
        torch.cuda.synchronize()
        at, ln, q = u32(starts), u32(lens), B.from_device(Q)
        B.paged_shared_attention(q, k, v, tab, at, ln, u32([0, rows]), u32([shared]), room, max_new=each, max_shared=shared, out=B.from_device(outs[0]))
        B.paged_attention(q, k, v, tab, at, ln, max_new=each, out=B.from_device(outs[1]))
        B.sync()
        size = float(Q.double().abs().sum(2).max() * pages[0].abs().max()) / math.sqrt(d)
        near = 2 * float(pages[1].abs().max()) * ((2 * (d + 6) * size + T + 34) * F32 + (4 * BF16 if store == "bf16" else 0))
        assert float((outs[0].double() - outs[1].double()).abs().max()) <= near, (each, count, shared)


def shared_launches(B, store, nh, nkv, d, new, shared, own=100, groups=1, window=0, max_new=None, page=64):
    """Launches of a call over rows behind one prefix: 3 where it is read once, 1 where rows read it for themselves."""
    import torch
    dtype, rows = torch.float32 if store == "f32" else torch.bfloat16, len(new)
    cols = -(-(shared + max(max(new), own)) // page)
    pages = [torch.zeros(cols, nkv, page, d, device="cuda", dtype=dtype) for _ in range(2)]
    q = torch.zeros(sum(new), nh, d, device="cuda", dtype=dtype)
    torch.cuda.synchronize()
    u32 = lambda a: put(B, np.asarray(a, np.uint32))[0]
    at = u32([g * rows // groups for g in range(groups + 1)])
    h = [B.from_device(x) for x in (q, *pages)] + [u32(x) for x in (np.tile(np.arange(cols), (rows, 1)), np.concatenate([[0], np.cumsum(new)]), [shared + max(n, own) for n in new])]
    most = max(new) if max_new is None else max_new
    work, out = B.paged_shared_work(h[0], h[1], h[3], at, max_new=most, max_shared=shared), B.from_device(torch.empty_like(q))
    B.sync()
    before = B.launch_count()
    B.paged_shared_attention(*h, at, u32([shared] * groups), work, max_new=most, max_shared=shared, window=window, out=out)
    B.sync()
    return B.launch_count() - before


@gpu
@pytest.mark.parametrize("store,nh,nkv,d", [("bf16", 8, 4, 128), ("bf16", 32, 8, 64), ("f32", 8, 4, 128)])
def test_shared_attention_with_a_prompt_in_the_batch(cuda, store, nh, nkv, d):
    """Rows that run share although one of the batch has a prompt, inside its group or outside all, or it is not known how many tokens a row has."""
    prompt, rows = 40, 24
    for groups, new in [([(rows + 1, 1500)], [1] * 10 + [prompt] + [1] * (rows - 10)), ([(rows, 1500), (1, None)], [1] * rows + [prompt])]:
        check_shared(cuda, Shared(groups, new, [n + 2 for n in new], 64, seed=nh), store, nh, nkv, d)
    check_shared(cuda, Shared([(rows, 1500)], [1] * rows, [3] * rows, 64, seed=nh), store, nh, nkv, d, max_new=0)
    assert shared_launches(cuda, store, nh, nkv, d, [1] * rows + [prompt], 1500) == 3
    assert shared_launches(cuda, store, nh, nkv, d, [1] * 64, 1500, max_new=0) == 3
    assert shared_launches(cuda, store, nh, nkv, d, [1, prompt, 100], 30000) == 1


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
def test_shared_attention_reads_no_more_than_windows_would(cuda, store):
    """Rows whose windows reach over less than the prefix read it for themselves where that is less than the prefix once."""
    e = 4 if store == "f32" else 2
    for rows, shared, window, launches in [(2, 16000, 4096, 1), (14, 16000, 512, 1), (14, 16000, 1024, 1), (14, 16000, 4096, 3), (40, 16000, 1024, 3), (40, 16000, 20000, 3), (14, 16000, 0, 3)]:
        assert shared_launches(cuda, store, 8, 8 // e * 2, 128, [1] * rows, shared, window=window) == launches, (rows, shared, window)
    check_shared(cuda, Shared([(3, 5000)], [1, 2, 1], [4, 90, 3], 64, seed=1), store, 4, 2, 128, window=300)


@gpu
def test_shared_attention_counts_what_its_parts_cost(cuda):
    """Rows of several tokens behind a short prefix read it for themselves where the parts of their queries cost more than that: so much the rule has to save."""
    for nh, nkv, each, shared, launches in [(32, 4, 4, 500, 1), (32, 4, 8, 500, 1), (32, 4, 4, 5000, 3), (32, 8, 4, 500, 3), (32, 8, 8, 500, 1), (32, 8, 1, 500, 3)]:
        assert shared_launches(cuda, "bf16", nh, nkv, 128, [each] * 40, shared) == launches, (nkv, each, shared)


@gpu
@pytest.mark.parametrize("store,nh,nkv,d,most", [("bf16", 8, 2, 128, 1), ("bf16", 8, 2, 128, 5), ("bf16", 4, 2, 256, 1), ("bf16", 8, 2, 64, 2), ("f32", 4, 2, 64, 1), ("f32", 4, 1, 128, 8)])
def test_shared_attention_joins_what_is_complete(always, store, nh, nkv, d, most):
    """Calls back to back over a workspace that is filled with NaN before each: the rows' own keys are few and read long before the chunks are, and the last rows, whose
    blocks leave at once, have no tokens.  Every call's outputs are the same, and the formula's."""
    import torch
    B = always
    rows = 30
    b = Shared([(rows, 6000)], [1 + r % most if r < rows - 3 else 0 for r in range(rows)], [most + r % 3 for r in range(rows)], 64, seed=d)
    check_shared(B, b, store, nh, nkv, d, stale=0.0)
    k, v = (put(B, b.pool(nkv, d, store, 0.0), store) for _ in range(2))
    q, out = (put(B, rounded(b.rng.standard_normal((b.M, nh, d)), store), store) for _ in range(2))
    table, starts, lens, groups, shared = (put(B, np.asarray(x, np.uint32))[0] for x in (b.table, b.starts, b.total, b.groups, b.shared))
    n = B.paged_shared_work(q[0], k[0], table, groups, max_new=most, max_shared=6000).shape[0]
    room = torch.zeros(n, device="cuda")
    work, seen = B.from_device(room), []
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(B.stream)):
        for _ in range(40):
            room.fill_(float("nan"))
            B.paged_shared_attention(q[0], k[0], v[0], table, starts, lens, groups, shared, work, max_new=most, max_shared=6000, out=out[0])
            seen.append(out[1].clone())
    B.sync()
    torch.cuda.synchronize()
    assert torch.isfinite(seen[0]).all()
    assert all(torch.equal(x, seen[0]) for x in seen[1:])


@gpu
@pytest.mark.parametrize("store,nh,nkv,d", [("bf16", 4, 2, 64), ("bf16", 32, 8, 128), ("bf16", 4, 4, 256), ("bf16", 6, 2, 96), ("bf16", 16, 1, 128), ("f32", 4, 2, 64), ("f32", 8, 2, 128), ("f32", 4, 4, 256)])
@pytest.mark.parametrize("cap,window", [(0.0, 0), (30.0, 1500)])
def test_shared_attention_of_single_tokens_has_all_parts(always, store, nh, nkv, d, cap, window):
    """Whether a prefix is read once or by each row does not change how many bits count: the bounds of cg_paged_attention's single tokens (test_paged.py)."""
    B = always
    b = Shared([(9, 2000), (4, 900)], [1] * 13, [3 + 25 * r for r in range(13)], 16, seed=d)
    k, v = (b.pool(nkv, d, store, None) for _ in range(2))
    q = rounded(b.rng.standard_normal((b.M, nh, d)) * 2.0, store)
    table, starts, lens, groups, shared = (put(B, np.asarray(x, np.uint32))[0] for x in (b.table, b.starts, b.total, b.groups, b.shared))
    Q, K, V, out = (put(B, x, store) for x in (q, k, v, np.zeros_like(q)))
    work = B.paged_shared_work(Q[0], K[0], table, groups, max_new=1, max_shared=2000)
    B.paged_shared_attention(Q[0], K[0], V[0], table, starts, lens, groups, shared, work, max_new=1, max_shared=2000, softcap=cap, window=window, out=out[0])
    got, want = back(B, out[1]), np.zeros((b.M, nh, d))
    for r, t in enumerate(b.total):
        kk, vv = (b.gather(x, r).astype(np.float64) for x in (k, v))
        lo = max(0, t - window) if window else 0
        want[r] = attention(q[r].astype(np.float64), kk[lo:], vv[lo:], t - 1 - lo, 1.0 / math.sqrt(d), 0, cap)[0]
    if store == "bf16":
        assert off_from_rounded(got, want) <= 0.02
    else:
        assert relative(got, want) <= (2.0 + 1.0) * PARTS


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d,new,total", [(4, 2, 64, 100, 3000), (8, 4, 128, 70, 3000), (4, 2, 256, 63, 3000), (4, 2, 64, 1, 5000), (4, 2, 128, 2, 3000)])
def test_attention_of_a_query_that_is_no_number(cuda, store, nh, nkv, d, new, total):
    """One row, whose keys are shared out among blocks: NaN comes out of that token's head, and of nothing else."""
    rng = np.random.default_rng(d)
    cols = total // 8
    k, v = (put(cuda, rounded(rng.standard_normal((cols, nkv, 8, d)), store), store) for _ in range(2))
    q = rounded(rng.standard_normal((new, nh, d)), store)
    q[new // 2, 1, 5] = np.nan
    out = put(cuda, np.zeros((new, nh, d), np.float32), store)
    u32 = lambda a: put(cuda, np.asarray(a, np.uint32))[0]
    cuda.paged_attention(put(cuda, q, store)[0], k[0], v[0], u32(rng.permutation(cols)[None]), u32([0, new]), u32([total]), max_new=new, out=out[0])
    none = np.isnan(back(cuda, out[1]))
    assert none[new // 2, 1].all() and none.sum() == d


# ---------------------------------------------------------------- all of them together


@gpu
@pytest.mark.parametrize("heat,page", [(0.0, 8), (1.0, 16)])
def test_drafts_are_served_from_one_cache(always, heat, page):
    """Requests behind one system prompt, served with drafts: pages from a stack, append, attention over the shared prefix, verification, and lengths without
    what was rejected, until each has its tokens; against the same decisions made from 64-bit logits of whole sequences without a cache.  2 layers of f32
    sums of at most 128 products leave logits of some 10 within 1e-4, so decisions nearer to a border than 1e-3 are taken from the device."""
    import torch
    B = always
    rng = np.random.default_rng(page)
    hidden, nh, nkv, d, vocab, layers, T = 64, 4, 2, 32, 211, 2, 160
    W = net(rng, hidden, nh, nkv, d, vocab, layers)
    system, prompts = rng.integers(0, vocab, 2 * page), [rng.integers(0, vocab, n) for n in (5, 17, 1, 9)]
    R, cols, pages = len(prompts), T // page, 60
    cos_t, sin_t = B.rope_tables(10000.0, T, d)
    cos, sin = B.to_numpy(cos_t), B.to_numpy(sin_t)
    up = lambda a: B.from_numpy(np.ascontiguousarray(a))
    Wd = {"embed": up(W["embed"]), "head": up(W["head"]), "layers": [{n: up(a) for n, a in L.items()} for L in W["layers"]]}
    kc, vc = (torch.full((layers, pages, nkv, page, d), float("nan"), device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    pools = [(B.from_device(kc[i]), B.from_device(vc[i])) for i in range(layers)]
    u32 = lambda *a: put(B, np.asarray(a, np.uint32))
    free, n_free = u32(*rng.permutation(pages)), u32(pages)
    work = []

    def forward(tokens, table, starts, lens, most, groups):
        M = len(tokens)
        x = B.index(Wd["embed"], 0, B.from_numpy(np.uint32(tokens)))
        for L, (kp, vp) in zip(Wd["layers"], pools):
            y = B.reshape(B.linear(B.fused_rmsnorm(x, L["n"], 1e-6), L["qkv"]), (M, nh + 2 * nkv, d))
            q, k, v = B.slice(y, 1, 0, nh), B.slice(y, 1, nh, nkv), B.slice(y, 1, nh + nkv, nkv)
            q = B.paged_append(k, v, kp, vp, table, starts, lens, q=q, cos=cos_t, sin=sin_t, q_gain=L["qg"], k_gain=L["kg"], eps=1e-6)
            if groups is None:
                o = B.paged_attention(q, kp, vp, table, starts, lens, max_new=most)
            else:
                room = B.paged_shared_work(q, kp, table, groups[0], max_new=most, max_shared=len(system))
                work.append(room.shape[0])
                o = B.paged_shared_attention(q, kp, vp, table, starts, lens, *groups, room, max_new=most, max_shared=len(system))
            x = B.add(x, B.linear(B.reshape(o, (M, nh * d)), L["o"]))
        return B.linear(x, Wd["head"])

    # the system prompt, once
    one_table, one = u32(*([0] * cols))[0], {n: u32(v) for n, v in dict(lens=0, new=len(system), held=0).items()}
    one_table = B.reshape(one_table, (1, cols))
    starts1 = u32(0, 0)
    B.paged_assign(one["lens"][0], one["new"][0], page, one["held"][0], one_table, free[0], n_free[0], starts1[0])
    forward(system, one_table, starts1[0], one["lens"][0], len(system), None)
    prefix = B.to_numpy(one_table)[0, :2]
    assert back(B, one["held"][1]).tolist() == [2] and back(B, n_free[1]).tolist() == [pages - 2]
    # the requests, each with the prefix's pages in front
    table = np.zeros((R, cols), np.uint32)
    table[:, :2] = prefix
    table, first, held, lens = put(B, table), u32(*[2] * R), u32(*[2] * R), u32(*[len(system)] * R)
    starts, slots = u32(*[0] * (R + 1)), u32(*[0] * 256)
    groups = u32(0, R)[0], u32(len(system))[0]
    texts, made = [list(system) + list(p) for p in prompts], [0] * R
    goal, stood, near_any = 9, 0, 0
    feed = [list(p) for p in prompts]
    for step in range(40):
        done = [m >= goal for m in made]
        new = u32(*[0 if f else len(x) for f, x in zip(done, feed)])
        B.paged_assign(lens[0], new[0], page, held[0], table[0], free[0], n_free[0], starts[0], done=u32(*[int(f) for f in done])[0], first=first[0], slots=slots[0])
        at = back(B, starts[1])
        active = [x if not f else [] for f, x in zip(done, feed)]
        assert at.tolist() == np.concatenate([[0], np.cumsum([len(x) for x in active])]).tolist()
        if all(done):
            break
        tokens = [t for x in active for t in x]
        slot, tab = back(B, slots[1]), back(B, table[1])
        for r, x in enumerate(active):
            end = int(back(B, lens[1])[r])
            assert slot[at[r]:at[r + 1]].tolist() == [tab[r, p // page] * page + p % page for p in range(end - len(x), end)]
        logits = forward(tokens, table[0], starts[0], lens[0], max(len(x) for x in active), groups)
        # a prompt's last token is drawn from, drafts are judged
        if step == 0:
            places = [int(at[r + 1]) - 1 for r in range(R)]
            logits, counts, judged = B.index(logits, 0, B.from_numpy(np.uint32(places))), [1] * R, [x[-1] for x in feed]
        else:
            counts, judged = [len(x) for x in active], tokens
        V = np.concatenate([[0], np.cumsum(counts)])
        uniform = np.minimum(rng.random(V[-1]).astype(np.float32), np.float32(1 - 2.0 ** -24))
        before = back(B, lens[1]).copy()
        out = u32(*[0] * R), u32(*[0] * R)
        B.verify_drafts(logits, B.from_numpy(np.uint32(judged)), put(B, V.astype(np.uint32))[0], put(B, uniform)[0], temperature=put(B, np.full(R, heat, np.float32))[0], lens=lens[0],
                        max_new=max(counts), out=(out[0][0], out[1][0], lens[0]))
        accepted, following, after = back(B, out[0][1]), back(B, out[1][1]), back(B, lens[1])
        # the same from whole sequences
        plain = np.zeros((V[-1], vocab))
        for r in range(R):
            for i in range(counts[r]):
                whole = texts[r] + ([] if step == 0 else active[r][1:1 + i])
                plain[V[r] + i] = plain_logits(W, np.array(whole), nh, nkv, d, cos, sin, 0)
        want, near = plain_verify(plain, None, np.array(judged), V, uniform, np.full(R, heat), before, 1e-3, 1e-3)
        near_any += len(near)
        for r in range(R):
            if counts[r] == 0:
                continue
            if r not in near:
                assert (accepted[r], following[r], after[r]) == want[r], (step, r)
            a = int(accepted[r])
            stood += a
            texts[r] += ([] if step == 0 else active[r][1:1 + a]) + [int(following[r])]
            made[r] += a + 1
            assert after[r] == len(texts[r]) - 1
            # the next drafts: the model's own, some of them wrong
            ahead, whole = [], list(texts[r])
            for i in range(int(rng.integers(0, 4))):
                t = int(np.argmax(plain_logits(W, np.array(whole), nh, nkv, d, cos, sin, 0)))
                ahead.append(t if rng.random() < 0.7 else int(rng.integers(0, vocab)))
                whole.append(ahead[-1])
            feed[r] = [int(following[r])] + ahead
    assert all(m >= goal for m in made) and stood > 0 and near_any <= 4 and min(work) > 1
    # all pages but the prefix's are free again, each once
    B.sync()
    count = int(back(B, n_free[1])[0])
    names = back(B, free[1])[:count]
    assert count == pages - 2 and len(set(names.tolist()) | set(prefix.tolist())) == pages and back(B, held[1]).tolist() == [2] * R


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
def test_captured_serving_steps(store):
    """The three operators in graphs, captured twice with a workspace each over the same buffers and replayed by turns while lengths, tables and inputs change."""
    import torch
    dtype = torch.bfloat16 if store == "bf16" else torch.float32
    S = torch.cuda.Stream()
    B = cg.CudaBackend(0, cg.PREC_F32, stream=S.cuda_stream)
    B.set_option("shared_prefix", 2)
    R, nh, nkv, d, page, cols, V, k = 6, 8, 2, 64, 16, 24, 3001, 3
    M = R * k
    gen = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    t = dict(q=rnd(M, nh, d), kp=rnd(R * cols, nkv, page, d), vp=rnd(R * cols, nkv, page, d), logits=rnd(M, V) * 3, probs=torch.softmax(rnd(M, V).float(), 1).to(dtype),
             uniform=torch.rand(M, generator=gen, device="cuda"), heat=torch.ones(R, device="cuda"), tokens=torch.randint(0, V, (M,), generator=gen, device="cuda").int(),
             lens=torch.full((R,), 200, device="cuda", dtype=torch.int32), new=torch.full((R,), k, device="cuda", dtype=torch.int32), done=ints(*[0] * R),
             held=torch.full((R,), 13, device="cuda", dtype=torch.int32), table=torch.randperm(R * cols, generator=gen, device="cuda").int().reshape(R, cols).contiguous(),
             free=torch.arange(R * cols, device="cuda").int(), n_free=ints(9), starts=ints(*[0] * (R + 1)), lens_out=ints(*[0] * R), held_out=ints(*[0] * R), n_free_out=ints(0),
             positions=ints(*[0] * M), slots=ints(*[0] * M), groups=ints(0, 2, R), shared=ints(170, 128), out=rnd(M, nh, d), accepted=ints(*[0] * R), next=ints(*[0] * R),
             left=ints(*[0] * R))
    torch.cuda.synchronize()
    h = {n: B.from_device(x) for n, x in t.items()}
    outs = [t[n] for n in ("table", "free", "starts", "lens_out", "held_out", "n_free_out", "positions", "slots", "out", "accepted", "next", "left")]

    def step(work):
        B.paged_assign(h["lens"], h["new"], page, h["held"], h["table"], h["free"], h["n_free"], h["starts"], done=h["done"], lens_out=h["lens_out"], held_out=h["held_out"],
                       n_free_out=h["n_free_out"], positions=h["positions"], slots=h["slots"])
        B.paged_shared_attention(h["q"], h["kp"], h["vp"], h["table"], h["starts"], h["lens_out"], h["groups"], h["shared"], work, max_new=k, max_shared=170, out=h["out"])
        B.verify_drafts(h["logits"], h["tokens"], h["starts"], h["uniform"], probs=h["probs"], temperature=h["heat"], lens=h["lens_out"], max_new=k,
                        out=(h["accepted"], h["next"], h["left"]))

    rooms = [B.paged_shared_work(h["q"], h["kp"], h["table"], h["groups"], max_new=k, max_shared=170) for _ in range(3)]
    B.sync()
    with torch.cuda.stream(S):
        step(rooms[2])   # (what is set up on first use)
    S.synchronize()
    reserved, graphs = B.bytes_reserved(), []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=S, capture_error_mode="relaxed"):
            step(rooms[i])
        graphs.append(g)
    moved = 0
    for i in range(6):
        with torch.cuda.stream(S):
            t["q"].copy_(rnd(M, nh, d)); t["logits"].copy_(rnd(M, V) * 3)
            t["uniform"].copy_(torch.rand(M, generator=gen, device="cuda"))
            t["lens"].fill_(172 + 5 * i); t["held"].fill_((172 + 5 * i + page - 1) // page)
            t["new"].copy_(torch.randint(0, k + 1, (R,), generator=gen, device="cuda"))
            t["done"].copy_((torch.arange(R, device="cuda") == i).int())
            t["heat"].fill_(float(i % 3))
            before = [x.clone() for x in outs]
            graphs[i % 2].replay()
        S.synchronize()
        replayed = [x.clone() for x in outs]
        for x, b in zip(outs, before):
            x.copy_(b)
        torch.cuda.synchronize()
        step(rooms[2])
        B.sync()
        torch.cuda.synchronize()
        for x, r in zip(outs, replayed):
            assert torch.equal(x, r)
        moved += int(t["starts"][-1])
    assert moved > 0 and B.bytes_reserved() == reserved
    B.close()


@gpu
def test_calls_on_two_streams_with_a_workspace_each():
    """Two contexts, each with its stream, at the same time over the same pages: every call's result is what it is alone."""
    import torch
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctx = [cg.CudaBackend(0, cg.PREC_F32, stream=s.cuda_stream) for s in streams]
    b = Shared([(20, 900)], [1 + r % 3 for r in range(20)], [3 + 9 * r for r in range(20)], 16, seed=1)
    nh, nkv, d = 8, 2, 128
    host_side = [b.pool(nkv, d, "bf16", None) for _ in range(2)] + [rounded(b.rng.standard_normal((b.M, nh, d)), "bf16") for _ in range(2)]
    calls = []
    for i, B in enumerate(ctx):
        B.set_option("shared_prefix", 2)
        k, v, q = (put(B, host_side[j], "bf16") for j in (0, 1, 2 + i))
        table, starts, lens, groups, shared = (put(B, np.asarray(x, np.uint32)) for x in (b.table, b.starts, b.total, b.groups, b.shared))
        out = put(B, np.zeros((b.M, nh, d), np.float32), "bf16")
        work = B.paged_shared_work(q[0], k[0], table[0], groups[0], max_new=3, max_shared=900)
        keep = (k, v, q, table, starts, lens, groups, shared, out, work)
        calls.append((lambda B=B, x=keep: B.paged_shared_attention(x[2][0], x[0][0], x[1][0], x[3][0], x[4][0], x[5][0], x[6][0], x[7][0], x[9], max_new=3, max_shared=900, out=x[8][0]), out[1]))
    alone = []
    for B, (call, out) in zip(ctx, calls):
        call()
        B.sync()
        alone.append(out.clone())
    torch.cuda.synchronize()
    for _ in range(30):
        for call, out in calls:
            call()
    for B in ctx:
        B.sync()
    torch.cuda.synchronize()
    for (call, out), want in zip(calls, alone):
        assert torch.equal(out, want)
    for B in ctx:
        B.close()


@gpu
def test_recorded_mode(cuda):
    """What is recorded runs before the calls that read it, and what they write is read by calls that are recorded behind them."""
    L = cg.CudaBackend(0, cg.PREC_F32)
    L.set_option("lazy", 1)
    b = Shared([(6, 200)], [1, 2, 1, 3, 1, 2], [5, 9, 1, 30, 2, 64], 16, seed=8)
    nh, nkv, d, V = 4, 2, 64, 515
    pool = [b.pool(nkv, d, "f32", None) for _ in range(2)]
    q = rounded(b.rng.standard_normal((b.M, nh, d)), "f32")
    c = Drafts([2, 1, 4], V, seed=1)
    s = requests(np.random.default_rng(5), 7, 16)
    results = []
    for B in (cuda, L):
        B.set_option("shared_prefix", 2)
        made = lambda x: B.cast(B.add(B.from_numpy(np.asarray(x, np.float32)), B.from_numpy(np.zeros(np.shape(x), np.float32))), cg.U32)   # (whole numbers, recorded)
        twice = lambda x: B.add(B.from_numpy(x), B.from_numpy(x))
        k, v = (put(B, x)[0] for x in pool)
        table, starts, lens, groups, shared = (made(x) for x in (b.table, b.starts, b.total, b.groups, b.shared))
        hq = twice(q)
        work = B.paged_shared_work(hq, k, table, groups, max_new=3, max_shared=200)
        o = B.paged_shared_attention(hq, k, v, table, starts, lens, groups, shared, work, max_new=3, max_shared=200)
        results.append([B.to_numpy(B.add(o, o))])
        got = B.verify_drafts(twice(c.logits), made(c.tokens), made(c.starts), B.mul(B.from_numpy(c.uniform), B.from_numpy(np.ones_like(c.uniform))), probs=twice(c.probs / 2),
                              temperature=twice(c.heat), lens=made(c.lens))
        results[-1] += [B.to_numpy(B.cast(x, cg.F32)) for x in got]
        held, n_free, free = made(s["held"]), made([s["n_free"]]), made(s["free"])
        tab, st, pos = made(s["table"]), B.zeros((8,), cg.U32), B.zeros((300,), cg.U32)
        le = made(s["lens"])
        B.paged_assign(le, made(s["new"]), 16, held, tab, free, n_free, st, done=made(s["done"]), first=made(s["first"]), positions=pos)
        results[-1] += [B.to_numpy(B.cast(x, cg.F32)) for x in (le, held, n_free, tab, st, pos)]
        B.set_option("shared_prefix", 1)
    for x, y in zip(*results):
        assert np.array_equal(x, y)
    assert L.lazy_stats()[0] > 0 and np.abs(results[0][0]).max() > 0 and results[0][8][-1] > 0
    L.close()


@gpu
@pytest.mark.parametrize("store,heat", [("f32", 1.0), ("bf16", 0.0)])
def test_prompts_begin_beside_drafts(cuda, store, heat):
    """Steps in which some rows run with drafts, one begins with its prompt and one waits for pages: what is judged is gathered from the packed tokens, a prompt's last one of
    its own.  Against the same steps on the host: lengths lose rejected drafts and nothing else, and what waited begins when pages come back."""
    B, rows, page, V, cols = cuda, 5, 8, 97, 12
    rng = np.random.default_rng(3)
    u32 = lambda a: put(B, np.asarray(a, np.uint32))
    n_pages = 30
    lens, held, first, done = np.array([40, 21, 0, 0, 16]), np.array([5, 3, 0, 0, 2]), np.array([0, 0, 0, 0, 2]), np.zeros(rows, int)   # (the last begins behind two shared pages)
    names = rng.permutation(n_pages)
    table = np.zeros((rows, cols), np.int64)
    at = 0
    for r in range(rows):
        table[r, :held[r]] = names[at:at + held[r]]
        at += held[r]
    stack = np.zeros(n_pages, np.int64)
    stack[:6] = names[at:at + 6]
    t = {n: u32(x) for n, x in dict(lens=lens, held=held, table=table, free=stack, n_free=[6], starts=[0] * (rows + 1), first=first).items()}
    feed = [[5, 6, 7, 8], [9], list(rng.integers(0, V, 11)), list(rng.integers(0, V, 40)), list(rng.integers(0, V, 4))]
    drafts, began = np.array([3, 0, 0, 0, 0]), [True, True, False, False, False]
    waited = 0
    for step in range(4):
        before, table_before, free_before, left = lens.copy(), table.copy(), stack.copy(), int(back(B, t["n_free"][1])[0])
        new = np.array([0 if done[r] else len(feed[r]) for r in range(rows)])
        want = plain_assign(before, new, done, first, held, table_before, free_before, left, page, 1 << 40)
        B.paged_assign(t["lens"][0], u32(new)[0], page, t["held"][0], t["table"][0], t["free"][0], t["n_free"][0], t["starts"][0], done=u32(done)[0], first=t["first"][0])
        starts = back(B, t["starts"][1])
        assert starts.tolist() == want[0]
        held, table, stack = np.array(want[2]), table_before, free_before
        places, counts = [], []
        for r in range(rows):
            counts.append(min(int(starts[r + 1] - starts[r]), 1 + int(drafts[r])))
            places += range(starts[r + 1] - counts[r], starts[r + 1])
        V0 = np.concatenate([[0], np.cumsum(counts)])
        tokens = np.array([x for r in range(rows) if starts[r + 1] > starts[r] for x in feed[r]], np.uint32)
        judged = B.index(B.from_numpy(tokens), 0, B.from_numpy(np.uint32(places)))
        logits = rounded(rng.standard_normal((len(places), V)) * 3, store)
        uniform = np.minimum(rng.random(len(places)).astype(np.float32), np.float32(1 - 2.0 ** -24))
        accepted, following, _ = out = *(u32([77] * rows) for _ in range(2)), t["lens"]
        B.verify_drafts(put(B, logits, store)[0], judged, u32(V0)[0], put(B, uniform)[0], temperature=put(B, np.full(rows, heat, np.float32))[0], lens=t["lens"][0],
                        max_new=4, out=[x[0] for x in out])
        verdicts, near = plain_verify(logits, None, tokens[places], V0, uniform, np.full(rows, heat), np.array(want[1]))
        assert not near
        B.sync()
        lens = back(B, t["lens"][1]).astype(np.int64)
        for r in range(rows):
            if counts[r] == 0:
                assert lens[r] == want[1][r]
                waited += not done[r]
                continue
            assert (back(B, accepted[1])[r], back(B, following[1])[r], lens[r]) == verdicts[r]
            assert lens[r] == before[r] + (int(back(B, accepted[1])[r]) + 1 if began[r] else len(feed[r]))
            began[r] = True
            drafts[r] = int(rng.integers(0, 4))
            feed[r] = [int(back(B, following[1])[r])] + list(rng.integers(0, V, drafts[r]))
        done[0] = step >= 1   # its pages go to the one that waits
    assert waited >= 1 and all(began) and done[0]


# ---------------------------------------------------------------- without a device


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """The library's entry points with a context and tensors that no device stands behind."""
    cg.load_library()
    out = str(tmp_path_factory.mktemp("serving") / "serving_host.so")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    tests = os.path.join(ROOT, "tests")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-I", os.path.join(ROOT, "catgrad-rs_b200", "csrc"), "-I", f"{cuda}/include", "-I", tests,
                           os.path.join(tests, "serving_host.cpp"), "-o", out, cg.library_path(), f"-Wl,-rpath,{os.path.dirname(cg.library_path())}", "-L", f"{cuda}/lib64", "-lcudart"])
    L = ctypes.CDLL(out)
    vp, i64, i64p = ctypes.c_void_p, ctypes.c_int64, ctypes.POINTER(ctypes.c_int64)
    L.host_ctx.restype = vp
    L.host_tensor.restype, L.host_tensor.argtypes = vp, [vp, ctypes.c_uint64, ctypes.c_int, ctypes.c_int, i64p, i64p]
    L.host_device.argtypes = [vp, ctypes.c_int]
    L.host_group_span.argtypes = [vp, vp, i64, i64, ctypes.c_int, i64, vp, vp, i64, i64, i64, vp, vp]
    L.host_position_of.argtypes, L.host_position_of.restype = [vp, vp, i64, i64, i64, i64], i64
    return L


SHAPE, DTYPE, INVALID, UNSUPPORTED = 1, 2, 3, 8


def refused(H, call, cases):
    for i, (want, kw) in enumerate(cases):
        assert call(**kw) == want, (i, want, H.lib.cg_last_error(H.ctx))


def test_assign_refusals(host):
    """Every call here is refused before anything is launched."""
    H = Host(host)
    u = lambda *d, **k: H.t(*d, store="u32", **k)
    order = ("lens", "new", "done", "first", "page", "most", "held", "n_free", "free", "table", "starts", "lens_out", "held_out", "n_free_out", "positions", "slots")

    def call(**kw):
        a = dict(lens=u(5), new=u(5), done=u(5), first=u(5), page=16, most=0, held=u(5), n_free=u(1), free=u(40), table=u(5, 8), starts=u(6), lens_out=u(5), held_out=u(5),
                 n_free_out=u(1), positions=u(99), slots=u(99))
        a.update(kw)
        return H._call(H.lib.cg_paged_assign, [ctypes.c_int64(a[n]) if n in ("page", "most") else a[n] for n in order])

    for name in ("lens", "new", "held", "n_free", "free", "table", "starts", "lens_out", "held_out", "n_free_out"):
        assert call(**{name: None}) == INVALID, name
    at = 7 << 44
    far = u(5)
    host.host_device(far, 1)
    refused(H, call, [(SHAPE, {n: u(4)}) for n in ("lens", "new", "done", "first", "held", "starts", "lens_out", "held_out", "n_free", "n_free_out")] +
            [(SHAPE, dict(table=u(40))), (SHAPE, dict(slots=u(98))), (SHAPE, dict(free=u(5, 8)))] +
            [(DTYPE, {n: H.t(5)}) for n in ("lens", "new", "done", "first", "held", "lens_out", "held_out")] + [(DTYPE, dict(table=H.t(5, 8))), (DTYPE, dict(free=H.t(40)))] +
            [(UNSUPPORTED, dict(page=p)) for p in (0, 4, 12, 2048, -16)] + [(INVALID, dict(most=-1)), (UNSUPPORTED, dict(table=u(5, 8, strides=[9, 1]))),
             (UNSUPPORTED, dict(lens=u(5, strides=[2]))), (INVALID, dict(lens=u(5, at=at), held_out=u(5, at=at))), (INVALID, dict(lens=u(5, at=at), lens_out=u(5, at=at, shift=4))),
             (INVALID, dict(table=u(5, 8, at=at), slots=u(99, at=at, shift=64))), (INVALID, dict(new=u(5, at=at), starts=u(6, at=at))), (INVALID, dict(done=far))])
    big = 65536
    assert call(lens=u(big), new=u(big), done=None, first=None, held=u(big), table=u(big, 8), starts=u(big + 1), lens_out=u(big), held_out=u(big)) == UNSUPPORTED


def test_verify_refusals(host):
    H = Host(host)
    u, t = (lambda *d, **k: H.t(*d, store="u32", **k)), H.t
    order = ("logits", "probs", "tokens", "starts", "uniform", "heat", "lens", "most", "accepted", "next", "lens_out")

    def call(**kw):
        a = dict(logits=t(9, 100), probs=t(9, 100, store="bf16"), tokens=u(9), starts=u(4), uniform=t(9), heat=t(3), lens=u(3), most=4, accepted=u(3), next=u(3), lens_out=u(3))
        a.update(kw)
        return H._call(H.lib.cg_verify_drafts, [ctypes.c_int64(a[n]) if n == "most" else a[n] for n in order])

    for name in ("logits", "tokens", "starts", "uniform", "accepted", "next", "lens", "lens_out"):
        assert call(**{name: None}) == INVALID, name
    at = 7 << 44
    far = u(9)
    host.host_device(far, 1)
    refused(H, call, [(SHAPE, dict(probs=t(9, 99))), (SHAPE, dict(probs=t(8, 100))), (SHAPE, dict(tokens=u(8))), (SHAPE, dict(uniform=t(8))), (SHAPE, dict(heat=t(4))),
                      (SHAPE, dict(accepted=u(4))), (SHAPE, dict(next=u(2))), (SHAPE, dict(lens_out=u(4))), (SHAPE, dict(starts=u(0))), (SHAPE, dict(logits=t(900))),
                      (SHAPE, dict(logits=t(9, 0), probs=None)), (DTYPE, dict(logits=u(9, 100))), (DTYPE, dict(tokens=t(9))), (DTYPE, dict(uniform=t(9, store="bf16"))),
                      (DTYPE, dict(heat=t(3, store="bf16"))), (DTYPE, dict(lens=t(3))), (INVALID, dict(most=-1)), (UNSUPPORTED, dict(logits=t(9, 100, strides=[200, 2]))),
                      (UNSUPPORTED, dict(logits=t(9, 100, strides=[99, 1]))), (UNSUPPORTED, dict(probs=t(9, 100, strides=[1, 9]))), (UNSUPPORTED, dict(tokens=u(9, strides=[2]))),
                      (UNSUPPORTED, dict(logits=t(9, (1 << 19) + 1), probs=None)), (INVALID, dict(accepted=u(3, at=at), next=u(3, at=at, shift=8))),
                      (INVALID, dict(tokens=u(9, at=at), lens_out=u(3, at=at))), (INVALID, dict(lens=u(3, at=at), lens_out=u(3, at=at, shift=4))), (INVALID, dict(tokens=far))])


def test_shared_attention_refusals(host):
    H = Host(host)
    u, t = (lambda *d, **k: H.t(*d, store="u32", **k)), (lambda *d, **k: H.t(*d, **{"store": "bf16", **k}))
    H.lib.cg_set_option.argtypes = [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_int64]
    assert H.lib.cg_set_option(H.ctx, b"shared_prefix", 2) == 0
    order = ("q", "k_pages", "v_pages", "table", "starts", "lens", "groups", "shared", "most", "longest", "scale", "window", "cap", "work", "out")
    work = 10 * 6 * 4 * 66

    def call(**kw):
        a = dict(q=t(6, 4, 64), k_pages=t(20, 2, 16, 64), v_pages=t(20, 2, 16, 64), table=u(3, 20), starts=u(4), lens=u(3), groups=u(3), shared=u(2), most=2, longest=300, scale=0.0, window=0,
                 cap=0.0, work=H.t(work), out=t(6, 4, 64))
        a.update(kw)
        return H._call(H.lib.cg_paged_shared_attention, [ctypes.c_int64(a[n]) if n in ("most", "longest", "window") else ctypes.c_float(a[n]) if n in ("scale", "cap") else a[n] for n in order])

    for name in ("q", "k_pages", "v_pages", "table", "starts", "lens", "groups", "shared", "work", "out"):
        assert call(**{name: None}) == INVALID, name
    at = 7 << 44
    far = u(3)
    host.host_device(far, 1)
    refused(H, call, [(SHAPE, dict(q=t(6, 5, 64), out=t(6, 5, 64))), (SHAPE, dict(shared=u(3))), (SHAPE, dict(groups=u(0))), (SHAPE, dict(groups=u(3, 1))), (SHAPE, dict(work=H.t(100))),
                      (SHAPE, dict(work=H.t(work, 1))), (SHAPE, dict(starts=u(5))), (DTYPE, dict(groups=t(3))), (DTYPE, dict(work=u(work))), (DTYPE, dict(work=t(work))),
                      (DTYPE, dict(out=t(6, 4, 64, store="f32"))), (INVALID, dict(most=-1)), (INVALID, dict(longest=-1)), (INVALID, dict(window=-1)), (INVALID, dict(cap=float("nan"))),
                      (UNSUPPORTED, dict(work=H.t(work, shift=4))), (UNSUPPORTED, dict(work=H.t(work, strides=[2]))), (UNSUPPORTED, dict(q=t(6, 4, 64, strides=[512, 128, 2]))),
                      (INVALID, dict(work=H.t(work, at=at), out=t(6, 4, 64, at=at))), (INVALID, dict(work=H.t(work, at=at), q=t(6, 4, 64, at=at, shift=64))),
                      (INVALID, dict(groups=u(3, at=at), out=t(6, 4, 64, at=at))), (INVALID, dict(groups=far))])
    # the workspace's size is what the call asks for
    f = H.lib.cg_paged_shared_floats
    f.restype, f.argtypes = ctypes.c_int64, [ctypes.c_void_p] * 5 + [ctypes.c_int64] * 2
    size = lambda q=t(6, 4, 64), k=t(20, 2, 16, 64), table=u(3, 20), groups=u(3), most=2, longest=300: f(H.ctx, q, k, table, groups, most, longest)
    n = size()
    assert n == 4 * 6 * 4 * 66 and call(work=H.t(n - 1)) == SHAPE     # (3 chunks of 128 keys, and the rows' own)
    assert size(most=33) == 0 or size(most=33) == n                    # (no row has more than all)
    assert size(q=t(99, 4, 64), most=33) == 0 and size(groups=u(1)) == 0 and size(q=t(0, 4, 64)) == 0
    assert [size(q=None), size(k=t(20, 2, 16)), size(q=t(6, 5, 64)), size(longest=-1), size(groups=u(0))] == [-1] * 5
    assert H.lib.cg_set_option(H.ctx, b"shared_prefix", 0) == 0 and size() == 0
    assert H.lib.cg_set_option(H.ctx, b"shared_prefix", 1) == 0 and size() == 0 and size(table=u(60, 4000), longest=9000) > 0


def test_shared_attention_room_for_smaller_steps(host):
    """What cg_paged_shared_floats gives for a step is no less than for any with fewer tokens, fewer of a row or shorter prefixes."""
    H = Host(host)
    f = H.lib.cg_paged_shared_floats
    f.restype, f.argtypes = ctypes.c_int64, [ctypes.c_void_p] * 5 + [ctypes.c_int64] * 2
    rows, cols = 48, 2000
    table = H.t(rows, cols, store="u32")
    for store in ("f32", "bf16"):
        for nh, nkv, d in [(32, 8, 128), (32, 8, 64), (32, 4, 128), (8, 4, 256), (4, 2, 64), (40, 1, 64), (12, 12, 40)]:
            k = H.t(9000, nkv, 16, d, store=store)
            for groups in (1, 3, 11):
                at = H.t(groups + 1, store="u32")
                size = lambda M, most, longest: f(H.ctx, H.t(M, nh, d, store=store), k, table, at, most, longest)
                for longest in (1500, 16001, 0):
                    # (all steps whose rows have up to `most` tokens and whose q is not padded)
                    steps = sorted((M, most) for M in (1, 7, 31, 32, 33, 48, 64, 65, 96, 130, 240, 500, 768, 2000) for most in (1, 2, 5, 16, 17, 500) if most <= M <= rows * most)
                    sizes = [size(M, most, longest) for M, most in steps]
                    assert sizes == sorted(sizes), (store, nh, d, groups, longest, list(zip(steps, sizes)))
                    assert sizes[-1] > 0 or longest == 1500
                assert size(240, 5, 16001) >= size(240, 5, 1500) and size(240, 5, 0) >= size(240, 5, 16001)


def test_tensors_that_another_context_has_recorded_are_refused(host):
    """They have no memory yet.  (In a process of its own, since a call that looked for that memory would end it.)"""
    out = ctypes.CDLL(host._name)._name
    r = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {os.path.dirname(__file__)!r}); import test_serving; test_serving.recorded_elsewhere({out!r})"],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


def recorded_elsewhere(path):
    L = ctypes.CDLL(path)
    L.host_ctx.restype = ctypes.c_void_p
    L.host_tensor.restype, L.host_tensor.argtypes = ctypes.c_void_p, [ctypes.c_void_p, ctypes.c_uint64, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_int64),
                                                                      ctypes.POINTER(ctypes.c_int64)]
    H = Host(L)
    other, lib = ctypes.c_void_p(L.host_ctx()), H.lib
    assert lib.cg_set_option(other, b"lazy", ctypes.c_int64(1)) == 0

    def waiting(shape, whole):
        t = ctypes.c_void_p()
        assert lib.cg_arange(other, ctypes.c_int64(int(np.prod(shape))), ctypes.byref(t)) == 0
        if not whole:
            assert lib.cg_cast(other, t, 0, ctypes.byref(t)) == 0
        assert lib.cg_reshape(other, t, (ctypes.c_int64 * len(shape))(*shape), len(shape), ctypes.byref(t)) == 0
        return t

    i64, f = ctypes.c_int64, ctypes.c_float
    calls = [(lib.cg_paged_assign, dict(lens=(5,), new=(5,), done=(5,), first=(5,), page=i64(16), most=i64(0), held=(5,), n_free=(1,), free=(40,), table=(5, 8), starts=(6,), lens_out=(5,),
                                        held_out=(5,), n_free_out=(1,), positions=(99,), slots=(99,)), ()),
             (lib.cg_verify_drafts, dict(logits=(9, 100), probs=(9, 100), tokens=(9,), starts=(4,), uniform=(9,), heat=(3,), lens=(3,), most=i64(4), accepted=(3,), next=(3,), lens_out=(3,)),
              ("logits", "probs", "uniform", "heat")),
             (lib.cg_paged_shared_attention, dict(q=(6, 4, 64), k=(20, 2, 16, 64), v=(20, 2, 16, 64), table=(3, 20), starts=(4,), lens=(3,), groups=(3,), shared=(2,), most=i64(2),
                                                  longest=i64(300), scale=f(0), window=i64(0), cap=f(0), work=(9999,), out=(6, 4, 64)), ("q", "k", "v", "work", "out"))]
    for fn, arguments, floats in calls:
        for name, shape in arguments.items():
            if isinstance(shape, tuple):
                a = [(waiting(x, n not in floats) if n == name else H.t(*x, store="f32" if n in floats else "u32")) if isinstance(x, tuple) else x for n, x in arguments.items()]
                assert H._call(fn, a) == INVALID, (fn, name)
                assert b"another context" in lib.cg_last_error(H.ctx), (fn, name)


def test_groups_that_cannot_be_are_not_followed(host):
    """group_span and position_of, on the CPU: what they let through lies inside the tensors, and a token's row is found among rows without tokens."""
    rng = np.random.default_rng(0)
    vp = lambda a: a.ctypes.data_as(ctypes.c_void_p)
    good = 0
    for _ in range(4000):
        rows, cols, lg, M = int(rng.integers(1, 7)), int(rng.integers(1, 5)), 4, int(rng.integers(0, 40))
        starts = np.concatenate([[0], np.cumsum(rng.integers(0, 8, rows))]).astype(np.uint32)
        if rng.random() < 0.3:
            starts[rng.integers(0, rows + 1)] = rng.choice([0, 5, 41, 0xFFFFFFFF])
        lens = (np.diff(starts.astype(np.int64)) + 50).astype(np.uint32)
        G = int(rng.integers(1, 4))
        groups = np.sort(rng.integers(0, rows + 1, G + 1)).astype(np.uint32)
        if rng.random() < 0.3:
            groups[rng.integers(0, G + 1)] = rng.choice([0, rows + 1, 0xFFFFFFFF])
        shared, most = rng.choice([0, 1, 16, 60, cols * 16, cols * 16 + 1, 0xFFFFFFFF], G).astype(np.uint32), int(rng.choice([1, 60, 1 << 40]))
        for g in range(G):
            out, err = np.zeros(5, np.int64), np.zeros(1, np.int32)
            ok = host.host_group_span(vp(starts), vp(lens), rows, cols, lg, M, vp(groups), vp(shared), G, most, g, vp(out), vp(err))
            a, b, s = int(groups[g]), int(groups[g + 1]), int(shared[g])
            can = a <= b <= rows and s <= min(most, cols * 16)
            can = can and int(starts[a]) <= int(starts[b]) <= M
            assert bool(ok) == can and err[0] == (0 if can else 1)
            if ok:
                good += 1
                assert out.tolist() == [a, b - a, int(starts[a]), int(starts[b]) - int(starts[a]), s]
                if (np.diff(starts[a:b + 1].astype(np.int64)) >= 0).all():
                    for r in range(a, b):
                        for m in range(int(starts[r]), int(starts[r + 1])):
                            assert host.host_position_of(vp(starts), vp(lens), rows, a, b - a, m) == int(lens[r]) - int(starts[r + 1]) + m
    assert good > 300


def test_joined_parts_are_waited_for_by_what_follows():
    """The kernels of the rows' own keys begin beside the chunks' and end behind them: each way out of them passes the dependency, so what waits for them
    waits for the chunks."""
    csrc = os.path.join(os.path.dirname(cg.__file__), "csrc")
    for name, kernel, wait in (("paged_fa.cu", "k_paged_fa(const", "dependency();"), ("paged_dec.cu", "k_paged_dec(const", "depend();"), ("paged_attn.cu", "k_paged_attn(Paged", "depend();")):
        body = open(os.path.join(csrc, name)).read()
        body = body[body.index(kernel):]
        body = body[:body.index("\n}\n")]
        lines = body.split("\n")
        at = [i for i, x in enumerate(lines) if x.strip().startswith("return;") or "return;" in x]
        # of a kernel's ways out, those of OWN have the wait in the two lines before; the others are of blocks of chunks, or of all keys
        for i in at + [len(lines)]:
            near = " ".join(lines[max(0, i - 3):i + 1])
            assert wait in near or "group_of_tile" in near or "x0 + x >= n * rep" in near or "MODE != ALL" in " ".join(lines[max(0, i - 5):i]), (name, lines[min(i, len(lines) - 1)])
