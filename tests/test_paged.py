"""The operators on a paged key/value cache and beam search against plain restatements in 64 bits.

Tolerances.  2^-24 is half a step of f32, 2^-8 of bf16, relative to the value; every bound below counts roundings.

* append, f32: a sum of at most 256 squares in a tree of 4 + 5 levels and 4 products (10 roundings, halved by the root), the root,
  the division, two products, then two products and a sum of the rotation: under 16 half steps of |u| + |w|, the pair's sizes.
  Kept in bf16 one half step of 2^-8 more.
* attention, f32: a score is a sum of d products (d + 2 roundings of the sum of their sizes), of which an exponential takes the
  difference to the maximum; a probability is then off by twice that, and the exponential's, the sums' and the division's
  roundings; the output by as much of the largest value.
* attention, bf16: products of bf16 values are exact in f32 and their sums as above; the probabilities may be rounded to bf16, above
  and below the fraction: 2 half steps of sum p |v|; the result one more.
"""
import ctypes
import gc
import math
import os
import subprocess
import sys
import threading
import weakref

import numpy as np
import pytest

from conftest import ROOT, cg

gpu = pytest.mark.gpu
F32, BF16 = 2.0 ** -24, 2.0 ** -8


# ---------------------------------------------------------------- on the GPU box


def put(B, a, store="f32"):
    """A device tensor of the library over torch memory, and that memory."""
    import torch
    a = np.asarray(a)
    t = torch.from_numpy(a.astype(np.int64) if a.dtype.kind in "ui" else a).cuda()
    t = t.to(torch.int32) if a.dtype.kind in "ui" else t.to({"f32": torch.float32, "bf16": torch.bfloat16}[store])
    t = t.contiguous()
    torch.cuda.synchronize()
    return B.from_device(t), t


def rounded(a, store):
    return cg.synth.bf16_round(np.asarray(a, np.float32)) if store == "bf16" else np.asarray(a, np.float32)


def back(B, t):
    B.sync()
    return t.float().cpu().numpy().astype(np.float64) if t.is_floating_point() else t.cpu().numpy()


class Batch:
    """Rows with new[r] of total[r] cached tokens, pages in any order; `spare` more packed tokens behind the last row, `extra` more columns and
    pages."""

    def __init__(self, new, total, page, seed=0, spare=0, extra=1):
        rng = np.random.default_rng(seed)
        self.new, self.total, self.page = new, total, page
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        self.M = int(self.starts[-1]) + spare
        self.cols = max(-(-t // page) for t in total) + extra
        self.n_pages = len(new) * self.cols + 3
        self.table = rng.permutation(self.n_pages)[:len(new) * self.cols].reshape(len(new), self.cols).astype(np.uint32)
        self.lens = np.array(total, np.uint32)
        self.rng = rng

    def up(self, B):
        return [put(B, x)[0] for x in (self.table, self.starts, self.lens)]

    def gather(self, pages, r):
        """[tokens, heads, d] of row r's cached tokens."""
        t = self.total[r]
        at = np.arange(t)
        return pages[self.table[r, at // self.page], :, at % self.page]

    def tokens(self):
        """(packed token, row, position)"""
        for r, (n, t) in enumerate(zip(self.new, self.total)):
            for i in range(n):
                yield int(self.starts[r]) + i, r, t - n + i


SHAPES = [([1], [1], 8), ([1, 1, 1], [5, 16, 17], 16), ([3, 0, 7, 1], [3, 0, 12, 64], 8), ([0, 0, 2], [9, 0, 2], 16), ([70, 1, 33], [70, 200, 40], 64),
          ([5] * 40, [5 + r for r in range(40)], 32)]


@gpu
@pytest.mark.parametrize("into,pages", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("nh,nkv,d,turned", [(4, 2, 64, 64), (3, 1, 128, 128), (8, 8, 256, 64), (2, 1, 8, 8), (5, 5, 24, 16), (4, 4, 40, 0), (7, 1, 96, 96)])
@pytest.mark.parametrize("norms,halves,plus", [(False, True, False), (True, True, False), (True, False, True)])
def test_append(cuda, into, pages, nh, nkv, d, turned, norms, halves, plus):
    for i, (new, total, page) in enumerate(SHAPES):
        check_append(cuda, Batch(new, total, page, seed=i, spare=i % 3), into, pages, nh, nkv, d, turned, norms, halves, plus)


def check_append(B, b, into, pages, nh, nkv, d, turned, norms, halves, plus, split=None):
    import torch
    rng = b.rng
    q, k, v = (rounded(rng.standard_normal((b.M, h, d)) * 1.5, into) for h in (nh, nkv, nkv))
    gains = [rounded(1.0 + 0.2 * rng.standard_normal(d), "f32") for _ in range(2)] if norms else [None, None]
    T = max(b.total) + 2
    angle = np.arange(T)[:, None] * 100.0 ** (-np.arange(turned // 2) / max(1, turned // 2))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    old = [rounded(rng.standard_normal((b.n_pages, nkv, b.page, d)), pages) for _ in range(2)]
    kp, vp = (put(B, x, pages) for x in old)
    q_old = rounded(rng.standard_normal((b.M, nh, d)), pages)
    qo = put(B, q_old, pages)
    if split is not None:   # three parts of one projection, from this place on
        both = torch.from_numpy(np.concatenate([q, k, v], 1)).to(torch.bfloat16 if into == "bf16" else torch.float32)
        flat = torch.zeros(both.numel() + split, dtype=both.dtype, device="cuda")
        flat[split:] = both.reshape(-1).cuda()
        whole = flat[split:].reshape(b.M, nh + 2 * nkv, d)
        torch.cuda.synchronize()
        qd, kd, vd = (B.from_device(x) for x in (whole[:, :nh], whole[:, nh:nh + nkv], whole[:, nh + nkv:]))
    else:
        qd, kd, vd = (put(B, x, into)[0] for x in (q, k, v))
    table, starts, lens = b.up(B)
    g = [None if x is None else put(B, x)[0] for x in gains]
    angles = [put(B, x)[0] for x in (cos, sin)] if turned else [None, None]
    B.paged_append(kd, vd, kp[0], vp[0], table, starts, lens, q=qd, q_out=qo[0], cos=angles[0], sin=angles[1], q_gain=g[0], k_gain=g[1], eps=1e-5,
                   plus_one=plus, rot_half=halves)
    want_q, want_k, want_v = q_old.astype(np.float64), old[0].astype(np.float64), old[1].astype(np.float64)
    lim_q, lim_k = np.zeros_like(want_q), np.zeros_like(want_k)
    n = turned // 2
    a0 = np.arange(n) if halves else 2 * np.arange(n)
    a1 = a0 + n if halves else a0 + 1
    for m, r, pos in b.tokens():
        done = []
        for x, gain in ((q[m], gains[0]), (k[m], gains[1])):
            x = x.astype(np.float64)
            if gain is not None:
                x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * (gain.astype(np.float64) + plus)
            size = np.abs(x)
            u, w = x[:, a0].copy(), x[:, a1].copy()
            c, s = cos[pos].astype(np.float64), sin[pos].astype(np.float64)
            x[:, a0], x[:, a1] = u * c - w * s, w * c + u * s
            size[:, a0] = size[:, a1] = np.abs(u) + np.abs(w)
            done.append((x, 16 * F32 * size + (BF16 * np.abs(x) * (1 + 2.0 ** -8) if pages == "bf16" else 0)))
        at, place = b.table[r, pos // b.page], pos % b.page
        want_q[m], lim_q[m] = done[0]
        want_k[at, :, place], lim_k[at, :, place] = done[1]
        want_v[at, :, place] = rounded(v[m], pages)
    assert (np.abs(back(B, qo[1]) - want_q) <= lim_q).all()
    assert (np.abs(back(B, kp[1]) - want_k) <= lim_k).all()
    assert np.array_equal(back(B, vp[1]), want_v)


@gpu
@pytest.mark.parametrize("into,pages", [("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (3, 1, 128), (2, 2, 40), (32, 4, 128), (5, 3, 32), (8, 4, 256), (32, 8, 64)])
@pytest.mark.parametrize("offset", [3, 8])
def test_append_parts_of_a_projection(cuda, into, pages, nh, nkv, d, offset):
    check_append(cuda, Batch([3, 1, 40], [3, 66, 41], 16, spare=2), into, pages, nh, nkv, d, d, True, True, False, split=offset)


@gpu
@pytest.mark.parametrize("nh,nkv,d", [(32, 4, 128), (32, 8, 64)])
def test_append_of_many_tokens(cuda, nh, nkv, d):
    """As many tokens as give each warp one."""
    check_append(cuda, Batch([2500, 1, 2400], [2500, 66, 2441], 64, spare=2), "bf16", "bf16", nh, nkv, d, d, True, False, False, split=0)


def attention(q, k, v, pos, scale, window, cap):
    """One query [heads, d] of kv-grouped keys [t, kv heads, d]: (output, sum p |v|, score size)."""
    rep = q.shape[0] // k.shape[1]
    t = np.arange(k.shape[0])
    seen = (t <= pos) & ((t > pos - window) if window else True)
    k, v = np.repeat(k[seen], rep, 1), np.repeat(v[seen], rep, 1)
    x = np.einsum("hd,thd->ht", q, k) * scale
    size = (np.einsum("hd,thd->ht", np.abs(q), np.abs(k)) * scale).max(1)
    if cap:
        x = cap * np.tanh(x / cap)
    p = np.exp(x - x.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    return np.einsum("ht,thd->hd", p, v), np.einsum("ht,thd->hd", p, np.abs(v)), size


def check_attention(B, b, store, nh, nkv, d, window=0, cap=0.0, scale=0.0, spread=1.0, stale=None, strided=False, max_new=None, check=None, offset=None):
    import torch
    rng = b.rng
    q = rounded(rng.standard_normal((b.M, nh, d)) * spread, store)
    k, v = (rounded(rng.standard_normal((b.n_pages, nkv, b.page, d)), store) for _ in range(2))
    if stale is not None:   # whatever is no row's token
        used = np.zeros((b.n_pages, b.page), bool)
        for r, t in enumerate(b.total):
            first = max(0, t - b.new[r] - window + 1) // b.page * b.page if window else 0
            at = np.arange(first, t)
            used[b.table[r, at // b.page], at % b.page] = True
        for x in (k, v):
            x.transpose(0, 2, 1, 3)[~used] = stale
    old = rounded(rng.standard_normal((b.M, nh, d)), store)
    out, kd, vd = put(B, old, store), put(B, k, store), put(B, v, store)
    if strided:
        wide = torch.zeros(b.M, nh + 3, d + 8, device="cuda").to(kd[1].dtype)
        wide[:, :nh, :d] = torch.from_numpy(q).cuda()
        torch.cuda.synchronize()
        qd = (B.from_device(wide[:, :nh, :d]), wide)
    elif offset is not None:   # from a place that no vector begins on
        flat = torch.zeros(q.size + offset, device="cuda").to(kd[1].dtype)
        flat[offset:] = torch.from_numpy(q).cuda().reshape(-1)
        torch.cuda.synchronize()
        qd = (B.from_device(flat[offset:].reshape(q.shape)), flat)
    else:
        qd = put(B, q, store)
    table, starts, lens = b.up(B)
    B.paged_attention(qd[0], kd[0], vd[0], table, starts, lens, max_new=max(b.new) if max_new is None else max_new, scale=scale, window=window,
                      softcap=cap, out=out[0])
    got = back(B, out[1])
    want, lim = old.astype(np.float64), np.zeros((b.M, nh, d))
    f = scale or 1.0 / math.sqrt(d)
    cache = {}
    for m, r, pos in b.tokens():
        if check is not None and m not in check:
            want[m] = got[m]
            continue
        if r not in cache:
            cache = {r: (b.gather(k, r).astype(np.float64), b.gather(v, r).astype(np.float64))}
        kk, vv = cache[r]
        lo = max(0, pos - window + 1) if window else 0
        want[m], mass, size = attention(q[m].astype(np.float64), kk[lo:pos + 1], vv[lo:pos + 1], pos - lo, f, 0, cap)
        off = 2 * (d + 6) * F32 * size[:, None] + (pos - lo + 24) * F32
        lim[m] = off * np.abs(vv[lo:pos + 1]).max() + (BF16 * (np.abs(want[m]) + 2 * mass) * (1 + 2.0 ** -7) if store == "bf16" else 0)
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4], np.abs(got - want).max())


HEADS = [(4, 2, 64), (8, 1, 128), (2, 2, 256), (3, 3, 24), (6, 2, 96), (5, 1, 64), (32, 1, 128), (2, 1, 8), (8, 2, 40)]


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("window,cap", [(0, 0.0), (7, 0.0), (0, 3.0), (33, 20.0)])
def test_attention(cuda, store, nh, nkv, d, window, cap):
    for i, (new, total, page) in enumerate(SHAPES):
        check_attention(cuda, Batch(new, total, page, seed=i, spare=i % 3), store, nh, nkv, d, window, cap, spread=2.0, strided=i % 2 == 1,
                        scale=0.0 if i % 3 else 0.3)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (4, 2, 128), (6, 1, 40), (2, 2, 256)])
@pytest.mark.parametrize("offset", [1, 2])
def test_attention_of_unaligned_queries(cuda, store, nh, nkv, d, offset):
    for i, (new, total, page) in enumerate(SHAPES):
        check_attention(cuda, Batch(new, total, page, seed=i, spare=1), store, nh, nkv, d, 9 * (i % 2), spread=2.0, stale=np.nan, offset=offset)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (2, 1, 256), (4, 2, 128)])
@pytest.mark.parametrize("cap,spread", [(1e4, 2.0), (1e30, 2.0), (2e38, 2.0), (0.5, 30.0), (8.0, 30.0), (1e-38, 2.0)])
def test_attention_caps_far_above_and_below_the_scores(cuda, store, nh, nkv, d, cap, spread):
    """A cap far above the scores leaves them their 24 bits; one far below makes them all but equal."""
    for new, total in (([1, 1], [300, 77]), ([150, 3], [400, 300])):
        check_attention(cuda, Batch(new, total, 16), store, nh, nkv, d, 0, cap, spread=spread)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("window", [303, 304, 305, 2 ** 31, 2 ** 63 - 1])
def test_attention_windows_longer_than_all(cuda, store, window):
    for new in ([1, 1], [150, 3]):
        check_attention(cuda, Batch(new, [300, 304], 16), store, 4, 2, 128, window, stale=np.nan)


@gpu
@pytest.mark.parametrize("nh,nkv,d", [(6, 2, 64), (10, 2, 128), (6, 2, 256)])
def test_capped_rows_do_not_depend_on_their_neighbours(cuda, nh, nkv, d):
    """A row's outputs, bit for bit, beside rows of small and of huge scores, or of NaN."""
    import torch
    rng = np.random.default_rng(d)
    R, n, t, page = 300, 8, 40, 16
    b = Batch([n if r % 2 == 0 else 5 for r in range(R)], [t] * R, page)
    mine = np.concatenate([np.arange(b.starts[r], b.starts[r + 1]) for r in range(0, R, 2)])
    q = rounded(rng.standard_normal((b.M, nh, d)) * 2, "bf16")
    k, v = (put(cuda, rounded(rng.standard_normal((b.n_pages, nkv, page, d)), "bf16"), "bf16") for _ in range(2))
    tables = b.up(cuda)
    got = []
    for factor in (1.0, 1000.0, np.nan, 0.0, 1.0):
        x = q * np.float32(factor)
        x[mine] = q[mine]
        out = put(cuda, np.zeros((b.M, nh, d), np.float32), "bf16")
        cuda.paged_attention(put(cuda, x, "bf16")[0], k[0], v[0], *tables, max_new=n, softcap=20.0, out=out[0])
        cuda.sync()
        got.append(out[1].view(torch.int16).cpu().numpy()[mine])
    assert np.abs(got[0]).max() > 0
    assert [int((x != got[0]).sum()) for x in got[1:]] == [0] * 4


# Errors of all outputs together, which show a part of the operands that was left out where the largest possible error of one does not.
#
# f32: operands are two tf32 parts, the upper one rounded (2^-11 at most left), of the lower one 11 bits read (2^-10 of it cut off at most: 2^-21 of the value),
# and the product of the lower parts left out (2^-22).  A product q k is then 2^-21 + 2^-21 + 2^-22 < 3 2^-21 off at most, a score of d such
# products of independent signs by `spread` (its standard deviation here) times as much, an output by that relative to itself, and as much again for p v.
PARTS = 3 * 2.0 ** -21


def relative(got, want):
    return math.sqrt(((got - want) ** 2).sum() / (want ** 2).sum())


def off_from_rounded(got, want):
    """The share of values that are not the 64-bit result rounded to bf16."""
    return float((got != rounded(want, "bf16").astype(np.float64)).mean())


def attention_of(B, b, store, nh, nkv, d, spread, window=0):
    """The kernel's outputs and the 64-bit ones."""
    rng = b.rng
    q = rounded(rng.standard_normal((b.M, nh, d)) * spread, store)
    k, v = (rounded(rng.standard_normal((b.n_pages, nkv, b.page, d)), store) for _ in range(2))
    out = put(B, np.zeros((b.M, nh, d), np.float32), store)
    B.paged_attention(put(B, q, store)[0], put(B, k, store)[0], put(B, v, store)[0], *b.up(B), max_new=max(b.new), window=window, out=out[0])
    got, want = back(B, out[1]), np.zeros((b.M, nh, d))
    rows = [tuple(b.gather(x, r).astype(np.float64) for x in (k, v)) for r in range(len(b.new))]
    for m, r, pos in b.tokens():
        kk, vv = rows[r]
        lo = max(0, pos - window + 1) if window else 0
        want[m] = attention(q[m].astype(np.float64), kk[lo:pos + 1], vv[lo:pos + 1], pos - lo, 1.0 / math.sqrt(d), 0, 0.0)[0]
    return got, want


@gpu
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (4, 2, 128), (2, 1, 256), (6, 2, 96), (3, 3, 24)])
@pytest.mark.parametrize("new,total", [([1, 1, 1], [300, 9001, 77]), ([3, 1], [3000, 40]), ([150, 40], [400, 300]), ([70], [2070])])
def test_attention_f32_has_all_parts_of_its_operands(cuda, nh, nkv, d, new, total):
    assert relative(*attention_of(cuda, Batch(new, total, 16, seed=d), "f32", nh, nkv, d, 2.0)) <= (2.0 + 1.0) * PARTS


@gpu
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (4, 2, 128), (2, 1, 256), (8, 1, 64), (16, 1, 128), (6, 2, 96)])
@pytest.mark.parametrize("new,total,window", [([1, 1, 1], [300, 9001, 77], 0), ([1] * 40, [50 + r for r in range(40)], 33), ([1], [4000], 0)])
def test_attention_of_single_tokens_is_rounded_once(cuda, nh, nkv, d, new, total, window):
    """Probabilities have two bf16 parts: 2^-16 of them is left out at most (and f32 sums of up to 256 products of either sign are as near).  An output is then 2^-16 of its usual size off
    before it is rounded, which leads to the other neighbour where a border of bf16 is as near: 2^-16 / 2^-8 of the values of that size, four times as many
    among smaller ones: 2 %."""
    assert off_from_rounded(*attention_of(cuda, Batch(new, total, 16, seed=d), "bf16", nh, nkv, d, 2.0, window)) <= 0.02


def tf32_parts(x):
    """The upper and the lower part of f32 values, as the tensor cores read them."""
    x = np.asarray(x, np.float32)
    hi = ((x.view(np.uint32) + np.uint32(0x1000)) & np.uint32(0xFFFFE000)).view(np.float32)
    lo = ((x - hi).view(np.uint32) & np.uint32(0xFFFFE000)).view(np.float32)
    return hi.astype(np.float64), lo.astype(np.float64)


@pytest.mark.parametrize("d,t", [(64, 300), (64, 9001), (128, 400), (256, 77), (24, 2070)])
def test_bounds_show_a_part_that_is_left_out(d, t):
    """The bounds above, on the CPU: what has all parts is within them, what lacks one is not."""
    rng = np.random.default_rng(d + t)
    rows = 40
    for store in ("f32", "bf16"):
        q = rounded(rng.standard_normal((rows, d)) * 2.0, store)
        k, v = (rounded(rng.standard_normal((t, d)), store) for _ in range(2))
        exact = [x.astype(np.float64) for x in (q, k, v)]
        s = exact[0] @ exact[1].T / math.sqrt(d)
        p = np.exp(s - s.max(1, keepdims=True))
        want = p @ exact[2] / p.sum(1, keepdims=True)

        def kernel(left_out):
            part = {n: [np.where(f"{n}{i}" in left_out, 0.0, x) for i, x in enumerate(tf32_parts(a))] for n, a in dict(q=q, k=k, v=v).items()}
            mul = lambda a, b: a[0] @ b[0] + a[1] @ b[0] + a[0] @ b[1]
            s = mul(part["q"], [x.T for x in part["k"]]) / math.sqrt(d)
            p = np.exp(s - s.max(1, keepdims=True)).astype(np.float32)
            ps = [np.where(f"p{i}" in left_out, 0.0, x) for i, x in enumerate(tf32_parts(p))]
            return mul(ps, part["v"]) / p.astype(np.float64).sum(1, keepdims=True)

        if store == "f32":
            assert relative(kernel(()), want) <= 3.0 * PARTS
            for name in ("q1", "k1", "p1", "v1"):
                assert relative(kernel((name,)), want) > 3 * 3.0 * PARTS, name
        else:
            hi = rounded(p, "bf16").astype(np.float64)
            two = hi + rounded(p - hi, "bf16").astype(np.float64)
            for probabilities, kept in ((two, True), (hi, False)):
                got = rounded(probabilities @ exact[2] / p.sum(1, keepdims=True), "bf16").astype(np.float64)
                assert (off_from_rounded(got, want) <= 0.02) == kept


# around tiles of 16 to 128 keys and queries, shares of the keys, pages that end inside a tile
EDGES = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300]


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(8, 2, 64), (4, 4, 128), (4, 2, 256), (16, 1, 64)])
@pytest.mark.parametrize("page", [8, 16, 128, 1024])
def test_attention_single_tokens(cuda, store, nh, nkv, d, page):
    """One token each over every length; the number of rows decides how many shares the keys have."""
    for lengths in (EDGES, EDGES[-3:], EDGES[-1:], [1], EDGES * 6):
        check_attention(cuda, Batch([1] * len(lengths), lengths, page), store, nh, nkv, d, spread=2.0, stale=np.nan)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (2, 1, 128), (2, 2, 256), (1, 1, 80)])
@pytest.mark.parametrize("page,window", [(8, 0), (16, 20), (64, 64), (256, 0), (32, 130)])
def test_attention_prompts(cuda, store, nh, nkv, d, page, window):
    """Rows of every length behind nothing and behind cached tokens; what is nobody's is NaN."""
    check_attention(cuda, Batch(EDGES, EDGES, page), store, nh, nkv, d, window, spread=2.0, stale=np.nan)
    check_attention(cuda, Batch(EDGES, [n + c for n, c in zip(EDGES, [90, 3, 64, 0, 1, 200, 31, 128, 5, 7, 61, 62, 63, 64, 65, 1])], page), store, nh, nkv, d,
                    window, spread=2.0, stale=np.nan)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (8, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("columns", [40, 4000])
def test_tables_much_wider_than_the_rows(cuda, store, nh, nkv, d, columns):
    """What a captured step has: columns for rows that grow, naming nothing yet.  The width decides into how many shares the keys are cut."""
    for new, total in (([1, 1, 1], [5, 130, 64]), ([1] * 20, [1 + 7 * r for r in range(20)]), ([40, 3, 90], [60, 100, 90]), ([70], [300])):
        b = Batch(new, total, 16, spare=1)
        b.table = np.concatenate([b.table, np.full((len(new), columns), 0xFFFFFFFF, np.uint32)], 1)
        check_attention(cuda, b, store, nh, nkv, d, 0, spread=2.0, stale=np.nan)
        check_attention(cuda, b, store, nh, nkv, d, 33, 20.0, spread=2.0, stale=np.nan)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_long(cuda, store, d):
    """Long contexts of unequal length, single tokens and a prompt's end; some tokens are checked."""
    check_attention(cuda, Batch([1, 1, 1], [9001, 40, 4096], 64), store, 4, 2, d, spread=3.0)
    check_attention(cuda, Batch([1], [33333], 16), store, 8, 1, d, spread=3.0)
    b = Batch([1500, 300], [2500, 4111], 32)
    check_attention(cuda, b, store, 4, 2, d, spread=3.0, check={0, 127, 128, 700, 1499, 1500, 1799})


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("d,n", [(64, 1), (64, 100), (128, 1), (128, 100), (256, 1), (256, 40)])
def test_attention_skips_pages_before_the_window(cuda, store, d, n):
    """Their table entries are stale: pages that do not exist, or that others filled with NaN."""
    for page in (8, 16, 64):
        b = Batch([n, n, 1], [n + 500, n + 77, 900], page)
        window = 70
        for r, (m, t) in enumerate(zip(b.new, b.total)):
            gone = max(0, t - m - window + 1) // page
            b.table[r, :gone] = 0xFFFFFFFF if r % 2 == 0 else b.n_pages - 1   # (the last page is nobody's, NaN)
        check_stale(cuda, b, store, d, window)


def check_stale(B, b, store, d, window):
    used = set(b.table[b.table < b.n_pages].tolist()) - {b.n_pages - 1}
    # the page that stands for freed ones belongs to no live column
    for r, t in enumerate(b.total):
        live = b.table[r, max(0, t - b.new[r] - window + 1) // b.page:]
        for i, p in enumerate(live):
            if p == b.n_pages - 1:
                live[i] = next(x for x in range(b.n_pages - 1) if x not in used)
                used.add(int(live[i]))
    rng = b.rng
    nh, nkv = 4, 2
    q = rounded(rng.standard_normal((b.M, nh, d)), store)
    k, v = (rounded(rng.standard_normal((b.n_pages, nkv, b.page, d)), store) for _ in range(2))
    k[-1], v[-1] = np.nan, np.nan
    out = put(B, np.zeros((b.M, nh, d), np.float32), store)
    qd, kd, vd = (put(B, x, store)[0] for x in (q, k, v))
    table, starts, lens = b.up(B)
    B.paged_attention(qd, kd, vd, table, starts, lens, max_new=max(b.new), window=window, out=out[0])
    got = back(B, out[1])      # (back() syncs: no error was raised)
    for m, r, pos in b.tokens():
        at = np.arange(max(0, pos - window + 1), pos + 1)
        ids = b.table[r, at // b.page]
        want, mass, size = attention(q[m].astype(np.float64), k[ids, :, at % b.page].astype(np.float64), v[ids, :, at % b.page].astype(np.float64), len(at) - 1,
                                     1.0 / math.sqrt(d), 0, 0.0)
        lim = (2 * (d + 6) * F32 * size.max() + 100 * F32) * 6 + (BF16 * (np.abs(want) + 2 * mass) * (1 + 2.0 ** -7) if store == "bf16" else 0)
        assert (np.abs(got[m] - want) <= lim).all(), (m, r, pos)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 40])
def test_bad_tables_are_reported_and_harm_nobody_else(cuda, store, n):
    """A page that does not exist, a length beyond the table, more new tokens than the length or than max_new."""
    def fresh():
        return Batch([n, n, n], [n + 20, n + 5, n + 33], 16)
    good = run_simple(cuda, fresh(), store)
    cuda.sync()
    spoil = [lambda b: b.table.__setitem__((1, 0), b.n_pages), lambda b: b.table.__setitem__((1, 0), 0xFFFFFFFF),
             lambda b: b.lens.__setitem__(1, b.cols * 16 + 1), lambda b: b.lens.__setitem__(1, n - 1), lambda b: b.lens.__setitem__(1, 0xFFFFFFFF)]
    for i, change in enumerate(spoil):
        b = fresh()
        change(b)
        with pytest.raises(cg.BackendPanic) as e:
            run_simple(cuda, b, store)
        assert e.value.status == 6
        got = run_simple(cuda, b, store, sync=False)
        for part, want in zip(got, good):
            if part.shape[0] == 3 * n:   # per token: the other rows' are right
                assert np.array_equal(part[:n], want[:n]) and np.array_equal(part[2 * n:], want[2 * n:])
                if i >= 2:
                    assert (part[n:2 * n] == 0).all()
    # a row of more tokens than the caller said
    b = fresh()
    with pytest.raises(cg.BackendPanic):
        run_simple(cuda, b, store, max_new=n - 1 if n > 1 else None, bad_starts=n == 1)
    cuda.sync()


def run_simple(B, b, store, sync=True, max_new=None, bad_starts=False, d=64):
    import torch
    rng = np.random.default_rng(5)
    nh, nkv = 4, 2
    q, k, v = (rounded(rng.standard_normal((b.M, h, d)), store) for h in (nh, nkv, nkv))
    kp, vp = (put(B, rounded(rng.standard_normal((b.n_pages, nkv, b.page, d)), store), store) for _ in range(2))
    qo, out = (put(B, np.zeros((b.M, nh, d), np.float32), store) for _ in range(2))
    qd, kd, vd = (put(B, x, store)[0] for x in (q, k, v))
    if bad_starts:
        b.starts[-1] = b.M + 1
    table, starts, lens = b.up(B)
    B.paged_append(kd, vd, kp[0], vp[0], table, starts, lens, q=qd, q_out=qo[0])
    B.paged_attention(qd, kp[0], vp[0], table, starts, lens, max_new=max(b.new) if max_new is None else max_new, out=out[0])
    if sync:
        B.sync()
    torch.cuda.synchronize()
    try:
        B.sync()
    except cg.BackendPanic:
        pass
    return [t.float().cpu().numpy() for t in (qo[1], out[1], kp[1], vp[1])]


@gpu
def test_new_outputs_and_empty_batches(cuda):
    b = Batch([2, 1], [5, 9], 8, spare=2)
    rng = b.rng
    q, k = (put(cuda, rng.standard_normal((b.M, h, 64)), "bf16") for h in (4, 2))
    kp, vp = (put(cuda, np.zeros((b.n_pages, 2, 8, 64)), "bf16") for _ in range(2))
    table, starts, lens = b.up(cuda)
    q_out = cuda.paged_append(k[0], k[0], kp[0], vp[0], table, starts, lens, q=q[0])
    out = cuda.paged_attention(q_out, kp[0], vp[0], table, starts, lens)
    assert out.shape == (b.M, 4, 64) and cuda.storage_of(out) == 2
    got = cuda.to_numpy(out)
    assert np.abs(got[:3]).min(axis=(1, 2)).max() > 0 and (got[3:] == 0).all() and np.array_equal(cuda.to_numpy(q_out)[:3], back(cuda, q[1])[:3])
    assert cuda.paged_append(k[0], k[0], kp[0], vp[0], table, starts, lens) is None
    none = put(cuda, np.zeros((0, 4, 64)), "bf16")[0]
    assert cuda.paged_attention(none, kp[0], vp[0], table, put(cuda, np.zeros(3, np.uint32))[0], lens).shape == (0, 4, 64)
    cuda.sync()


# ---------------------------------------------------------------- beam search


def best(logits, scores, K, finished=None, end=None):
    B, J, V = logits.shape
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64) + 0.0
    total = np.full((B, J, V), -np.inf)
    for b in range(B):
        for j in range(J):
            s, m = float(scores[b, j]), x[b, j].max()
            if not np.isfinite(s):
                continue
            if finished is not None and finished[b, j]:
                total[b, j, end] = s
            elif np.isfinite(m):
                d = x[b, j] - m
                total[b, j] = s + (d - np.log(np.exp(d).sum()))
    flat = total.reshape(B, -1)
    order = np.argsort(-flat, axis=1, kind="stable")[:, :K]
    parent, token = order // V, order % V
    done = (np.take_along_axis(finished, parent, 1) != 0 if finished is not None else False) | (token == (end if end is not None else -1))
    return np.take_along_axis(flat, order, 1), token, parent, np.broadcast_to(done, order.shape)


def check_select(B, logits, scores, K, finished=None, end=None, store="f32", pitch=0):
    import torch
    x = rounded(logits, store)
    if pitch:
        wide = torch.full((*x.shape[:2], x.shape[2] + pitch), 1e9, device="cuda", dtype=torch.bfloat16 if store == "bf16" else torch.float32)
        wide[..., :x.shape[2]] = torch.from_numpy(x).cuda()
        torch.cuda.synchronize()
        ld = B.from_device(wide[..., :x.shape[2]])
    else:
        ld = put(B, x, store)[0]
    scores = np.asarray(scores, np.float32)
    fd = None if finished is None else put(B, finished.astype(np.uint32))[0]
    more = {} if end is None else {"end": end}
    got = B.beam_select(ld, put(B, scores)[0], K, finished=fd, **more)
    s, t, p, f = (B.to_numpy(a) for a in got)
    ws, wt, wp, wf = best(x, scores, K, finished, end)
    assert np.array_equal(t, wt) and np.array_equal(p, wp) and np.array_equal(f, wf.astype(np.uint32)), (t, wt, p, wp)
    # sums of exponentials 2^-20 of their value (f32 of 32 values, 5 levels of a warp; the exponential 2^-22 and its argument's rounding
    # 2^-24 of up to 100), the result one rounding
    fine = np.isfinite(ws)
    assert np.array_equal(fine, np.isfinite(s)) and (np.abs(s[fine] - ws[fine]) <= F32 * np.abs(ws[fine]) + 2.0 ** -17).all()


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("B,J,K,V", [(1, 1, 1, 1), (1, 1, 4, 5), (2, 3, 3, 31), (3, 4, 4, 999), (1, 8, 16, 8191), (2, 2, 2, 8193), (1, 4, 4, 32000), (5, 1, 32, 50257),
                                     (1, 32, 32, 4097), (2, 16, 8, 65537), (1, 2, 32, 256000)])
def test_select(cuda, store, B, J, K, V):
    """Distinct values (in bf16 with ties between tokens, which go to the lower one)."""
    rng = np.random.default_rng(B + J + K + V)
    logits = rng.standard_normal((B, J, V)) * 3
    scores = -10 - 3 * np.abs(rng.standard_normal((B, J)))
    check_select(cuda, logits, scores, K, store=store)
    done = (rng.random((B, J)) < 0.4).astype(np.uint32)
    check_select(cuda, logits, scores, K, done, V // 3, store=store)
    check_select(cuda, logits, scores, K, done * 0, V - 1, store=store, pitch=(V % 5) + 1)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("V", [40, 3000, 20001, 70000])
def test_select_ties_and_masks(cuda, store, V):
    rng = np.random.default_rng(V)
    J, K = 4, 6
    scores = np.float32([[-1.0, -1.0, -3.0, -2.0]])
    level = np.zeros((1, J, V))
    check_select(cuda, level, scores, K, store=store)                           # all alike: the lowest places of the best beam
    check_select(cuda, level, np.float32([[-2.0] * 4]), K, store=store)         # of all beams
    check_select(cuda, level - 0.0 * np.sign(rng.standard_normal(level.shape)), scores, K, store=store)   # 0 and -0
    steps = np.floor(rng.standard_normal((1, J, V)) * 2)                         # few distinct values
    check_select(cuda, steps, scores, K, store=store)
    lowest = float(np.finfo(np.float32).min) if store == "f32" else -3.3895313892515355e38
    for masked in (-np.inf, lowest, np.nan):
        x = rng.standard_normal((1, J, V)) * 3
        x[:, :, rng.random(V) < 0.9] = masked
        check_select(cuda, x, scores, K, store=store)
        x[:, :, :] = masked
        x[:, 1, V - 1] = x[:, 2, 5] = 0.5                                        # one token left, or none
        check_select(cuda, x, scores, K, store=store)
        check_select(cuda, x, np.float32([[-np.inf, -np.inf, -3.0, np.nan]]), K, store=store)
        check_select(cuda, x, scores, K, np.uint32([[0, 1, 0, 1]]), 7, store=store)
    check_select(cuda, level - np.inf, scores, K, store=store)
    x = rng.standard_normal((1, J, V))
    x[0, 1, 3] = np.inf
    check_select(cuda, x, scores, K, store=store)
    check_select(cuda, rng.standard_normal((1, J, V)) * 3, np.float32([[0.0, -np.inf, -np.inf, -np.inf]]), K, store=store)   # the first step
    check_select(cuda, rng.standard_normal((1, J, V)) * 3, np.float32([[-np.inf, np.inf, -5.0, -np.inf]]), K, np.uint32([[1, 1, 0, 0]]), 3, store=store)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("V", [9, 999, 8195, 50257, 128255, 256000])
@pytest.mark.parametrize("pitch", [0, 1, 4, 6])
def test_select_equal_beams_at_any_alignment(cuda, store, V, pitch):
    """Beams with the same logits and scores have the same totals, wherever their rows begin, and masked is masked, by -inf or by NaN: the
    lower beam comes first, token by token."""
    rng = np.random.default_rng(V + pitch)
    row = rng.standard_normal(V) * 3
    x = np.stack([row, row, rng.standard_normal(V) * 3, row, row, row])[None]
    x[:, :, rng.random(V) < 0.05] = -np.inf
    x[0, 3:5][:, np.isinf(x[0, 0])] = np.nan
    K = min(24, V)
    check_select(cuda, x, np.float32([[-7.25, -7.25, -8.0, -7.25, -7.25, -7.25]]), K, store=store, pitch=pitch)
    check_select(cuda, np.repeat(x, 3, 0), np.full((3, 6), -1.0, np.float32), K, store=store, pitch=pitch)


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("V", [40, 1001, 70001])
def test_select_totals_that_64_bits_do_not_tell_apart(cuda, store, V):
    """Scores beside which logits vanish, logits beside which others do: equal totals go to the lower beam, then to the lower token."""
    rng = np.random.default_rng(V)
    x = rng.standard_normal((2, 3, V)) * 3
    x[1, :, rng.random(V) < 0.5] = -np.inf
    x[1, 2, V // 3:] = np.nan
    for K in (1, 8, 32):
        check_select(cuda, x, np.full((2, 3), -1e30, np.float32), K, store=store)
        check_select(cuda, x, np.float32([[-3.0, -1e30, -1e25], [-1e25, -np.inf, 1e30]]), K, store=store)
        check_select(cuda, x, np.float32([[-1e30, -1e30, 2.0]] * 2), K, np.uint32([[0, 0, 1], [1, 0, 0]]), V - 2, store=store, pitch=1)
    tiny = np.where(rng.random((1, 2, V)) < 0.3, rng.integers(-3, 4, (1, 2, V)) * 1e-30, -1.0 - rng.random((1, 2, V)))
    tiny[0, 0, V - 1] = tiny[0, 1, V // 2] = 4.0   # (a few tokens are told apart, the next are not)
    tiny[0, 1, V // 2 + 3] = 3.0
    for K in (1, 4, 31):
        check_select(cuda, tiny, np.float32([[-1.0, -1.0]]), K, store=store)
        check_select(cuda, tiny, np.float32([[-1.0, -2.5]]), K, store=store)
    zeros = np.float32([[-0.0, 0.0, -0.0]] * 2)
    check_select(cuda, x, zeros, 8, np.ones((2, 3), np.uint32), 5, store=store)


@gpu
def test_select_in_place(cuda):
    rng = np.random.default_rng(1)
    x, s, f = rng.standard_normal((3, 4, 1000)) * 3, -np.abs(rng.standard_normal((3, 4))).astype(np.float32), np.uint32(rng.random((3, 4)) < 0.3)
    x32 = rounded(x, "f32")
    ld, sd, fd = put(cuda, x32)[0], put(cuda, s), put(cuda, f)
    t, p = (put(cuda, np.zeros((3, 4), np.uint32)) for _ in range(2))
    cuda.beam_select(ld, sd[0], 4, finished=fd[0], end=9, out=(sd[0], t[0], p[0], fd[0]))
    ws, wt, wp, wf = best(x32, s, 4, f, 9)
    assert np.array_equal(back(cuda, t[1]), wt) and np.array_equal(back(cuda, p[1]), wp) and np.array_equal(back(cuda, fd[1]), wf)
    assert np.abs(back(cuda, sd[1]) - ws).max() < 1e-5


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("K,layers,page,d,length", [(1, 0, 8, 64, 5), (2, 1, 16, 8, 16), (4, 3, 16, 64, 37), (5, 2, 8, 24, 40), (8, 2, 64, 128, 63), (16, 1, 32, 64, 33),
                                                    (32, 2, 8, 64, 21), (3, 0, 32, 256, 1), (4, 1, 16, 64, 0)])
def test_reorder(cuda, store, K, layers, page, d, length):
    import torch
    B, nkv = 3, 2
    rng = np.random.default_rng(K + page)
    cols = length // page + 2
    n_pages = B * K * cols + 2
    own = rng.permutation(n_pages)[:B * K * cols].reshape(B * K, cols).astype(np.uint32)
    table = own.copy()
    for b in range(B):
        table[b * K:(b + 1) * K, :length // page] = own[b * K + rng.integers(0, K, (K, length // page)), np.arange(length // page)]
    shape = (layers,) * (layers > 0) + (n_pages, nkv, page, d)
    k, v = (rounded(rng.standard_normal(shape), store) for _ in range(2))
    parents = np.stack([np.roll(np.arange(K), 1), np.zeros(K, np.int64), rng.integers(0, K, K)]).astype(np.uint32)   # a cycle, one for all, any
    kd, vd, td = put(cuda, k, store), put(cuda, v, store), put(cuda, table)
    pd, ld, od = put(cuda, parents)[0], put(cuda, np.full(B * K, length, np.uint32))[0], put(cuda, own)[0]
    cuda.paged_reorder(pd, ld, od, td[0], kd[0], vd[0])
    full, begun = divmod(length, page)
    want_t, want = own.copy(), [k.copy(), v.copy()]
    for b in range(B):
        for j in range(K):
            parent = b * K + int(parents[b, j])
            want_t[b * K + j, :full] = table[parent, :full]
            for to, x in zip(want, (k, v)):
                to[..., own[b * K + j, full], :, :begun, :] = x[..., own[parent, full], :, :begun, :]
    assert np.array_equal(back(cuda, td[1]).view(np.uint32), want_t)
    assert np.array_equal(back(cuda, kd[1]), want[0]) and np.array_equal(back(cuda, vd[1]), want[1])


@gpu
def test_reorder_leaves_a_bad_group_as_it_was(cuda):
    B, K, cols, page = 3, 4, 3, 8
    rng = np.random.default_rng(3)
    own = rng.permutation(40)[:B * K * cols].reshape(B * K, cols).astype(np.uint32)
    k = rounded(rng.standard_normal((40, 2, page, 16)), "f32")
    parents = np.uint32([[1, 1, 1, 1]] * B)
    for name, change in [("parent", lambda p, l, o: p.__setitem__((1, 2), 4)), ("lens", lambda p, l, o: l.__setitem__(5, 12)),
                         ("long", lambda p, l, o: l.__setitem__(slice(4, 8), 25)), ("page", lambda p, l, o: o.__setitem__((6, 1), 40)),
                         ("same", lambda p, l, o: o.__setitem__((6, 1), o[5, 1]))]:
        p, l, o, t = parents.copy(), np.full(B * K, 13, np.uint32), own.copy(), own.copy()
        change(p, l, o)
        kd, vd, td = put(cuda, k), put(cuda, k), put(cuda, t)
        cuda.paged_reorder(put(cuda, p)[0], put(cuda, l)[0], put(cuda, o)[0], td[0], kd[0], vd[0])
        with pytest.raises(cg.BackendPanic) as e:
            cuda.sync()
        assert e.value.status == 6, name
        got_t, got = back(cuda, td[1]).view(np.uint32), back(cuda, kd[1])
        assert np.array_equal(got_t[4:8], own[4:8]), name
        for b in (0, 2):
            assert (got_t[b * K:(b + 1) * K, 0] == own[b * K + 1, 0]).all() and np.array_equal(got[own[b * K + 3, 1]][:, :5], k[own[b * K + 1, 1]][:, :5])
        mine = own[4:8, 1]
        assert np.array_equal(got[mine], k[mine].astype(np.float64)), name


# ---------------------------------------------------------------- together


def net(rng, hidden, nh, nkv, d, vocab, layers, std=0.35):
    """A small pre-norm attention model with norms per head; weights of about unit gain, so that choices are clear."""
    w = lambda *s: (rng.standard_normal(s) * std / math.sqrt(s[-1] / 8)).astype(np.float32)
    return {"embed": rng.standard_normal((vocab, hidden)).astype(np.float32), "head": w(vocab, hidden) * 4,
            "layers": [{"qkv": w((nh + 2 * nkv) * d, hidden), "o": w(hidden, nh * d), "n": 1 + 0.1 * rng.standard_normal(hidden).astype(np.float32),
                        "qg": 1 + 0.1 * rng.standard_normal(d).astype(np.float32), "kg": 1 + 0.1 * rng.standard_normal(d).astype(np.float32)} for _ in range(layers)]}


def plain_logits(W, tokens, nh, nkv, d, cos, sin, window):
    """The logits behind the last token, in 64 bits, without a cache."""
    x = W["embed"][tokens].astype(np.float64)
    T = len(tokens)
    c, s = cos[:T, None].astype(np.float64), sin[:T, None].astype(np.float64)

    def turn(v):
        a, b = v[..., :d // 2], v[..., d // 2:]
        return np.concatenate([a * c - b * s, b * c + a * s], -1)

    norm = lambda v, g: v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6) * g
    for L in W["layers"]:
        y = norm(x, L["n"]) @ L["qkv"].T.astype(np.float64)
        q, k, v = (y.reshape(T, -1, d)[:, a:b] for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
        q, k = turn(norm(q, L["qg"])), turn(norm(k, L["kg"]))
        o = np.stack([attention(q[t], k, v, t, 1 / math.sqrt(d), window, 0.0)[0] for t in range(T)])
        x = x + o.reshape(T, -1) @ L["o"].T.astype(np.float64)
    return x[-1] @ W["head"].T.astype(np.float64)


@gpu
@pytest.mark.parametrize("page,window", [(8, 0), (16, 9)])
def test_beam_search_over_the_cache(cuda, page, window):
    """Prompts of unequal length, one row each; then a step of the search selects, reorders all layers' caches at once, and
    runs the new tokens, against a search that keeps whole sequences and no cache.  Selections are the same, and scores as close
    as f32 layers are: 2 layers of sums of at most 128 products, 2^-24 each, far below 1e-4 of scores of some 10."""
    import torch
    rng = np.random.default_rng(page)
    hidden, nh, nkv, d, vocab, layers, K, steps = 64, 4, 2, 32, 211, 2, 4, 12
    W = net(rng, hidden, nh, nkv, d, vocab, layers)
    prompts = [rng.integers(0, vocab, n) for n in (11, 24, 3)]
    G, end, T = len(prompts), 7, 64
    cos_t, sin_t = cuda.rope_tables(10000.0, T, d)
    cos, sin = cuda.to_numpy(cos_t), cuda.to_numpy(sin_t)
    up = lambda a: cuda.from_numpy(np.ascontiguousarray(a))
    Wd = {"embed": up(W["embed"]), "head": up(W["head"]), "layers": [{n: up(a) for n, a in L.items()} for L in W["layers"]]}
    cols = T // page
    own = np.arange(G * K * cols, dtype=np.uint32).reshape(G * K, cols)[:, ::-1].copy()
    own_d, table = put(cuda, own)[0], put(cuda, own)[0]
    kc, vc = (torch.zeros(layers, G * K * cols, nkv, page, d, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    pools = [(cuda.from_device(kc[i]), cuda.from_device(vc[i])) for i in range(layers)]
    whole = cuda.from_device(kc), cuda.from_device(vc)

    def forward(tokens, table, new, total):
        """[packed tokens] -> logits of every token; rows with `new` tokens each."""
        starts, lens = put(cuda, np.concatenate([[0], np.cumsum(new)]).astype(np.uint32))[0], put(cuda, np.uint32(total))[0]
        M = len(tokens)
        x = cuda.index(Wd["embed"], 0, cuda.from_numpy(np.uint32(tokens)))
        for L, (kp, vp) in zip(Wd["layers"], pools):
            y = cuda.reshape(cuda.linear(cuda.fused_rmsnorm(x, L["n"], 1e-6), L["qkv"]), (M, nh + 2 * nkv, d))
            q, k, v = cuda.slice(y, 1, 0, nh), cuda.slice(y, 1, nh, nkv), cuda.slice(y, 1, nh + nkv, nkv)
            q = cuda.paged_append(k, v, kp, vp, table, starts, lens, q=q, cos=cos_t, sin=sin_t, q_gain=L["qg"], k_gain=L["kg"], eps=1e-6)
            o = cuda.paged_attention(q, kp, vp, table, starts, lens, max_new=max(new), window=window)
            x = cuda.add(x, cuda.linear(cuda.reshape(o, (M, nh * d)), L["o"]))
        return cuda.linear(x, Wd["head"])

    # prompts: the rows of each group's first beam
    first = [put(cuda, own[g * K:g * K + 1])[0] for g in range(G)]
    logits = [cuda.slice(forward(p, first[g], [len(p)], [len(p)]), 0, len(p) - 1, 1) for g, p in enumerate(prompts)]
    x = cuda.concat(cuda.concat(logits[0], logits[1], 0), logits[2], 0)
    scores, tokens, parents, finished = cuda.beam_select(cuda.reshape(x, (G, 1, vocab)), cuda.zeros((G, 1), 0), K, finished=cuda.zeros((G, 1), 1), end=end)
    rows = [[(0.0, list(p), False)] for p in prompts]
    for step in range(steps):
        # the plain search, and the same step's selection on the device
        for g in range(G):
            logit = np.stack([plain_logits(W, np.array(t), nh, nkv, d, cos, sin, window) for _, t, _ in rows[g]])[None]
            s, t, p, f = best(logit, np.array([[r[0] for r in rows[g]]]), K, np.array([[int(r[2]) for r in rows[g]]]), end)
            assert np.array_equal(cuda.to_numpy(tokens)[g], t[0]) and np.array_equal(cuda.to_numpy(parents)[g], p[0]), (step, g)
            assert np.array_equal(cuda.to_numpy(finished)[g], f[0].astype(np.uint32))
            assert np.abs(cuda.to_numpy(scores)[g] - s[0]).max() < 1e-4
            rows[g] = [(float(cuda.to_numpy(scores)[g, j]), rows[g][p[0, j]][1] + [int(t[0, j])], bool(f[0, j])) for j in range(K)]
        total = np.repeat([len(p) + step for p in prompts], K).astype(np.uint32)
        cuda.paged_reorder(parents, put(cuda, total)[0], own_d, table, *whole)
        logits = forward(cuda.to_numpy(tokens).reshape(-1), table, [1] * (G * K), total + 1)
        scores, tokens, parents, finished = cuda.beam_select(cuda.reshape(logits, (G, K, vocab)), scores, K, finished=finished, end=end)
    cuda.sync()


@gpu
@pytest.mark.parametrize("store", ["f32", "bf16"])
def test_captured_steps_replay_with_new_lengths_and_tables(store):
    """A step of each operator in a graph of its own, captured twice over the same buffers and replayed by turns while lengths, tables and
    inputs change: the operators keep nothing between calls, and take no memory."""
    import torch
    dtype = torch.bfloat16 if store == "bf16" else torch.float32
    S = torch.cuda.Stream()
    B = cg.CudaBackend(0, cg.PREC_F32, stream=S.cuda_stream)
    G, K, nh, nkv, d, page, cols, V = 2, 4, 4, 2, 64, 16, 6, 1000
    R = G * K
    gen = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)
    q, k, v, logits = rnd(R, nh, d), rnd(R, nkv, d), rnd(R, nkv, d), rnd(G, K, V)
    kp, vp = rnd(R * cols, nkv, page, d), rnd(R * cols, nkv, page, d)
    own = torch.randperm(R * cols, generator=gen, device="cuda").int().reshape(R, cols).contiguous()
    table, lens, starts = own.clone(), torch.full((R,), 40, device="cuda", dtype=torch.int32), torch.arange(R + 1, device="cuda").int()
    q_out, out, scores = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(G, K, device="cuda")
    ints = [torch.zeros(G, K, device="cuda", dtype=torch.int32) for _ in range(3)]
    torch.cuda.synchronize()
    h = {n: B.from_device(t) for n, t in dict(q=q, k=k, v=v, logits=logits, kp=kp, vp=vp, own=own, table=table, lens=lens, starts=starts, q_out=q_out, out=out, scores=scores).items()}
    hi = [B.from_device(t) for t in ints]

    def step():
        B.paged_append(h["k"], h["v"], h["kp"], h["vp"], h["table"], h["starts"], h["lens"], q=h["q"], q_out=h["q_out"])
        B.paged_attention(h["q_out"], h["kp"], h["vp"], h["table"], h["starts"], h["lens"], max_new=1, out=h["out"])
        B.beam_select(h["logits"], h["scores"], K, finished=hi[2], end=3, out=(h["scores"], *hi))
        B.paged_reorder(hi[1], h["lens"], h["own"], h["table"], h["kp"], h["vp"])

    everything = (kp, vp, table, q_out, out, scores, *ints)
    with torch.cuda.stream(S):
        step()   # (what is set up on first use)
    S.synchronize()
    reserved = B.bytes_reserved()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=S, capture_error_mode="relaxed"):
            step()
        graphs.append(g)
    for i in range(6):
        with torch.cuda.stream(S):
            q.copy_(rnd(R, nh, d)); k.copy_(rnd(R, nkv, d)); v.copy_(rnd(R, nkv, d)); logits.copy_(rnd(G, K, V) * 3)
            lens.fill_(1 + 19 * i)
            table.copy_(own)   # (lengths begin anew, so rows share no pages)
            before = [t.clone() for t in everything]
            graphs[i % 2].replay()
        S.synchronize()
        replayed = [t.clone() for t in everything]
        for t, b in zip(everything, before):
            t.copy_(b)
        torch.cuda.synchronize()
        step()
        B.sync()
        torch.cuda.synchronize()
        for t, r in zip(everything, replayed):
            assert torch.equal(t, r)
    assert B.bytes_reserved() == reserved
    B.close()


@gpu
@pytest.mark.parametrize("d", [64, 40])
def test_append_starts_that_do_not_ascend(cuda, d):
    """Reported, and no token is placed by a row that it is not of: no page but the rows' own first ones is touched."""
    B, page, cols, M = cuda, 8, 2, 12
    for starts in ([0, 10, 2, 4], [0, 12, 0, 3], [5, 1, 9, 2], [0, 0xFFFFFFFF, 1, 2]):
        k = put(B, np.ones((M, 2, d)))[0]
        kp, vp = (put(B, np.zeros((6, 2, page, d))) for _ in range(2))
        B.paged_append(k, k, kp[0], vp[0], put(B, np.arange(6, dtype=np.uint32).reshape(3, cols))[0], put(B, np.array(starts, np.uint32))[0],
                       put(B, np.array([10, 10, 2], np.uint32))[0])
        with pytest.raises(cg.BackendPanic) as e:
            B.sync()
        assert e.value.status == 6
        got = back(B, kp[1])
        n = [b - a for a, b in zip(starts, starts[1:])]
        for r, (new, length) in enumerate(zip(n, (10, 10, 2))):
            placed = got[r * cols:(r + 1) * cols, 0, :, 0].reshape(-1)
            lo = length - new if 0 < new <= length else length
            assert not placed[:lo].any() and not placed[length:].any()


@gpu
def test_what_the_library_knows_of_a_tensor_ends_when_it_is_written(cuda):
    """A product's rounded copy of its operand and a literal's value are not used behind a write in place, a replayed one either."""
    import torch
    S = torch.cuda.Stream()
    B = cg.CudaBackend(0, cg.PREC_BF16, stream=S.cuda_stream)
    new, nh, nkv, d, page = 16, 2, 2, 64, 16
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k = (torch.randn(new, h, d, generator=gen, device="cuda") for h in (nh, nkv))
    eye = B.from_numpy(np.eye(nh * d, dtype=np.float32))
    kp, vp, q_out = B.zeros((1, nkv, page, d), cg.F32), B.zeros((1, nkv, page, d), cg.F32), B.zeros((new, nh, d), cg.F32)
    ints = [torch.tensor(x, device="cuda", dtype=torch.int32) for x in ([[0]], [0, new], [new])]
    torch.cuda.synchronize()
    hq, hk = B.from_device(q), B.from_device(k)
    table, starts, lens = (B.from_device(x) for x in ints)

    def append():
        B.paged_append(hk, hk, kp, vp, table, starts, lens, q=hq, q_out=q_out)

    def product():
        return B.to_numpy(B.linear(B.reshape(q_out, (new, nh * d)), eye))   # (a bf16 weight: the operand is rounded)

    append()
    assert np.array_equal(product(), rounded(q.cpu().numpy(), "bf16").reshape(new, -1))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=S, capture_error_mode="relaxed"):
        append()
    for _ in range(2):
        with torch.cuda.stream(S):
            q.copy_(torch.randn(new, nh, d, generator=gen, device="cuda"))
            g.replay()
        S.synchronize()
        assert np.array_equal(product(), rounded(q.cpu().numpy(), "bf16").reshape(new, -1))
    B.close()
    B = cuda
    # one beam, one group: a literal is its score, and a view of it is read as another type
    score = B.ndarray_from_vec_f32([7.0], (1, 1))
    view = B.reshape(score, (1,))
    outs = [B.zeros((1, 1), cg.U32) for _ in range(3)]
    B.beam_select(B.from_numpy(np.zeros((1, 1, 1), np.float32)), score, 1, out=(score, *outs))
    assert B.to_numpy(score)[0, 0] == 7.0
    B.beam_select(B.from_numpy(np.array([[[3.0, 3.0, 3.0, 3.0]]], np.float32)), score, 1, out=(score, *outs))
    want = np.float32(7 - math.log(4))
    assert abs(B.to_numpy(score)[0, 0] - want) <= 8 * 2.0 ** -24 * 7
    for t in (view, B.reshape(score, (1,))):
        assert B.to_numpy(B.cast(t, cg.U32))[0] == int(want) == 5


@gpu
def test_recorded_mode_and_two_contexts(cuda):
    """What is recorded runs first (lazy mode); two contexts' calls at the same time, on streams of their own, do not meet."""
    import torch
    L = cg.CudaBackend(0, cg.PREC_F32)
    L.set_option("lazy", 1)
    b = Batch([3, 1], [5, 18], 8)
    q, k = (rounded(b.rng.standard_normal((b.M, h, 64)), "f32") for h in (4, 2))
    results = []
    for B in (cuda, L):
        kp, vp = (put(B, np.zeros((b.n_pages, 2, 8, 64)))[0] for _ in range(2))
        table, starts, lens = b.up(B)
        qd, kd = B.add(B.from_numpy(q), B.from_numpy(q)), B.add(B.from_numpy(k), B.from_numpy(k))
        q2 = B.paged_append(kd, kd, kp, vp, table, starts, lens, q=qd)
        o = B.paged_attention(B.add(q2, q2), kp, vp, table, starts, lens)
        results.append(B.to_numpy(B.add(o, o)))
    assert np.array_equal(*results) and np.abs(results[0]).max() > 0
    L.close()
    two = [cg.CudaBackend(0, cg.PREC_F32) for _ in range(2)]
    x = [rounded(np.random.default_rng(i).standard_normal((4, 4, 70001)) * 3, "f32") for i in range(2)]
    s = np.zeros((4, 4), np.float32)
    held = [(put(B, x[i])[0], put(B, s)[0]) for i, B in enumerate(two)]
    for _ in range(20):
        got = [B.beam_select(l, t, 4) for B, (l, t) in zip(two, held)]
    for i, B in enumerate(two):
        want = best(x[i], s, 4)
        assert np.array_equal(B.to_numpy(got[i][1]), want[1]) and np.array_equal(B.to_numpy(got[i][2]), want[2])
        B.close()


@gpu
def test_recorded_calls_read_the_callers_memory_when_they_are_made():
    """Recorded mode: the caller's memory, and what a replayed graph writes, may change before a recorded call would run."""
    import torch
    S = torch.cuda.Stream()
    L = cg.CudaBackend(0, cg.PREC_F32, stream=S.cuda_stream)
    L.set_option("lazy", 1)
    rng = np.random.default_rng(4)
    a, z = (rounded(rng.random((3, 5, 8)) + 0.5, "f32") for _ in range(2))
    lz = L.from_numpy(z)
    calls = [(lambda h: L.add(h, lz), a + z), (lambda h: L.sub(lz, h), z - a), (lambda h: L.mul(h, h), a * a), (lambda h: L.div(lz, h), z / a),
             (lambda h: L.pow(h, L.from_numpy(np.full_like(a, 2.0))), a * a), (lambda h: L.lt(h, lz), (a < z).astype(np.float32)), (lambda h: L.neg(h), -a),
             (lambda h: L.max(h), a.max(-1, keepdims=True)), (lambda h: L.sum(h), a.sum(-1, keepdims=True)), (lambda h: L.cast(h, cg.U32), a.astype(np.uint32)),
             (lambda h: L.matmul(h, L.transpose(lz, 1, 2)), a @ z.transpose(0, 2, 1)), (lambda h: L.concat(L.neg(lz), h, 1), np.concatenate([-z, a], 1)),
             (lambda h: L.add(L.transpose(L.slice(h, 1, 1, 3), 1, 2), L.transpose(L.slice(lz, 1, 1, 3), 1, 2)), (a + z)[:, 1:4].transpose(0, 2, 1)),
             (lambda h: L.add(L.neg(L.neg(lz)), L.reshape(h, a.shape)), a + z)]
    with torch.cuda.stream(S):
        for i, (call, want) in enumerate(calls):
            x = torch.from_numpy(a).cuda()
            y = call(L.from_device(x))
            x.fill_(0)
            # sums of 8 products or values, each side in any order: 16 half steps of 8 values below 2.25 at most
            assert np.abs(L.to_numpy(y).astype(np.float64) - want).max() <= (16 * F32 * 8 * 2.25 if want.dtype == np.float32 else 0), i
        y = L.add(L.from_device(torch.from_numpy(a).cuda().float()), lz)        # (nobody else holds that memory)
        others = [torch.full((3, 5, 8), 9.0, device="cuda") for _ in range(8)]
        assert np.array_equal(L.to_numpy(y), a + z)
        del others
        # the library's own tensor, written by a replay
        new, nh, nkv, d, page = 4, 2, 1, 64, 8
        q, k = (torch.randn(new, h, d, device="cuda") for h in (nh, nkv))
        ints = [torch.tensor(x, device="cuda", dtype=torch.int32) for x in ([[0]], [0, new], [new])]
        hq, hk, *tables = (L.from_device(t) for t in (q, k, *ints))
        kp, vp, q_out = L.zeros((1, nkv, page, d), cg.F32), L.zeros((1, nkv, page, d), cg.F32), L.zeros((new, nh, d), cg.F32)
        append = lambda: L.paged_append(hk, hk, kp, vp, *tables, q=hq, q_out=q_out)
        append()
        L.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=S, capture_error_mode="relaxed"):
        append()
    with torch.cuda.stream(S):
        want = 2 * q.cpu().numpy()
        y = L.add(q_out, q_out)
        q.fill_(0)
        g.replay()
        assert np.array_equal(L.to_numpy(y), want)
    assert L.lazy_stats()[0] > 0
    S.synchronize()
    L.close()


@gpu
def test_tensors_over_device_memory(cuda):
    import torch
    t = torch.arange(24, device="cuda", dtype=torch.float32).reshape(2, 3, 4)
    torch.cuda.synchronize()
    assert np.array_equal(cuda.to_numpy(cuda.from_device(t)), t.cpu().numpy())
    view = t.transpose(0, 2)[:, 1:]
    assert np.array_equal(cuda.to_numpy(cuda.add(cuda.from_device(view), cuda.from_device(view))), 2 * view.cpu().numpy())
    b = cuda.from_device(t.bfloat16())
    del t
    assert cuda.storage_of(b) == 2 and np.array_equal(cuda.to_numpy(cuda.to_f32(b)).ravel(), np.arange(24))
    with pytest.raises(TypeError):
        cuda.from_device(torch.zeros(3, device="cuda", dtype=torch.float16))
    with pytest.raises(TypeError):
        cuda.from_device(torch.zeros(3))
    with pytest.raises(cg.BackendPanic) as e:
        cuda._ext1("cg_tensor_from_device", np.zeros(4, np.float32).ctypes.data, 0, (ctypes.c_int64 * 1)(4), None, 1)
    assert e.value.status == 3


# ---------------------------------------------------------------- refusals and index arithmetic, without a device


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """The library's entry points with a context and tensors that no device stands behind: what is refused is refused before anything
    is launched."""
    cg.load_library()
    out = str(tmp_path_factory.mktemp("paged") / "paged_host.so")
    csrc = os.path.join(ROOT, "catgrad-rs_b200", "csrc")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-I", csrc, "-I", f"{cuda}/include", os.path.join(ROOT, "tests", "paged_host.cpp"), "-o", out,
                           cg.library_path(), f"-Wl,-rpath,{os.path.dirname(cg.library_path())}", "-L", f"{cuda}/lib64", "-lcudart"])
    L = ctypes.CDLL(out)
    vp, i64p = ctypes.c_void_p, ctypes.POINTER(ctypes.c_int64)
    L.host_ctx.restype = vp
    L.host_tensor.restype, L.host_tensor.argtypes = vp, [vp, ctypes.c_uint64, ctypes.c_int, ctypes.c_int, i64p, i64p]
    L.host_device.argtypes = [vp, ctypes.c_int]
    L.host_row_span.argtypes = [vp, vp, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, vp, vp]
    L.host_page_of.argtypes = [vp, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int64, ctypes.c_int64, vp]
    L.host_page_of.restype = ctypes.c_int64
    return L


class Host:
    """Calls with named arguments that can be changed one at a time."""

    def __init__(self, L):
        self.L, self.ctx, self.next = L, ctypes.c_void_p(L.host_ctx()), 1 << 40
        self.lib = ctypes.CDLL(cg.library_path())   # (functions of its own: their argument types are set here)
        self.lib.cg_last_error.restype = ctypes.c_char_p
        self.lib.cg_last_error.argtypes = [ctypes.c_void_p]

    def t(self, *dims, store="f32", strides=None, at=None, shift=0):
        n = len(dims)
        if strides is None:
            strides = [int(np.prod(dims[i + 1:], dtype=np.int64)) for i in range(n)]
        if at is None:
            at, self.next = self.next, self.next + (1 << 32)
        a = lambda v: (ctypes.c_int64 * max(1, n))(*v)
        return ctypes.c_void_p(self.L.host_tensor(self.ctx, at + shift, {"f32": 0, "u32": 1, "bf16": 2}[store], n, a(dims), a(strides)))

    def _call(self, fn, wrap):
        fn.argtypes = [ctypes.c_void_p] + [type(w) if w is not None else ctypes.c_void_p for w in wrap]
        fn.restype = ctypes.c_int32
        return fn(self.ctx, *wrap)


VIEWS = [lambda B, t: B.reshape(t, (4, 6)), lambda B, t: B.transpose(t, 0, 1), lambda B, t: B.slice(t, 2, 1, 2), lambda B, t: B.broadcast(t, (5, 2, 3, 4)),
         lambda B, t: B.cast(t, cg.F32)]


@gpu
def test_views_keep_the_callers_memory(cuda):
    import torch
    for i, view in enumerate(VIEWS):
        x = torch.arange(24, device="cuda").reshape(2, 3, 4).to(torch.bfloat16)
        want = cuda.to_numpy(view(cuda, cuda.from_numpy(np.arange(24, dtype=np.float32).reshape(2, 3, 4))))
        torch.cuda.synchronize()
        alive = weakref.ref(x)
        t = view(cuda, cuda.from_device(x))
        del x
        gc.collect()
        assert alive() is not None, i
        t = cuda.transpose(t, 0, 1)
        assert alive() is not None and np.array_equal(cuda.to_numpy(t), want.swapaxes(0, 1))
        del t
        gc.collect()
        assert alive() is None, i


def test_views_know_who_owns_their_memory(oracle):
    """The same on the CPU: a view of a view too, and no new tensor."""
    class Owner:
        pass
    for view in VIEWS:
        t = oracle.from_numpy(np.arange(24, dtype=np.float32).reshape(2, 3, 4))
        assert view(oracle, t)._memory is None
        t._memory = Owner()
        assert view(oracle, t)._memory is t._memory and oracle.transpose(view(oracle, t), 0, 1)._memory is t._memory
        assert oracle.add(t, t)._memory is None


def test_recorded_mode_records_no_call_on_the_callers_memory(host):
    """Without a device: a call over memory that the library does not own is made at once (here it finds no device to be made on)."""
    H = Host(host)
    L, c = H.lib, ctypes.c_void_p(H.ctx.value)
    for f in (L.cg_set_option, L.cg_lazy_stats, L.cg_add, L.cg_neg, L.cg_max, L.cg_sum, L.cg_cast, L.cg_matmul, L.cg_concat, L.cg_arange, L.cg_reshape):
        f.argtypes = None
        f.restype = ctypes.c_int32
    assert L.cg_set_option(c, b"lazy", ctypes.c_int64(1)) == 0

    def recorded():
        n = [ctypes.c_int64() for _ in range(3)]
        assert L.cg_lazy_stats(c, *(ctypes.byref(x) for x in n)) == 0
        return n[0].value

    out = ctypes.c_void_p()
    x, y, u = H.t(0, 4), H.t(4, 0), H.t(0, 4, store="u32")     # (no elements: nothing to launch wherever this runs)
    L.cg_add(c, x, x, ctypes.byref(out))
    L.cg_add(c, u, u, ctypes.byref(out))
    L.cg_neg(c, x, ctypes.byref(out))
    L.cg_max(c, x, ctypes.byref(out))
    L.cg_sum(c, x, ctypes.byref(out))
    L.cg_cast(c, x, 1, ctypes.byref(out))
    L.cg_matmul(c, x, y, ctypes.byref(out))
    assert recorded() == 0
    end = ctypes.c_void_p()
    assert L.cg_arange(c, ctypes.c_int64(0), ctypes.byref(end)) == 0 and recorded() == 1   # (what has no such input is)
    assert L.cg_cast(c, end, 0, ctypes.byref(out)) == 0 and recorded() == 2
    assert L.cg_set_option(c, b"lazy", ctypes.c_int64(1)) == 0
    L.cg_concat(c, out, H.t(0), 0, ctypes.byref(out))
    assert recorded() == 2


def test_append_refusals(host):
    """Every call here is refused (a call that were not would return CG_ERR_CUDA: there is no device)."""
    H = Host(host)
    u, t = (lambda *d: H.t(*d, store="u32")), H.t

    def call(**kw):
        a = dict(q=t(6, 4, 64), k=t(6, 2, 64), v=t(6, 2, 64), q_gain=t(64), k_gain=t(64), eps=1e-6, plus=0, cos=t(50, 32), sin=t(50, 32), half=1, table=u(3, 5),
                 starts=u(4), lens=u(3), k_pages=t(20, 2, 16, 64, store="bf16"), v_pages=t(20, 2, 16, 64, store="bf16"), q_out=t(6, 4, 64, store="bf16"))
        a.update(kw)
        order = ("q", "k", "v", "q_gain", "k_gain", "eps", "plus", "cos", "sin", "half", "table", "starts", "lens", "k_pages", "v_pages", "q_out")
        wrap = [ctypes.c_int32(a[n]) if n in ("plus", "half") else ctypes.c_float(a[n]) if n == "eps" else a[n] for n in order]
        return H._call(H.lib.cg_paged_append, wrap)

    SHAPE, DTYPE, INVALID, UNSUPPORTED = 1, 2, 3, 8
    for name in ("k", "v", "table", "starts", "lens", "k_pages", "v_pages", "q", "q_out", "cos", "sin"):
        assert call(**{name: None}) == INVALID, name
    cases = [(SHAPE, dict(k=t(6, 3, 64))), (SHAPE, dict(v=t(5, 2, 64))), (SHAPE, dict(q=t(7, 4, 64))), (SHAPE, dict(q=t(6, 4, 32))), (SHAPE, dict(k=t(6, 128))),
             (SHAPE, dict(q_out=t(6, 5, 64, store="bf16"))), (SHAPE, dict(k_gain=t(32))), (SHAPE, dict(cos=t(50, 40), sin=t(50, 40))), (SHAPE, dict(sin=t(49, 32))),
             (SHAPE, dict(starts=u(3))), (SHAPE, dict(lens=u(4))), (SHAPE, dict(v_pages=t(20, 2, 16, 32, store="bf16"))), (SHAPE, dict(table=u(15))),
             (DTYPE, dict(k=t(6, 2, 64, store="bf16"))), (DTYPE, dict(q_out=t(6, 4, 64))), (DTYPE, dict(v_pages=t(20, 2, 16, 64))), (DTYPE, dict(table=t(3, 5))),
             (DTYPE, dict(lens=t(3))), (DTYPE, dict(cos=t(50, 32, store="bf16"))), (DTYPE, dict(q_gain=t(64, store="bf16"))), (DTYPE, dict(k=u(6, 2, 64))),
             (UNSUPPORTED, dict(k=t(6, 2, 64, strides=[256, 128, 2]))), (UNSUPPORTED, dict(q_out=t(6, 4, 64, store="bf16", strides=[512, 64, 1]))),
             (UNSUPPORTED, dict(k_pages=t(20, 2, 16, 64, store="bf16", strides=[4096, 2048, 128, 1]))), (UNSUPPORTED, dict(table=H.t(3, 5, store="u32", strides=[6, 1]))),
             (UNSUPPORTED, dict(k_pages=t(20, 2, 16, 64, store="bf16", shift=2)))]
    for page, d in ((12, 64), (4, 64), (2048, 64), (16, 12), (16, 264), (16, 4)):
        cases.append((UNSUPPORTED, dict(k=t(6, 2, d), v=t(6, 2, d), q=t(6, 4, d), k_pages=t(20, 2, page, d, store="bf16"), v_pages=t(20, 2, page, d, store="bf16"))))
    at = 7 << 44
    cases += [(INVALID, dict(k_pages=t(20, 2, 16, 64, store="bf16", at=at), v_pages=t(20, 2, 16, 64, store="bf16", at=at))),
              (INVALID, dict(k=t(6, 2, 64, at=at), k_pages=t(20, 2, 16, 64, store="bf16", at=at))),
              (INVALID, dict(q_out=t(6, 4, 64, store="bf16", at=at), v_pages=t(20, 2, 16, 64, store="bf16", at=at, shift=64))),
              (INVALID, dict(lens=H.t(3, store="u32", at=at), q_out=t(6, 4, 64, store="bf16", at=at)))]
    for i, (want, kw) in enumerate(cases):
        assert call(**kw) == want, (i, want, H.lib.cg_last_error(H.ctx))
    far = t(6, 2, 64)
    host.host_device(far, 1)
    assert call(v=far) == INVALID and b"another device" in H.lib.cg_last_error(H.ctx)


def test_append_without_heads_returns(host):
    """Pages without heads and no queries, or queries without heads: there is nothing to write, and the call says so at once."""
    H = Host(host)
    u, t = (lambda *d: H.t(*d, store="u32")), H.t
    for d in (64, 128, 40):
        for q in (None, t(6, 0, d)):
            wrap = [q, t(6, 0, d), t(6, 0, d), None, None, ctypes.c_float(1e-6), ctypes.c_int32(0), None, None, ctypes.c_int32(1), u(3, 5), u(4), u(3),
                    t(20, 0, 16, d, store="bf16"), t(20, 0, 16, d, store="bf16"), None if q is None else t(6, 0, d, store="bf16")]
            got = []
            call = threading.Thread(target=lambda: got.append(H._call(H.lib.cg_paged_append, wrap)), daemon=True)
            call.start()
            call.join(20)
            assert got == [0], (d, q is None)


def test_attention_refusals(host):
    H = Host(host)
    u, t = (lambda *d: H.t(*d, store="u32")), (lambda *d, **k: H.t(*d, **{"store": "bf16", **k}))

    def call(**kw):
        a = dict(q=t(6, 4, 64), k_pages=t(20, 2, 16, 64), v_pages=t(20, 2, 16, 64), table=u(3, 5), starts=u(4), lens=u(3), most=6, scale=0.0, window=0, cap=0.0, out=t(6, 4, 64))
        a.update(kw)
        order = ("q", "k_pages", "v_pages", "table", "starts", "lens", "most", "scale", "window", "cap", "out")
        wrap = [ctypes.c_int64(a[n]) if n in ("most", "window") else ctypes.c_float(a[n]) if n in ("scale", "cap") else a[n] for n in order]
        return H._call(H.lib.cg_paged_attention, wrap)

    SHAPE, DTYPE, INVALID, UNSUPPORTED = 1, 2, 3, 8
    for name in ("q", "k_pages", "v_pages", "table", "starts", "lens", "out"):
        assert call(**{name: None}) == INVALID, name
    at = 7 << 44
    for i, (want, kw) in enumerate([(SHAPE, dict(q=t(6, 5, 64), out=t(6, 5, 64))), (SHAPE, dict(q=t(6, 4, 32), out=t(6, 4, 32))), (SHAPE, dict(out=t(6, 4, 32))), (SHAPE, dict(q=t(24, 64))),
                                    (SHAPE, dict(starts=u(5))), (DTYPE, dict(q=t(6, 4, 64, store="f32"))), (DTYPE, dict(out=t(6, 4, 64, store="f32"))), (DTYPE, dict(starts=t(4))),
                                    (INVALID, dict(most=-1)), (INVALID, dict(window=-1)), (INVALID, dict(cap=-1.0)), (INVALID, dict(cap=float("nan"))), (INVALID, dict(scale=float("inf"))),
                                    (INVALID, dict(scale=-0.5)), (UNSUPPORTED, dict(q=t(6, 4, 64, strides=[512, 128, 2]))), (UNSUPPORTED, dict(out=t(6, 4, 64, strides=[512, 64, 1]))),
                                    (UNSUPPORTED, dict(k_pages=t(20, 2, 24, 64), v_pages=t(20, 2, 24, 64))), (SHAPE, dict(k_pages=t(0, 2, 16, 64), v_pages=t(0, 2, 16, 64))), (INVALID, dict(q=t(6, 4, 64, at=at), out=t(6, 4, 64, at=at))),
                                    (INVALID, dict(k_pages=t(20, 2, 16, 64, at=at), out=t(6, 4, 64, at=at, shift=1024)))]):
        assert call(**kw) == want, (i, want, H.lib.cg_last_error(H.ctx))


def test_select_and_reorder_refusals(host):
    H = Host(host)
    u, t = (lambda *d, **k: H.t(*d, store="u32", **k)), H.t
    SHAPE, DTYPE, INVALID, UNSUPPORTED = 1, 2, 3, 8

    def select(**kw):
        a = dict(logits=t(2, 4, 100), scores=t(2, 4), finished=u(2, 4), end=7, so=t(2, 3), to=u(2, 3), po=u(2, 3), fo=u(2, 3))
        a.update(kw)
        return H._call(H.lib.cg_beam_select, [a["logits"], a["scores"], a["finished"], ctypes.c_uint32(a["end"]), a["so"], a["to"], a["po"], a["fo"]])

    for name in ("logits", "scores", "so", "to", "po", "fo"):
        assert select(**{name: None}) == INVALID, name
    at = 7 << 44
    wide = lambda k: dict(so=t(2, k), to=u(2, k), po=u(2, k), fo=u(2, k))
    for i, (want, kw) in enumerate([(SHAPE, dict(scores=t(2, 5))), (SHAPE, dict(logits=t(8, 100))), (SHAPE, dict(so=t(3, 3))), (SHAPE, dict(po=u(2, 4))), (SHAPE, dict(finished=u(8))),
                                    (SHAPE, dict(logits=t(2, 4, 2), end=1)), (DTYPE, dict(logits=u(2, 4, 100))), (DTYPE, dict(scores=t(2, 4, store="bf16"))), (DTYPE, dict(so=t(2, 3, store="bf16"))),
                                    (DTYPE, dict(to=t(2, 3))), (INVALID, dict(end=100)), (UNSUPPORTED, dict(logits=t(2, 4, 100, strides=[800, 200, 2]))), (UNSUPPORTED, wide(33)),
                                    (UNSUPPORTED, dict(logits=t(2, 33, 100), scores=t(2, 33), finished=u(2, 33))), (UNSUPPORTED, dict(to=u(2, 3, strides=[4, 1]))),
                                    (SHAPE, dict(logits=t(2, 0, 100), scores=t(2, 0), finished=u(2, 0))), (UNSUPPORTED, dict(logits=t(1, 32, 1 << 24), scores=t(1, 32), finished=None, **{k: v for k, v in dict(so=t(1, 32), to=u(1, 32), po=u(1, 32), fo=u(1, 32)).items()})),
                                    (INVALID, dict(scores=t(2, 4, at=at), so=t(2, 3, at=at))), (INVALID, dict(to=u(2, 3, at=at), po=u(2, 3, at=at))),
                                    (INVALID, dict(logits=t(2, 4, 100, at=at), fo=u(2, 3, at=at))), (INVALID, dict(scores=t(2, 4, at=at), **{**wide(4), "so": t(2, 4, at=at, shift=4)}))]):
        assert select(**kw) == want, (i, want, H.lib.cg_last_error(H.ctx))

    def reorder(**kw):
        a = dict(parents=u(2, 4), lens=u(8), own=u(8, 5), table=u(8, 5), k=t(3, 20, 2, 16, 64), v=t(3, 20, 2, 16, 64))
        a.update(kw)
        return H._call(H.lib.cg_paged_reorder, [a[n] for n in ("parents", "lens", "own", "table", "k", "v")])

    for name in ("parents", "lens", "own", "table", "k", "v"):
        assert reorder(**{name: None}) == INVALID, name
    for i, (want, kw) in enumerate([(SHAPE, dict(parents=u(8))), (SHAPE, dict(lens=u(7))), (SHAPE, dict(own=u(8, 6))), (SHAPE, dict(table=u(7, 5))), (SHAPE, dict(k=t(20, 2, 16, 64))),
                                    (SHAPE, dict(k=t(3, 20, 64), v=t(3, 20, 64))), (DTYPE, dict(parents=t(2, 4))), (DTYPE, dict(v=t(3, 20, 2, 16, 64, store="bf16"))),
                                    (UNSUPPORTED, dict(parents=u(1, 33), lens=u(33), own=u(33, 5), table=u(33, 5))), (UNSUPPORTED, dict(table=u(8, 5, strides=[6, 1]))),
                                    (INVALID, dict(own=u(8, 5, at=at), table=u(8, 5, at=at))), (INVALID, dict(lens=u(8, at=at), k=t(3, 20, 2, 16, 64, at=at))),
                                    (INVALID, dict(table=u(8, 5, at=at), v=t(3, 20, 2, 16, 64, at=at)))]):
        assert reorder(**kw) == want, (i, want, H.lib.cg_last_error(H.ctx))


def test_tensors_that_another_context_has_recorded_are_refused(host):
    """They have no memory yet.  (In a process of its own, since a call that looked for that memory would end it.)"""
    out = ctypes.CDLL(host._name)._name
    r = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {os.path.dirname(__file__)!r}); import test_paged; test_paged.recorded_elsewhere({out!r})"],
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

    def waiting(shape, dtype):
        t = ctypes.c_void_p()
        assert lib.cg_arange(other, ctypes.c_int64(int(np.prod(shape))), ctypes.byref(t)) == 0
        if dtype == 0:
            assert lib.cg_cast(other, t, 0, ctypes.byref(t)) == 0
        assert lib.cg_reshape(other, t, (ctypes.c_int64 * len(shape))(*shape), len(shape), ctypes.byref(t)) == 0
        return t

    u, f, i32, i64 = (lambda *d: H.t(*d, store="u32")), H.t, ctypes.c_int32, ctypes.c_int64
    calls = [(lib.cg_paged_attention, dict(q=f(6, 4, 64), k=f(20, 2, 16, 64), v=f(20, 2, 16, 64), table=u(3, 5), starts=u(4), lens=u(3)),
              [i64(6), ctypes.c_float(0), i64(0), ctypes.c_float(0)], dict(out=f(6, 4, 64))),
             (lib.cg_beam_select, dict(logits=f(2, 4, 100), scores=f(2, 4), finished=u(2, 4)), [ctypes.c_uint32(7)], dict(s=f(2, 3), t=u(2, 3), p=u(2, 3), f=u(2, 3))),
             (lib.cg_paged_reorder, dict(parents=u(2, 4), lens=u(8), own=u(8, 5), table=u(8, 5), k=f(20, 2, 16, 64), v=f(20, 2, 16, 64)), [], {})]
    shapes = dict(q=((6, 4, 64), 0), k=((20, 2, 16, 64), 0), v=((20, 2, 16, 64), 0), table=((3, 5), 1), starts=((4,), 1), lens=((3,), 1), out=((6, 4, 64), 0),
                  logits=((2, 4, 100), 0), scores=((2, 4), 0), finished=((2, 4), 1), s=((2, 3), 0), t=((2, 3), 1), p=((2, 3), 1), f=((2, 3), 1))
    for i, (fn, a, scalars, b) in enumerate(calls):
        for name in {**a, **b}:
            shape, dtype = dict(shapes, lens=((8,), 1), table=((8, 5), 1), own=((8, 5), 1), parents=((2, 4), 1))[name] if i == 2 else shapes[name]
            w = waiting(shape, dtype)
            assert H._call(fn, [w if n == name else x for n, x in a.items()] + scalars + [w if n == name else x for n, x in b.items()]) == 3, (i, name)
            assert b"another context" in lib.cg_last_error(H.ctx)


def test_rows_that_cannot_be_are_not_followed(host):
    """row_span and page_of, on the CPU: everything they let through lies inside the tensors."""
    rng = np.random.default_rng(0)
    vp = lambda a: a.ctypes.data_as(ctypes.c_void_p)
    some = 0
    for _ in range(4000):
        rows, cols, lg, M = int(rng.integers(1, 6)), int(rng.integers(1, 5)), 4, int(rng.integers(0, 40))
        starts = np.sort(rng.integers(0, 40, rows + 1)).astype(np.uint32)
        if rng.random() < 0.3:
            starts[rng.integers(0, rows + 1)] = rng.choice([0, 5, 41, 0xFFFFFFFF, 0x80000000])
        lens = rng.choice([0, 1, 7, 16, 30, cols * 16, cols * 16 + 1, 0xFFFFFFFF, 0x7FFFFFFF], rows).astype(np.uint32)
        most = int(rng.choice([1, 5, 40]))
        for r in range(rows):
            out, err = np.zeros(3, np.int64), np.zeros(1, np.int32)
            ok = host.host_row_span(vp(starts), vp(lens), rows, cols, lg, M, r, most, vp(out), vp(err))
            a, b, n = int(starts[r]), int(starts[r + 1]), int(lens[r])
            good = a < b <= M and b - a <= min(most, n) and n <= cols * 16
            assert bool(ok) == good and err[0] == (0 if good or a == b else 1)
            if ok:
                some += 1
                assert 0 <= out[0] and out[0] + out[1] <= M and 0 <= out[2] - out[1] and out[2] <= cols << lg
    assert some > 300
    table, err = np.uint32([3, 9, 10, 0xFFFFFFFF, 0, 1, 2, 4]), np.zeros(1, np.int32)
    got = [host.host_page_of(vp(table), 4, 10, 4, r, p, vp(err)) for r in (0, 1) for p in (0, 15, 16, 31, 63, 47)]
    assert got == [3, 3, 9, 9, -1, -1, 0, 0, 1, 1, 4, 2] and err[0] == 1


def test_prompt_attention_takes_tmem_between_its_dependency_and_its_trigger():
    """After the wait no earlier kernel holds columns, and before the trigger no later one runs that could hold what this one waits for.
    Blocks without tokens leave before they take any."""
    text = open(os.path.join(os.path.dirname(cg.__file__), "csrc", "paged_fa.cu")).read()
    body = text[text.index("k_paged_fa(const __grid_constant__"):]
    body = body[:body.index("\n}\n")]
    order = ["griddepcontrol.wait;", "if (i0 >= n) return;", "tcgen05.alloc.", "griddepcontrol.launch_dependents;", "tcgen05.dealloc."]
    assert all(body.count(x) == 1 for x in order)
    assert [body.index(x) for x in order] == sorted(body.index(x) for x in order)
