"""Serving several sequences from a paged key/value cache, and beam search over it, as operators to be timed.

Four operators, each a call of the library's (`cg.CudaBackend`):

* `paged_append`: the new tokens' queries and keys get their norm per head (where the model has one) and their
  rotation, and keys and values go to the pages that the table names;
* `paged_attention`: causal attention of the new tokens, whole prompts or single ones, over the cached pages;
* `beam_select`: the best continuations of a search over beams and vocabulary;
* `paged_reorder`: every beam goes on from its parent: full pages are shared, the begun page is copied.

Cached tensors are [pages, key heads, tokens of a page, head size]; row r of a batch has the packed tokens
starts[r] .. starts[r + 1], its first lens[r] cached tokens count (the new ones among them), and its token at
position p lies in page table[r, p // page] at place p % page.

The sizes are those of the models the repository is benchmarked and tested on: heads and vocabularies of the
Llama-3.2-1B, Llama-3-8B, Qwen3-30B-A3B and Gemma-2-2B shapes, and of the small f32 Llama.
"""
from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
# query heads, key heads, head size, norms per head, soft-cap, window, base of the rotation, vocabulary
MODELS = {
    "llama1b": (32, 8, 64, False, 0.0, 0, 500000.0, 128256),
    "llama8b": (32, 8, 128, False, 0.0, 0, 500000.0, 128256),
    "qwen3moe": (32, 4, 128, True, 0.0, 0, 1e6, 151936),
    "gemma2": (8, 4, 256, False, 50.0, 4096, 10000.0, 256000),
    "tiny": (4, 2, 64, False, 0.0, 0, 10000.0, 32000),
}


def listed():
    def append(name, model, rows, new, cached, page, inputs, pages="bf16", ragged=False):
        return {"name": name, "op": "append", "model": model, "rows": rows, "new": new, "cached": cached, "page": page,
                "inputs": inputs, "pages": pages, "ragged": ragged}

    def attend(name, model, rows, new, cached, page, pages="bf16", ragged=False):
        return {"name": name, "op": "attend", "model": model, "rows": rows, "new": new, "cached": cached, "page": page,
                "pages": pages, "ragged": ragged}

    def select(name, batch, beams, keep, vocab, logits, finished):
        return {"name": name, "op": "select", "batch": batch, "beams": beams, "keep": keep, "vocab": vocab, "logits": logits,
                "finished": finished}

    def reorder(name, model, batch, beams, layers, prompt, made, page, pages="bf16"):
        return {"name": name, "op": "reorder", "model": model, "batch": batch, "beams": beams, "layers": layers, "prompt": prompt,
                "made": made, "page": page, "pages": pages}

    return [
        # a layer of one decode step of the benchmark's batch: launches and latency are all there is
        append("append-step", "llama1b", 8, 1, 577, 16, "f32"),
        # a layer of a prompt batch as requests come in, with norms per head
        append("append-prompts", "qwen3moe", 6, 2903, 0, 64, "bf16", ragged=True),
        # the f32 model, rows that go on behind what is cached
        append("append-f32", "tiny", 5, 801, 333, 32, "f32", "f32", True),
        # attention of one decode step of the benchmark's batch
        attend("attend-step", "llama1b", 8, 1, 577, 16),
        # a decode step of a few long contexts of unequal length
        attend("attend-long", "llama8b", 7, 1, 32001, 64, ragged=True),
        # one document
        attend("attend-prompt", "llama8b", 1, 8191, 0, 64),
        # wide heads, capped scores and a window, rows that go on behind what is cached
        attend("attend-chunks", "gemma2", 6, 700, 5003, 32, ragged=True),
        # the f32 model, the same
        attend("attend-f32", "tiny", 3, 213, 1500, 16, "f32", True),
        # one user's beams
        select("select-turn", 1, 4, 4, 128256, "f32", False),
        # many users' beams over the largest vocabulary, some of them finished
        select("select-batch", 24, 8, 8, 256000, "bf16", True),
        # the cache of all layers behind a step of one user's beams
        reorder("reorder-turn", "llama1b", 1, 4, 16, 601, 11, 16),
        # the same for many users, some layers of a wide model
        reorder("reorder-batch", "llama8b", 12, 8, 8, 407, 57, 32),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("append", "attend", "attend", "select", "reorder"))
    model = rng.choice(list(MODELS))
    pages = "f32" if model == "tiny" else "bf16"
    page = rng.choice((16, 32, 64, 128))
    if op == "append":
        rows = spread(1, 64)
        return {"op": op, "model": model, "rows": rows, "new": 1 if rng.random() < 0.4 else spread(2, 8000 // rows), "cached": spread(1, 4000),
                "page": page, "inputs": "f32" if pages == "f32" else rng.choice(("f32", "bf16")), "pages": pages, "ragged": rng.random() < 0.7}
    if op == "attend":
        rows = spread(1, 32)
        if rng.random() < 0.5:
            return {"op": op, "model": model, "rows": rows, "new": 1, "cached": spread(1, 60000 // rows), "page": page, "pages": pages,
                    "ragged": rng.random() < 0.7}
        most = 1200 if pages == "f32" else 6000
        return {"op": op, "model": model, "rows": rows, "new": spread(2, max(2, most // rows)), "cached": spread(1, 4000 // rows), "page": page,
                "pages": pages, "ragged": rng.random() < 0.7}
    if op == "select":
        beams = spread(1, 16)
        return {"op": op, "batch": spread(1, max(1, 190 // beams)), "beams": beams, "keep": spread(1, 16), "vocab": spread(999, 256000),
                "logits": rng.choice(("f32", "bf16")), "finished": rng.random() < 0.5}
    beams = spread(2, 16)
    return {"op": op, "model": model, "batch": spread(1, max(1, 90 // beams)), "beams": beams, "layers": spread(1, 8), "prompt": spread(1, 900),
            "made": spread(1, 100), "page": page, "pages": pages}


# ---------------------------------------------------------------- sizes


def lengths(case):
    """(new tokens, cached tokens with them) of every row."""
    n, rows = case["new"], case["rows"]
    part = [0.25 + 0.75 * ((7 * r + 3) % rows + 1) / rows if case["ragged"] else 1.0 for r in range(rows)]
    new = [max(1, int(n * f)) for f in part]
    return new, [m + int(case["cached"] * f) for m, f in zip(new, part)]


def work(case):
    elem = {"bf16": 2, "f32": 4}
    if case["op"] == "select":
        values = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": float(elem[case["logits"]] * values + 16 * case["batch"] * case["keep"]), "flops": 3.0 * values}
    nh, nkv, d, norms, cap, window, _, _ = MODELS[case["model"]]
    e = elem[case["pages"]]
    if case["op"] == "reorder":
        B, K = case["batch"], case["beams"]
        length, page = case["prompt"] + case["made"], case["page"]
        begun = (length % page) * nkv * d * e * 2 * case["layers"]
        # of K independent parents 1 - (1 - 1 / K)^K differ, and one in K is the beam itself
        moved = B * begun * (K * (1.0 - (1.0 - 1.0 / K) ** K) + K - 1)
        return {"bytes": float(moved + 3 * 4 * B * K * columns(length, page)), "flops": 0.0}
    new, total = lengths(case)
    M = sum(new)
    if case["op"] == "append":
        i = elem[case["inputs"]]
        return {"bytes": float(M * (nh + 2 * nkv) * d * (i + e) + M * d * 4), "flops": float(M * (nh + nkv) * d * (7 if norms else 3))}
    seen = [min(t, (window or 1 << 40) + n - 1) for n, t in zip(new, total)]
    pairs = 0.0
    for n, t in zip(new, total):
        w = window or 1 << 40
        whole = max(0, min(n, t - w + 1))              # queries whose window is full
        rest = n - whole
        pairs += whole * min(w, t) + rest * (t - n + 1) + rest * (rest - 1) / 2
    return {"bytes": float(2 * M * nh * d * e + 2 * sum(seen) * nkv * d * e), "flops": 4.0 * pairs * nh * d}


def columns(length, page):
    """Columns of a table that also names the page behind the last one."""
    return length // page + 2


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    s = dict(case)
    if case["op"] == "select":
        B, J, K, V = case["batch"], case["beams"], case["keep"], case["vocab"]
        # logits of a language model: a few stand out; sums of log-probabilities some steps into the search
        s["logits"] = normal(B, J, V, std=2.5, dtype=TYPES[case["logits"]])
        s["scores"] = -12.0 - 2.0 * normal(B, J).abs()
        done = torch.rand(B, J, generator=gen, device="cuda") < (0.2 if case["finished"] else 0.0)
        s["finished_in"] = done.to(torch.int32)
        s["end"] = V - 7
        s["out"] = (torch.zeros(B, K, device="cuda"), *(torch.zeros(B, K, dtype=torch.int32, device="cuda") for _ in range(3)))
        return s
    nh, nkv, d, norms, cap, window, base, _ = MODELS[case["model"]]
    page, dtype = case["page"], TYPES[case["pages"]]
    if case["op"] == "reorder":
        B, K, L = case["batch"], case["beams"], case["layers"]
        length = case["prompt"] + case["made"]
        P, shared = columns(length, page), case["prompt"] // page
        # a prompt's full pages are one for all its beams; from there on every beam has pages of its own
        ids = torch.randperm(B * (shared + K * (P - shared)), generator=gen, device="cuda").to(torch.int32)
        common = ids[:B * shared].reshape(B, 1, shared).expand(B, K, shared)
        s["own"] = torch.cat([common, ids[B * shared:].reshape(B, K, P - shared)], 2).reshape(B * K, P).contiguous()
        s["table"] = s["own"].clone()
        s["parents"] = torch.randint(0, K, (B, K), generator=gen, device="cuda", dtype=torch.int32)
        s["lens"] = torch.full((B * K,), length, dtype=torch.int32, device="cuda")
        s["k_pages"], s["v_pages"] = (normal(L, ids.numel(), nkv, page, d, dtype=dtype) for _ in range(2))
        return s
    new, total = lengths(case)
    rows, M = len(new), sum(new)
    P = max(columns(t, page) for t in total)
    need = rows * P
    s["table"] = torch.randperm(need, generator=gen, device="cuda").to(torch.int32).reshape(rows, P).contiguous()
    s["starts"], s["lens"], s["most"] = ints(np.concatenate([[0], np.cumsum(new)]).tolist()), ints(total), max(new)
    if case["op"] == "append":
        both = normal(M, (nh + 2 * nkv), d, dtype=TYPES[case["inputs"]])   # one projection makes all three
        s["q"], s["k"], s["v"] = both[:, :nh], both[:, nh:nh + nkv], both[:, nh + nkv:]
        if norms:
            s["q_gain"], s["k_gain"] = 1.0 + normal(d, std=0.1), 1.0 + normal(d, std=0.1)
        angle = np.arange(max(total))[:, None] * base ** (-np.arange(0, d, 2) / d)
        s["cos"], s["sin"] = (torch.tensor(f(angle), dtype=torch.float32, device="cuda") for f in (np.cos, np.sin))
        s["k_pages"], s["v_pages"] = (torch.zeros(need, nkv, page, d, dtype=dtype, device="cuda") for _ in range(2))
        s["out"] = torch.zeros(M, nh, d, dtype=dtype, device="cuda")
        return s
    s["q"] = normal(M, nh, d, std=1.5, dtype=dtype)
    s["k_pages"], s["v_pages"] = (normal(need, nkv, page, d, dtype=dtype) for _ in range(2))
    s["out"] = torch.zeros(M, nh, d, dtype=dtype, device="cuda")
    return s


# ---------------------------------------------------------------- one pass


EPS = 1e-6
_library = {}


def library():
    """The program's backend."""
    if not _library:
        cg = importlib.import_module("catgrad-rs_b200")
        _library["backend"] = cg.CudaBackend(0, cg.PREC_BF16)
    return _library["backend"]


def held(s):
    """What a program of the library holds its tensors by: handles around the device memory they lie in, made when it
    gets them.  (Nothing is copied or laid out.)"""
    if "held" not in s:
        B = library()
        s["held"] = {n: B.from_device(t) for n, t in s.items() if torch.is_tensor(t)}
        if isinstance(s.get("out"), tuple):
            s["held"]["out"] = tuple(B.from_device(t) for t in s["out"])
    return library(), s["held"]


def run(s):
    return {"append": append, "attend": attend, "select": select, "reorder": reorder}[s["op"]](s)


def append(s):
    if own:
        B, h = held(s)
        B.paged_append(h["k"], h["v"], h["k_pages"], h["v_pages"], h["table"], h["starts"], h["lens"], q=h["q"], q_out=h["out"],
                       cos=h["cos"], sin=h["sin"], q_gain=h.get("q_gain"), k_gain=h.get("k_gain"), eps=EPS)
    else:
        row, pos = places(s)
        cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
        at, place = s["table"][row, pos // s["page"]].long(), pos % s["page"]
        s["out"].copy_(turned(normed(s["q"].float(), s.get("q_gain")), cos, sin))
        s["k_pages"][at, :, place] = turned(normed(s["k"].float(), s.get("k_gain")), cos, sin).to(s["k_pages"].dtype)
        s["v_pages"][at, :, place] = s["v"].to(s["v_pages"].dtype)
    return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def places(s):
    """Row and position of every packed token."""
    starts, lens = s["starts"].long(), s["lens"].long()
    m = torch.arange(s["k"].shape[0], device="cuda")
    row = (m[:, None] >= starts[None, 1:]).sum(1)
    return row, lens[row] - starts[row + 1] + m


def normed(x, gain):
    return x if gain is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gain


def turned(x, cos, sin):
    """Component i turns with component i + d / 2."""
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def attend(s):
    nh, nkv, d, _, cap, window, _, _ = MODELS[s["model"]]
    if own:
        B, h = held(s)
        B.paged_attention(h["q"], h["k_pages"], h["v_pages"], h["table"], h["starts"], h["lens"], max_new=s["most"], window=window,
                          softcap=cap, out=h["out"])
        return s["out"]
    rows, most, page = s["table"].shape[0], s["most"], s["page"]
    starts, lens = s["starts"].long(), s["lens"].long()
    new = starts[1:] - starts[:-1]
    i = torch.arange(most, device="cuda")
    token = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)                       # [rows, most]
    q = s["q"][token].float().reshape(rows, most, nkv, nh // nkv, d).permute(0, 2, 3, 1, 4).reshape(rows, nkv, -1, d)
    T = s["table"].shape[1] * page
    k, v = (s[n][s["table"].long()].float().permute(0, 2, 1, 3, 4).reshape(rows, nkv, T, d) for n in ("k_pages", "v_pages"))
    x = (q @ k.transpose(2, 3) / math.sqrt(d)).reshape(rows, nkv, nh // nkv, most, T)
    if cap:
        x = cap * torch.tanh(x / cap)
    at = (lens - new)[:, None] + i                                                        # [rows, most]
    key = torch.arange(T, device="cuda")
    seen = key <= at[..., None]
    if window:
        seen &= key > at[..., None] - window
    x = torch.where(seen[:, None, None], x, -torch.inf)
    x = torch.exp(x - x.max(-1, keepdim=True).values)
    o = (x / x.sum(-1, keepdim=True)).reshape(rows, nkv, -1, T) @ v
    o = o.reshape(rows, nkv, nh // nkv, most, d).permute(0, 3, 1, 2, 4).reshape(rows * most, nh, d)
    m = torch.arange(s["q"].shape[0], device="cuda")
    row = (m[:, None] >= starts[None, 1:]).sum(1)
    s["out"].copy_(o[row * most + m - starts[row]])
    return s["out"]


def select(s):
    K = s["keep"]
    if own:
        B, h = held(s)
        B.beam_select(h["logits"], h["scores"], K, finished=h["finished_in"], end=s["end"], out=h["out"])
    else:
        # in 64 bits: which of two close candidates is taken must not depend on a sum's last bits
        x = s["logits"].double()
        V = x.shape[-1]
        x = x - x.max(-1, keepdim=True).values
        x = x - torch.log(torch.exp(x).sum(-1, keepdim=True))
        v = torch.arange(V, device="cuda")
        done = s["finished_in"][..., None] != 0
        x = torch.where(done, torch.where(v == s["end"], 0.0, -torch.inf), x)
        x = (s["scores"].double()[..., None] + x).reshape(x.shape[0], -1)
        # the K largest; of equal ones those with the lowest place among beams and vocabulary
        least = torch.topk(x, K).values[:, -1:]
        above, level = x > least, x == least
        taken = above | (level & (torch.cumsum(level, 1) <= K - above.sum(1, keepdim=True)))
        place = torch.arange(x.shape[1], device="cuda")
        place = torch.topk(torch.where(taken, place, x.shape[1]), K, largest=False, sorted=True).values
        total, order = torch.sort(x.gather(1, place), descending=True, stable=True)
        place = place.gather(1, order)
        parent, token = place // V, place % V
        s["out"][0].copy_(total)
        s["out"][1].copy_(token)
        s["out"][2].copy_(parent)
        s["out"][3].copy_((s["finished_in"].gather(1, parent) != 0) | (token == s["end"]))
    return dict(zip(("scores", "tokens", "parents", "finished"), s["out"]))


def reorder(s):
    if own:
        B, h = held(s)
        B.paged_reorder(h["parents"], h["lens"], h["own"], h["table"], h["k_pages"], h["v_pages"])
    else:
        B, K = s["parents"].shape
        P, page = s["table"].shape[1], s["page"]
        parent = (torch.arange(B, device="cuda")[:, None] * K + s["parents"]).reshape(-1)
        full = (s["lens"] // page).long()
        row = torch.arange(B * K, device="cuda")
        source, target = s["own"][parent, full].long(), s["own"][row, full].long()
        begun = (torch.arange(page, device="cuda") < (s["lens"] % page)[:, None])[None, :, None, :, None]
        s["k_pages"][:, target] = torch.where(begun, s["k_pages"][:, source], s["k_pages"][:, target])
        s["v_pages"][:, target] = torch.where(begun, s["v_pages"][:, source], s["v_pages"][:, target])
        s["table"].copy_(torch.where(torch.arange(P, device="cuda") < full[:, None], s["table"][parent], s["own"]))
    return {"table": s["table"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ---------------------------------------------------------------- the same in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "reorder":
        return None   # copies
    if case["op"] == "select":
        V = case["vocab"]
        total = torch.log_softmax(s["logits"].double(), -1)
        for b, j in torch.nonzero(s["finished_in"]).tolist():
            total[b, j] = -torch.inf
            total[b, j, s["end"]] = 0.0
        total = (total + s["scores"].double()[..., None]).reshape(case["batch"], -1)
        best = torch.sort(total, dim=1, descending=True, stable=True).values[:, :case["keep"]]
        return {"scores": best, "tokens": None, "parents": None, "finished": None}
    nh, nkv, d, _, cap, window, _, _ = MODELS[case["model"]]
    new, total = lengths(case)
    page, table = case["page"], s["table"].tolist()
    if case["op"] == "append":
        out = torch.zeros(sum(new), nh, d, dtype=torch.float64, device="cuda")
        pages = [s[n].double() for n in ("k_pages", "v_pages")]
        m = 0
        for r, (n, t) in enumerate(zip(new, total)):
            c, z = (s[x][t - n:t].double()[:, None] for x in ("cos", "sin"))
            vectors = []
            for x, gain in ((s["q"], s.get("q_gain")), (s["k"], s.get("k_gain"))):
                x = x[m:m + n].double()
                if gain is not None:
                    x = x * gain.double() * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
                z1, z2 = x[..., :d // 2] + 0.0, x[..., d // 2:] + 0.0
                turn = torch.complex(z1, z2) * torch.complex(c, z)
                vectors.append(torch.cat([turn.real, turn.imag], -1))
            out[m:m + n] = vectors[0]
            for p in range((t - n) // page, (t - 1) // page + 1):
                lo, hi = max(t - n, p * page), min(t, (p + 1) * page)
                for to, x in zip(pages, (vectors[1], s["v"][m:m + n].double())):
                    to[table[r][p], :, lo - p * page:hi - p * page] = x[lo - (t - n):hi - (t - n)].transpose(0, 1)
            m += n
        return {"q": out, "k_pages": pages[0], "v_pages": pages[1]}
    out = torch.zeros(sum(new), nh, d, dtype=torch.float64, device="cuda")
    m = 0
    for r, (n, t) in enumerate(zip(new, total)):
        ids = s["table"][r, :(t - 1) // page + 1].long()
        k, v = (s[x][ids].double().transpose(0, 1).reshape(nkv, -1, d)[:, :t] for x in ("k_pages", "v_pages"))
        at = torch.arange(t - n, t, device="cuda")[:, None]
        key = torch.arange(t, device="cuda")[None]
        hidden = (key > at) | (key <= at - (window or 1 << 40))
        for h in range(nh):
            x = s["q"][m:m + n, h].double() @ k[h // (nh // nkv)].T * d ** -0.5
            if cap:
                x = torch.tanh(x / cap) * cap
            x = torch.softmax(x.masked_fill(hidden, -torch.inf), -1)
            out[m:m + n, h] = x @ v[h // (nh // nkv)]
        m += n
    return out
