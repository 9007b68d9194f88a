"""Serving many requests from one paged key/value cache, as operators to be timed: pages for the next step, attention
over a prefix that many requests share, and the verification of drafted tokens.

Three operators, each a call of the library's (`cg.CudaBackend`), which follow each other in a step of serving:

* `paged_assign`: from the requests' lengths and the tokens that come next, which of them fit, the pages they get from a
  stack of free ones (and what ended requests give back), packed places, positions and slots;
* `paged_shared_attention`: attention of the new tokens over the cached pages, where groups of neighbouring rows have
  their first tokens in common (a system prompt, a document): these are read once for a group;
* `verify_drafts`: how many of a row's drafted tokens stand before the target's probabilities, from given random numbers,
  and the token behind them.

Cached tensors are [pages, key heads, tokens of a page, head size]; row r of a batch has the packed tokens
starts[r] .. starts[r + 1], its first lens[r] cached tokens count (the new ones among them), and its token at
position p lies in page table[r, p // page] at place p % page.

The sizes are those of the models the repository is benchmarked and tested on: heads and vocabularies of the
Llama-3.2-1B, Llama-3-8B, Qwen3-30B-A3B and Gemma-2-2B shapes, of GPT-2, and of the small f32 Llama.
"""
from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
# query heads, key heads, head size, soft-cap, window, vocabulary
MODELS = {
    "llama1b": (32, 8, 64, 0.0, 0, 128256),
    "llama8b": (32, 8, 128, 0.0, 0, 128256),
    "qwen3moe": (32, 4, 128, 0.0, 0, 151936),
    "gemma2": (8, 4, 256, 50.0, 4096, 256000),
    "tiny": (4, 2, 64, 0.0, 0, 32000),
}


def listed():
    def assign(name, rows, drafts, cached, prompt, waiting, page, budget, room):
        return {"name": name, "op": "assign", "rows": rows, "drafts": drafts, "cached": cached, "prompt": prompt, "waiting": waiting, "page": page,
                "budget": budget, "room": room}

    def attend(name, model, groups, rows, new, shared, mine, page, pages="bf16", ragged=False):
        return {"name": name, "op": "attend", "model": model, "groups": groups, "rows": rows, "new": new, "shared": shared, "mine": mine, "page": page,
                "pages": pages, "ragged": ragged}

    def verify(name, rows, drafts, vocab, logits, probs, heat, ragged=False):
        return {"name": name, "op": "verify", "rows": rows, "drafts": drafts, "vocab": vocab, "logits": logits, "probs": probs, "heat": heat,
                "ragged": ragged}

    return [
        # pages of a decode step of the benchmark's batch: launches and latency are all there is
        assign("assign-step", 8, 0, 577, 1, 0.0, 16, 64, 1.0),
        # many requests that run with drafts, some that end, prompts that wait for more pages and places than there are
        assign("assign-mixed", 391, 4, 3001, 2003, 0.3, 32, 16384, 0.5),
        # attention of a decode step of the benchmark's batch behind a short system prompt
        attend("share-step", "llama1b", 1, 8, 1, 512, 65, 16),
        # questions about one long document
        attend("share-document", "llama8b", 1, 64, 1, 16001, 700, 64, ragged=True),
        # drafted tokens of requests behind three system prompts
        attend("share-drafts", "qwen3moe", 3, 30, 5, 4003, 901, 32, ragged=True),
        # wide heads, capped scores and a window that reaches into the prefix
        attend("share-window", "gemma2", 2, 14, 1, 3001, 1999, 32, ragged=True),
        # the f32 model
        attend("share-f32", "tiny", 2, 12, 2, 1501, 213, 16, "f32", True),
        # one user's drafts
        verify("verify-turn", 1, 4, 128256, "f32", "f32", 1.0),
        # many users' drafts
        verify("verify-batch", 40, 4, 151936, "bf16", "bf16", 0.8, True),
        # drafts looked up in the prompt, which have no probabilities, over the largest vocabulary
        verify("verify-lookup", 32, 7, 256000, "bf16", "none", 1.0, True),
        # greedy decoding, rows of logits that begin off a 16-byte boundary
        verify("verify-greedy", 16, 3, 50257, "f32", "none", 0.0),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    op = rng.choice(("assign", "attend", "attend", "verify", "verify"))
    if op == "assign":
        rows = spread(1, 391)
        return {"op": op, "rows": rows, "drafts": rng.randint(0, 7), "cached": spread(1, 3001), "prompt": spread(1, 2003), "waiting": rng.uniform(0.0, 0.3),
                "page": rng.choice((16, 32, 64, 128)), "budget": spread(64, 16384), "room": rng.uniform(0.3, 1.0)}
    if op == "attend":
        model = rng.choice(list(MODELS))
        pages = "f32" if model == "tiny" else "bf16"
        rows, new = spread(1, 64), rng.choice((1, 1, 2, 3, 5, 8))
        most = min(1500 if pages == "f32" else 16000, 64 * 16000 // (rows * new))
        return {"op": op, "model": model, "groups": rng.randint(1, max(1, min(4, rows // 2))), "rows": rows, "new": new, "shared": spread(64, most),
                "mine": spread(9, 700), "page": rng.choice((16, 32, 64, 128)), "pages": pages, "ragged": rng.random() < 0.7}
    rows = spread(1, 64)
    drafts = rng.randint(0, 7)
    vocab = spread(999, min(256000, 60_000_000 // (rows * (drafts + 1))))
    return {"op": op, "rows": rows, "drafts": drafts, "vocab": vocab, "logits": rng.choice(("f32", "bf16")), "probs": rng.choice(("f32", "bf16", "none")),
            "heat": rng.choice((0.0, 0.6, 1.0, 1.0)), "ragged": rng.random() < 0.5}


# ---------------------------------------------------------------- sizes


def shares(case):
    """What part of the largest size each row has."""
    rows = case["rows"]
    return [0.25 + 0.75 * ((7 * r + 3) % rows + 1) / rows if case["ragged"] else 1.0 for r in range(rows)]


def grouped(case):
    """First rows of the groups, and the number of tokens that each shares."""
    G, rows = case["groups"], case["rows"]
    first = [g * rows // G for g in range(G + 1)]
    return first, [max(1, int(case["shared"] * (1.0 - 0.3 * g / G))) for g in range(G)]


def lengths(case):
    """(new tokens, cached tokens with them) of every row of an attention case."""
    first, shared = grouped(case)
    new = [max(1, round(case["new"] * f)) for f in shares(case)]
    own_part = [max(n, int(case["mine"] * f)) for n, f in zip(new, shares(case))]
    group = [g for g in range(case["groups"]) for _ in range(first[g], first[g + 1])]
    return new, [shared[g] + m for g, m in zip(group, own_part)]


def drafted(case):
    """Tokens that each row has run: the last one it had and its drafts."""
    return [1 + max(min(1, case["drafts"]), round(case["drafts"] * f)) for f in shares(case)]


def work(case):
    elem = {"bf16": 2, "f32": 4, "none": 0}
    if case["op"] == "assign":
        rows, page = case["rows"], case["page"]
        tokens = min(case["budget"], rows * (1 + case["drafts"] / 2) + case["waiting"] * rows * case["prompt"] / 2)
        return {"bytes": float(4 * 8 * rows + 8 * tokens + 8 * tokens / page), "flops": float(10 * rows + 4 * tokens)}
    if case["op"] == "verify":
        # a row's positions up to the first draft that does not stand, about two of three do; the drafter's probabilities there
        V, values, judged = case["vocab"], 0.0, 0.0
        for n in drafted(case):
            values += V * sum(0.65 ** i for i in range(n))
            judged += V * (1.0 - 0.65 ** (n - 1))
        return {"bytes": float(elem[case["logits"]] * values + elem[case["probs"]] * judged), "flops": 4.0 * values}
    nh, nkv, d, _, window, _ = MODELS[case["model"]]
    e = elem[case["pages"]]
    new, total = lengths(case)
    first, shared = grouped(case)
    keys, pairs = float(sum(shared)), 0.0
    for g in range(case["groups"]):
        for r in range(first[g], first[g + 1]):
            seen = min(total[r], (window or 1 << 40) + new[r] - 1)
            keys += min(total[r] - shared[g], seen)
            pairs += new[r] * (min(total[r], window or 1 << 40) - (new[r] - 1) / 2)
    return {"bytes": float(2 * sum(new) * nh * d * e + 2 * keys * nkv * d * e), "flops": 4.0 * pairs * nh * d}


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    {"assign": prepare_assign, "attend": prepare_attend, "verify": prepare_verify}[case["op"]](case, s, gen, seed)
    return s


def ints(v):
    return torch.tensor(np.asarray(v, np.int64).astype(np.int32), dtype=torch.int32, device="cuda")


def normal(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def prepare_assign(case, s, gen, seed):
    """Requests in the middle of their lives: most run, some have ended, some wait with their prompts."""
    rng = np.random.default_rng(seed)
    rows, page = case["rows"], case["page"]
    longest = max(case["cached"], case["prompt"]) + case["drafts"] + 1
    cols = -(-longest // page) + 1
    waits = rng.random(rows) < case["waiting"]
    ends = ~waits & (rng.random(rows) < (0.1 if rows > 8 else 0.0))
    lens = np.where(waits, 0, rng.integers(max(1, case["cached"] // 2), case["cached"] + 1, rows))
    new = np.where(waits, rng.integers(max(1, case["prompt"] // 2), case["prompt"] + 1, rows), 1 + rng.integers(0, case["drafts"] + 1, rows))
    # one in four of the requests that run has its first pages from a prompt that others share
    first = np.where(waits | (rng.random(rows) < 0.75), 0, lens // page // 3)
    held = -(-lens // page)
    need = int((-(-(lens + new) // page) - held).clip(0).sum())
    free = max(1, int(case["room"] * need))
    pages = rng.permutation(int(held.sum()) + free + 5)
    table = np.full((rows, cols), 0x7FFFFFFF)
    at = 0
    for r in range(rows):
        table[r, :held[r]] = pages[at:at + held[r]]
        at += held[r]
    stack = np.zeros(2 * rows * cols + 6, np.int64)
    stack[:free] = pages[at:at + free]
    s.update(lens=ints(lens), new=ints(new), done=ints(ends), first=ints(first), held=ints(held), table=ints(table), free=ints(stack), n_free=ints([free]))
    T = case["budget"]
    s.update(held_out=ints(np.zeros(rows)), n_free_out=ints([0]), starts=ints(np.zeros(rows + 1)), lens_out=ints(np.zeros(rows)), positions=ints(np.zeros(T)),
             slots=ints(np.zeros(T)))


def prepare_attend(case, s, gen, seed):
    nh, nkv, d, _, _, _ = MODELS[case["model"]]
    page, dtype, rows = case["page"], TYPES[case["pages"]], case["rows"]
    new, total = lengths(case)
    first, shared = grouped(case)
    cols = max(-(-t // page) for t in total) + 1
    # the full pages of a prefix are one for all of a group; from there on every row has pages of its own
    whole = [n // page for n in shared]
    count = sum(whole) + sum((first[g + 1] - first[g]) * (cols - whole[g]) for g in range(case["groups"]))
    ids = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)
    s["k_pages"], s["v_pages"] = (normal(gen, count, nkv, page, d, dtype=dtype) for _ in range(2))
    table, at = torch.zeros(rows, cols, dtype=torch.int32, device="cuda"), 0
    for g, w in enumerate(whole):
        a, b = first[g], first[g + 1]
        table[a:b, :w] = ids[at:at + w]
        at += w
        n = (b - a) * (cols - w)
        table[a:b, w:] = ids[at:at + n].reshape(b - a, cols - w)
        at += n
        # the prefix's begun page is copied to all of them
        for pages in (s["k_pages"], s["v_pages"]):
            begun = pages[table[a, w].long(), :, :shared[g] % page].clone()
            pages[table[a:b, w].long(), :, :shared[g] % page] = begun
    s["table"], s["starts"], s["lens"] = table, ints(np.concatenate([[0], np.cumsum(new)])), ints(total)
    s["groups_at"], s["shared_by"] = ints(first), ints(shared)
    s["most"], s["longest"] = max(new), max(shared)
    s["q"] = normal(gen, sum(new), nh, d, std=1.5, dtype=dtype)
    s["out"] = torch.zeros(sum(new), nh, d, dtype=dtype, device="cuda")


def prepare_verify(case, s, gen, seed):
    V, rows = case["vocab"], case["rows"]
    n = drafted(case)
    M = sum(n)
    # logits of a language model: a token stands out; the drafter's are much like them
    logits = normal(gen, M, V, std=2.5)
    top = torch.randint(0, V, (M, 1), generator=gen, device="cuda")
    logits.scatter_(1, top, math.log(V) + 2.0 + 3.0 * torch.rand(M, 1, generator=gen, device="cuda"))
    drafter = logits + normal(gen, M, V, std=0.7)
    s["logits"] = logits.to(TYPES[case["logits"]])
    heat = case["heat"] if case["heat"] > 0.0 else 1.0
    if case["probs"] == "none":
        tokens = torch.argmax(drafter, 1)
    else:
        q = torch.softmax(drafter / heat, 1)
        race = torch.rand(M, V, generator=gen, device="cuda").clamp_min(1e-30).log().neg()
        tokens = torch.argmax(q / race, 1)
        s["probs_in"] = q.to(TYPES[case["probs"]])
    starts = np.concatenate([[0], np.cumsum(n)])
    # the draft that the logits at a place judge is the token at the next
    fed = torch.randint(0, V, (M,), generator=gen, device="cuda")
    fed[1:] = torch.where(torch.isin(torch.arange(1, M, device="cuda"), torch.tensor(starts, device="cuda")), fed[1:], tokens[:-1])
    s["tokens"], s["starts"], s["most"] = fed.to(torch.int32), ints(starts), max(n)
    s["uniform"] = torch.rand(M, generator=gen, device="cuda")
    s["temperature"] = case["heat"] * (0.75 + 0.5 * torch.rand(rows, generator=gen, device="cuda")) if case["heat"] != 1.0 else torch.ones(rows, device="cuda")
    s["lens"] = ints([100 + 7 * r + k for r, k in enumerate(n)])
    s["out"] = tuple(torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(3))


# ---------------------------------------------------------------- one pass


_library = {}


def library():
    """The program's backend."""
    if not _library:
        cg = importlib.import_module("catgrad-rs_b200")
        _library["backend"] = cg.CudaBackend(0, cg.PREC_BF16)
    return _library["backend"]


def held(s):
    """What a program of the library holds its tensors by: handles around the device memory they lie in, made when it
    gets them.  (Nothing is copied or laid out.)  And the memory in which the parts of a shared attention are joined."""
    B = library()
    if "handles" not in s:
        h = {n: B.from_device(t) for n, t in s.items() if torch.is_tensor(t)}
        if isinstance(s.get("out"), tuple):
            h["out"] = tuple(B.from_device(t) for t in s["out"])
        if s["op"] == "attend":
            h["work"] = B.paged_shared_work(h["q"], h["k_pages"], h["table"], h["groups_at"], max_new=s["most"], max_shared=s["longest"])
        s["handles"] = h
    return B, s["handles"]


def run(s):
    return {"assign": assign, "attend": attend, "verify": verify}[s["op"]](s)


def assign(s):
    page, T = s["page"], s["budget"]
    if own:
        B, h = held(s)
        B.paged_assign(h["lens"], h["new"], page, h["held"], h["table"], h["free"], h["n_free"], h["starts"], done=h["done"], first=h["first"],
                       lens_out=h["lens_out"], held_out=h["held_out"], n_free_out=h["n_free_out"], positions=h["positions"], slots=h["slots"])
    else:
        lens, new, first, has = (s[n].long() for n in ("lens", "new", "first", "held"))
        done = s["done"] != 0
        rows, cols = s["table"].shape
        col = torch.arange(cols, device="cuda")
        # what ended rows give back, in the order of rows and columns
        back = (done[:, None] & (col >= first[:, None]) & (col < has[:, None])).reshape(-1)
        room = s["free"].shape[0]
        place = s["n_free"].long() + torch.cumsum(back, 0) - 1
        stack = torch.cat([s["free"], s["free"].new_zeros(1)])
        stack[torch.where(back, place, room)] = s["table"].reshape(-1)
        s["free"].copy_(stack[:room])
        count = s["n_free"].long() + back.sum()
        # rows that run go before rows that begin, each kind in order; none overtakes another of its kind
        want = torch.where(done, 0, new)
        need = torch.where(want > 0, ((lens + want + page - 1) // page - has).clamp(min=0), 0)
        runs = lens > first * page

        def total(x):
            a, b = torch.where(runs, x, 0), torch.where(runs, 0, x)
            return torch.where(runs, torch.cumsum(a, 0), a.sum() + torch.cumsum(b, 0))

        fits = (want > 0) & ((need == 0) | (total(need) <= count)) & (total(want) <= T)
        n, take = torch.where(fits, want, 0), torch.where(fits, need, 0)
        begin = total(take) - take
        j = col - has[:, None]
        mine = (j >= 0) & (j < take[:, None])
        at = (count - 1 - begin[:, None] - j).clamp(min=0, max=room - 1)
        s["table"].copy_(torch.where(mine, s["free"][at], s["table"]))
        ends = torch.cumsum(n, 0)
        s["starts"][0] = 0
        s["starts"][1:] = ends
        s["held_out"].copy_(torch.where(done, first, has + take))
        s["lens_out"].copy_(torch.where(done, 0, lens + n))
        s["n_free_out"].copy_(count - take.sum())
        m = torch.arange(T, device="cuda")
        row = (m[:, None] >= ends[None]).sum(1)
        there, row = row < rows, row.clamp(max=rows - 1)
        pos = lens[row] + m - (ends - n)[row]
        slot = s["table"][row, (pos // page).clamp(0, cols - 1)].long() * page + pos % page
        s["positions"].copy_(torch.where(there, pos, s["positions"].long()))
        s["slots"].copy_(torch.where(there, slot, s["slots"].long()))
    return {n: s[n] for n in ("starts", "lens_out", "held_out", "n_free_out", "table", "free", "positions", "slots")}


def attend(s):
    nh, nkv, d, cap, window, _ = MODELS[s["model"]]
    if own:
        B, h = held(s)
        B.paged_shared_attention(h["q"], h["k_pages"], h["v_pages"], h["table"], h["starts"], h["lens"], h["groups_at"], h["shared_by"], h["work"],
                                 max_new=s["most"], max_shared=s["longest"], window=window, softcap=cap, out=h["out"])
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


def verify(s):
    if own:
        B, h = held(s)
        B.verify_drafts(h["logits"], h["tokens"], h["starts"], h["uniform"], probs=h.get("probs_in"), temperature=h["temperature"], lens=h["lens"],
                        max_new=s["most"], out=h["out"])
    else:
        # in 64 bits: which token a random number falls on must not depend on a sum's last bits
        starts = s["starts"].long()
        M, V = s["logits"].shape
        rows = starts.shape[0] - 1
        m = torch.arange(M, device="cuda")
        row = (m[:, None] >= starts[None, 1:]).sum(1)
        v = torch.arange(V, device="cuda")
        x = s["logits"].double()
        best = x.max(1, keepdim=True).values
        best_at = torch.where(x == best, v, V).min(1).values
        heat = s["temperature"].double()[row, None]
        p = torch.exp((x - best) / torch.where(heat > 0, heat, 1.0))
        p = p / p.sum(1, keepdim=True)
        p = torch.where(heat > 0, p, (v == best_at[:, None]).double())
        draft = s["tokens"].long().roll(-1)
        last = m == starts[row + 1] - 1
        px = p.gather(1, draft[:, None])[:, 0]
        qx = s["probs_in"].gather(1, draft[:, None])[:, 0].double() if "probs_in" in s else torch.ones_like(px)
        stands = torch.where(heat[:, 0] > 0, s["uniform"].double() * qx < px, draft == best_at)
        # the first place of a row whose draft does not stand, or its last
        stop = ~stands | last
        place = torch.full((rows,), M, device="cuda").scatter_reduce(0, row, torch.where(stop, m, M), "amin")
        w = p[place]
        kept = last[place]
        if "probs_in" in s:
            rest = (w - s["probs_in"][place].double()).clamp(min=0.0)
        else:
            rest = torch.where(v == draft[place][:, None], 0.0, w)
        rest = torch.where(kept[:, None] | (rest.sum(1, keepdim=True) <= 0.0), w, rest)
        c = torch.cumsum(rest, 1)
        t = s["uniform"][starts[1:] - 1].double()[:, None] * c[:, -1:]
        end = torch.where(rest > 0, v, 0).max(1).values
        token = torch.minimum((c <= t).sum(1), end)
        s["out"][0].copy_(place - starts[:-1])
        s["out"][1].copy_(torch.where(s["temperature"] > 0, token, best_at[place]))
        s["out"][2].copy_(s["lens"].long() - (starts[1:] - 1 - place))
    return dict(zip(("accepted", "next", "lens"), s["out"]))


# ---------------------------------------------------------------- the same in 64 bits


def exact(case, seed):
    if case["op"] == "assign":
        return None   # whole numbers
    s = prepare(case, seed)
    if case["op"] == "verify":
        accepted, following, left = [], [], []
        starts, tokens, heat = s["starts"].tolist(), s["tokens"].tolist(), s["temperature"].tolist()
        u, lens = s["uniform"].tolist(), s["lens"].tolist()
        for r in range(case["rows"]):
            a, b = starts[r], starts[r + 1]
            for m in range(a, b):
                x = s["logits"][m].double()
                if heat[r] > 0:
                    p = torch.softmax(x / heat[r], 0)
                else:
                    p = torch.zeros_like(x)
                    p[int(torch.nonzero(x == x.max())[0])] = 1.0
                if m == b - 1:
                    rest = p
                    break
                q = s["probs_in"][m].double() if "probs_in" in s else torch.zeros_like(p).index_fill_(0, torch.tensor([tokens[m + 1]], device="cuda"), 1.0)
                if u[m] * float(q[tokens[m + 1]]) >= float(p[tokens[m + 1]]):
                    rest = torch.relu(p - q) if heat[r] > 0 else p
                    break
            c = torch.cumsum(rest, 0)
            t = u[b - 1] * float(c[-1])
            accepted.append(m - a)
            following.append(min(int(torch.searchsorted(c, torch.tensor([t], dtype=torch.float64, device="cuda"), right=True)), int(torch.nonzero(rest)[-1])))
            left.append(lens[r] - (b - 1 - m))
        return dict(zip(("accepted", "next", "lens"), (ints(x) for x in (accepted, following, left))))
    nh, nkv, d, cap, window, _ = MODELS[case["model"]]
    new, total = lengths(case)
    page, rep = case["page"], nh // nkv
    out = torch.zeros(sum(new), nh, d, dtype=torch.float64, device="cuda")
    m = 0
    for r, (n, t) in enumerate(zip(new, total)):
        ids = s["table"][r, :(t - 1) // page + 1].long()
        k, v = (s[x][ids].double().transpose(0, 1).reshape(nkv, -1, d)[:, :t] for x in ("k_pages", "v_pages"))
        at = torch.arange(t - n, t, device="cuda")[:, None]
        key = torch.arange(t, device="cuda")[None]
        hidden = (key > at) | (key <= at - (window or 1 << 40))
        for h in range(nkv):
            x = s["q"][m:m + n, h * rep:(h + 1) * rep].double() @ k[h].T * d ** -0.5
            if cap:
                x = torch.tanh(x / cap) * cap
            out[m:m + n, h * rep:(h + 1) * rep] = torch.softmax(x.masked_fill(hidden[:, None], -torch.inf), -1) @ v[h]
        m += n
    return out
