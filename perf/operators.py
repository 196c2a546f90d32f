"""What stands between two steps of a sequence, as operators: attention that keeps the weights every cached position
received, eviction of the positions that received least, and the verification of drafted tokens.

A case names an operator (``op``) and its sizes:

* ``weights``: attention of the last ``new`` tokens of each of ``batch`` sequences over the paged cache (``low`` to ``high``
  positions, these tokens included), with the output; ``scores`` gain each position's weight, summed over rows and query heads.
* ``window``: the same without the output, for the last ``new`` rows of a prompt: which positions they look at.
* ``evict``: of every (cache entry, sequence, kv head) the ``first`` places, the ``recent`` last ones and those of the largest
  scores stay, ``keep`` in all, and move up into pages of their own; ``turn``: rotary keys are turned to their new places.
* ``verify``: ``drafts`` drafted tokens a sequence against the target's logits and the drafter's probabilities.

With ``own`` the calls are those of ``camelid_b200.csrc.ops``; without it the same mathematics in elementary torch operations.
"""
from __future__ import annotations

import math

import torch

own = False
PAGE = 64
_DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    llama1b, llama8b = {"heads": 32, "kv_heads": 8, "dim": 64}, {"heads": 32, "kv_heads": 8, "dim": 128}
    bf16 = {"dtype": "bfloat16"}
    return [
        # one user's next token behind a short prompt: the smallest call, bound by its launches
        {"name": "weights 1b next token of 1", "op": "weights", **llama1b, **bf16, "batch": 1, "low": 517, "high": 517, "new": 1},
        # several users' next tokens behind unequal prompts
        {"name": "weights 8b next token of 8", "op": "weights", **llama8b, **bf16, "batch": 8, "low": 300, "high": 8191, "new": 1},
        # a busy service with long contexts: the cache streams from memory
        {"name": "weights 8b next token of 16 long", "op": "weights", **llama8b, **bf16, "batch": 16, "low": 24001, "high": 32768, "new": 1},
        # a step of the last token and four drafted ones
        {"name": "weights 1b drafts of 8", "op": "weights", **llama1b, **bf16, "batch": 8, "low": 1500, "high": 4100, "new": 5},
        # the 32-bit path at a head size of its own
        {"name": "weights float32 96", "op": "weights", "heads": 12, "kv_heads": 4, "dim": 96, "dtype": "float32", "batch": 4,
         "low": 700, "high": 2047, "new": 1},
        # what a prompt's last 32 tokens look at
        {"name": "window 1b prompt", "op": "window", **llama1b, **bf16, "batch": 1, "low": 2000, "high": 2000, "new": 32},
        # long prompts of several users, 64 rows each
        {"name": "window 8b prompts", "op": "window", **llama8b, **bf16, "batch": 4, "low": 9001, "high": 16384, "new": 64},
        # a chat that passed its budget, all layers of the small model at once
        {"name": "evict 1b chat", "op": "evict", "entries": 16, "kv_heads": 8, "dim": 64, **bf16, "batch": 1, "low": 641, "high": 641,
         "keep": 512, "first": 4, "recent": 64, "turn": True},
        # long contexts cut to half
        {"name": "evict 8b long", "op": "evict", "entries": 4, "kv_heads": 8, "dim": 128, **bf16, "batch": 4, "low": 24001, "high": 32768,
         "keep": 16384, "first": 4, "recent": 1024, "turn": True},
        # one user's four drafted tokens
        {"name": "verify of 1", "op": "verify", "vocab": 128256, "batch": 1, "drafts": 4, "probs": True, "temperature": 0.8, "top_k": 0,
         "top_p": 1.0, "min_p": 0.0},
        # several users, tokens drafted by look-up (no probabilities of their own), the sampler's filters on
        {"name": "verify of 8 filtered", "op": "verify", "vocab": 128256, "batch": 8, "drafts": 4, "probs": False, "temperature": 0.7,
         "top_k": 0, "top_p": 0.9, "min_p": 0.02},
        # a full batch of a service
        {"name": "verify of 64", "op": "verify", "vocab": 128256, "batch": 64, "drafts": 7, "probs": True, "temperature": 1.0, "top_k": 0,
         "top_p": 1.0, "min_p": 0.0},
    ]


def _between(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("weights", "weights", "window", "evict", "verify", "verify"))
    if op in ("weights", "window"):
        kv_heads = rng.choice((1, 2, 4, 8, 8))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 8))
        dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
        dim = rng.choice((64, 128, 64, 128, 16, 80, 96, 256))
        batch = _between(rng, 1, 16)
        new = _between(rng, 1, 8) if op == "weights" else _between(rng, 2, 64)
        fast = dtype == "bfloat16" and dim in (64, 128)
        room = (500_000 if fast else 40_000) if op == "weights" else (4_000_000 if fast else 300_000) // new
        high = _between(rng, 1, max(2, min(32768, room // batch)))
        return {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "batch": batch,
                "low": rng.randint(max(1, high // 8), high), "high": high, "new": new}
    if op == "evict":
        entries, kv_heads, batch = _between(rng, 1, 16), rng.choice((1, 2, 4, 8)), _between(rng, 1, 16)
        dtype, dim = rng.choice(("bfloat16", "bfloat16", "float32")), rng.choice((64, 128, 80, 16, 256))
        room = 1_500_000_000 // (4 * dim * (4 if dtype == "float32" else 2) + 16)
        high = _between(rng, 2, max(3, min(32768, room // (entries * batch * kv_heads))))
        keep = rng.randint(1, high)
        return {"op": "evict", "entries": entries, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "batch": batch,
                "low": rng.randint(max(1, high // 4), high), "high": high, "keep": keep, "first": rng.randint(0, 8), "recent": rng.randint(0, keep), "turn": rng.random() < 0.6}
    vocab = rng.choice((128256, 32000, 50257, _between(rng, 100, 128256)))
    drafts = rng.randint(0, 7)
    batch = _between(rng, 1, 64)
    filters = rng.random() < 0.4
    return {"op": "verify", "vocab": vocab, "batch": batch, "drafts": drafts, "probs": rng.random() < 0.6,
            "temperature": rng.choice((0.0, 0.6, 0.8, 1.0, 1.5)), "top_k": rng.choice((0, 40, 1000)) if filters else 0,
            "top_p": rng.choice((1.0, 0.9, 0.5)) if filters else 1.0, "min_p": rng.choice((0.0, 0.05)) if filters else 0.0}


# ---- inputs ------------------------------------------------------------------------------------------------------
def _lengths(case):
    n, low, high = case["batch"], min(case["low"], case["high"]), case["high"]
    spread = [low + (high - low) * i // max(n - 1, 1) for i in range(n)] if n > 1 else [high]
    return spread[::2] + spread[1::2][::-1]                                   # neither sorted nor by turns


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(pages_each, ids, width=None):
    """Rows of page ids taken from ``ids`` one after another, padded with -1."""
    width = width or max(pages_each)
    rows, at = [], 0
    for n in pages_each:
        rows.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return rows


def _pages_of(n):
    return (n + PAGE - 1) // PAGE


def _old_scores(gen, shape):
    """Weights as they add up: a few large ones, many small ones, exact ties among the smallest."""
    s = torch.rand(shape, generator=gen, device="cuda").pow_(8.0).mul_(40.0)
    return torch.where(s < 1e-4, torch.zeros_like(s), s)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    if case["op"] == "verify":
        return _prepare_verify(case, gen)
    dt = _DTYPES[case["dtype"]]
    lengths = _lengths(case)
    kvh, dim = case["kv_heads"], case["dim"]
    used = [_pages_of(n) for n in lengths]
    if case["op"] == "evict":
        keeps = [min(case["keep"], n) for n in lengths]
        kept_pages = [_pages_of(n) for n in keeps]
        n_pages = sum(used) + sum(kept_pages) + 3
        ids = torch.randperm(n_pages, generator=gen, device="cuda").tolist()
        shape = (case["entries"], n_pages, kvh, PAGE, dim)
        state = {"case": case, "lengths": lengths, "keeps": keeps,
                 "k": torch.randn(shape, generator=gen, device="cuda", dtype=dt), "v": torch.randn(shape, generator=gen, device="cuda", dtype=dt),
                 "scores": _old_scores(gen, shape[:-1]), "table": _ints(_table(used, ids)),
                 "out_table": _ints(_table(kept_pages, ids[sum(used):])), "lengths_dev": _ints(lengths), "keeps_dev": _ints(keeps),
                 "kept": torch.full((case["entries"], len(lengths), kvh, max(keeps)), -1, dtype=torch.int32, device="cuda"),
                 "inv_freq": (500000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)).float()}
        return state
    news = [min(case["new"], n) for n in lengths]
    n_pages = sum(used) + 3
    ids = torch.randperm(n_pages, generator=gen, device="cuda").tolist()
    rows = sum(news)
    shape = (n_pages, kvh, PAGE, dim)
    k = torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    v = torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    q = (2.0 * torch.randn(rows, case["heads"] * dim, generator=gen, device="cuda")).to(dt)
    scores = _old_scores(gen, shape[:-1])
    row0 = [sum(news[:i]) for i in range(len(news))]
    state = {"case": case, "lengths": lengths, "news": news, "row0": row0, "q": q, "k": k, "v": v, "scores": scores,
             "scores_out": scores.clone(), "table": _ints(_table(used, ids, max(used) + 1)), "row0_dev": _ints(row0),
             "start_dev": _ints([n - m for n, m in zip(lengths, news)]), "new_dev": _ints(news),
             "out": torch.zeros_like(q) if case["op"] == "weights" else None}
    if own:
        from camelid_b200.csrc import ops
        state["scratch"] = torch.empty(ops.attn_weights_floats(len(news), case["heads"], kvh, dim, dt, max(news), max(lengths),
                                                               case["op"] == "weights"), dtype=torch.float32, device="cuda")
    return state


def _prepare_verify(case, gen):
    n, k, vocab = case["batch"], case["drafts"], case["vocab"]
    lens = [max(0, k - (i % 3 if n > 1 else 0)) for i in range(n)]             # some sequences drafted fewer tokens
    row0 = [sum(lens[:i]) + i for i in range(n)]
    rows = sum(lens) + n
    logits = 2.5 * torch.randn(rows, vocab, generator=gen, device="cuda")
    logits += 6.0 * (torch.rand(rows, vocab, generator=gen, device="cuda") < 8.0 / vocab)
    temperature = case["temperature"] or 1.0
    # the drafter: the target's logits and a good deal of noise; its tokens are drawn from its own probabilities
    drafts = torch.zeros(n, max(k, 1), dtype=torch.int32, device="cuda")
    probs = torch.zeros(n, max(k, 1), vocab, device="cuda") if case["probs"] else None
    for i in range(n):
        if lens[i] == 0:
            continue
        own_rows = logits[row0[i]:row0[i] + lens[i]]
        guess = torch.softmax((own_rows + 0.5 * torch.randn(own_rows.shape, generator=gen, device="cuda")) / temperature, -1)
        token = torch.multinomial(guess, 1, generator=gen)[:, 0] if case["probs"] else own_rows.argmax(-1)
        drafts[i, :lens[i]] = token.int()
        if case["probs"]:
            probs[i, :lens[i]] = guess
    state = {"case": case, "lens": lens, "logits": logits, "row0_dev": _ints(row0), "lens_dev": _ints(lens), "drafts": drafts,
             "probs": probs, "accept": torch.rand(n, max(k, 1), generator=gen, device="cuda"),
             "next": torch.rand(n, generator=gen, device="cuda")}
    if own:
        from camelid_b200.csrc import ops
        state["counts"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        state["tokens"] = torch.zeros(n, max(k, 1) + 1, dtype=torch.int32, device="cuda")
        state["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        state["scratch"] = torch.empty(ops.verify_bytes(rows, n, vocab), dtype=torch.uint8, device="cuda")
    return state


# ---- the calls ---------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "verify":
        return _run_verify(state)
    if case["op"] == "evict":
        return _run_evict(state)
    scale = 1.0 / math.sqrt(case["dim"])
    if own:
        from camelid_b200.csrc import ops
        ops.attn_paged_weights(state["q"], state["out"], state["k"], state["v"] if state["out"] is not None else None, state["scores"],
                               state["table"], state["row0_dev"], state["start_dev"], state["new_dev"], case["heads"],
                               max(state["news"]), max(state["lengths"]), scale, state["scratch"], scores_out=state["scores_out"])
        return {"out": state["out"], "scores": state["scores_out"]}
    kvh, dim, heads = case["kv_heads"], case["dim"], case["heads"]
    group = heads // kvh
    for i, (length, new, row0) in enumerate(zip(state["lengths"], state["news"], state["row0"])):
        pages = state["table"][i, :_pages_of(length)].long()
        keys = state["k"][pages].transpose(0, 1).reshape(kvh, -1, dim)[:, :length].float()
        q = state["q"][row0:row0 + new].float().view(new, kvh, group, dim).permute(1, 2, 0, 3).reshape(kvh, group * new, dim)
        s = torch.matmul(q, keys.transpose(1, 2)) * scale
        place = torch.arange(length, device="cuda")
        last = length - new + torch.arange(new, device="cuda").repeat(group)
        s = s.masked_fill(place[None, None, :] > last[None, :, None], -math.inf)
        w = torch.exp(s - s.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        if state["out"] is not None:
            values = state["v"][pages].transpose(0, 1).reshape(kvh, -1, dim)[:, :length].float()
            o = torch.matmul(w, values).view(kvh, group, new, dim).permute(2, 0, 1, 3).reshape(new, heads * dim)
            state["out"][row0:row0 + new] = o.to(state["out"].dtype)
        gained = w.sum(1)
        page_of, at = pages[place // PAGE], place % PAGE
        old = state["scores"][page_of, :, at] * (place < length - new)[:, None]
        state["scores_out"][page_of, :, at] = old + gained.transpose(0, 1)
    return {"out": state["out"], "scores": state["scores_out"]}


def _run_evict(state):
    case = state["case"]
    outputs = {"kept": state["kept"], "k": state["k"], "v": state["v"], "scores": state["scores"]}
    if own:
        from camelid_b200.csrc import ops
        ops.evict_positions(state["k"], state["v"], state["scores"], state["table"], state["out_table"], state["lengths_dev"],
                            state["keeps_dev"], state["kept"], case["first"], case["recent"],
                            inv_freq=state["inv_freq"] if case["turn"] else None)
        return outputs
    half = case["dim"] // 2
    for i, (length, keep) in enumerate(zip(state["lengths"], state["keeps"])):
        place = torch.arange(length, device="cuda")
        page_of, at = state["table"][i].long()[place // PAGE], place % PAGE
        first = min(case["first"], keep)
        recent = min(case["recent"], keep - first)
        rank = state["scores"][:, page_of, :, at].permute(1, 2, 0).clone()     # (places, entries, heads) -> entries, heads, places
        rank[..., :first] = math.inf
        rank[..., length - recent:] = math.inf
        order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
        chosen = torch.sort(order, dim=-1).values                              # entries, heads, keep
        state["kept"][:, i, :, :keep] = chosen.int()
        entry = torch.arange(case["entries"], device="cuda")[:, None, None]
        head = torch.arange(case["kv_heads"], device="cuda")[None, :, None]
        src = (entry, page_of[chosen], head, at[chosen])
        new = torch.arange(keep, device="cuda")
        dst = (entry, state["out_table"][i].long()[new // PAGE][None, None, :], head, (new % PAGE)[None, None, :])
        keys = state["k"][src]
        if case["turn"]:
            angle = (new[None, None, :] - chosen).double()[..., None] * state["inv_freq"].double()
            cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
            a, b = keys[..., :half].float(), keys[..., half:].float()
            keys = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(keys.dtype)
        state["k"][dst] = keys
        state["v"][dst] = state["v"][src]
        state["scores"][dst] = state["scores"][src]
    return outputs


def _target(logits, case):
    """The target's probabilities in 64 bits, filtered as the sampler filters them."""
    if case["temperature"] == 0.0:
        best = logits.argmax(-1, keepdim=True)
        return torch.zeros(logits.shape, dtype=torch.float64, device="cuda").scatter_(1, best, 1.0)
    z = logits.double()
    z = (z - z.amax(-1, keepdim=True)) / float(torch.tensor(case["temperature"], dtype=torch.float32))
    e = torch.exp(z)
    if case["top_k"] or case["min_p"] > 0.0 or case["top_p"] < 1.0:
        top_p, min_p = (float(torch.tensor(case[x], dtype=torch.float32)) for x in ("top_p", "min_p"))
        order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
        e = e.gather(1, order)
        if case["top_k"]:
            e[:, case["top_k"]:] = 0.0
        if min_p > 0.0:
            e = e * (e >= min_p)
        if top_p < 1.0:
            before = torch.cumsum(e / e.sum(-1, keepdim=True), -1)
            before = torch.cat([torch.zeros_like(before[:, :1]), before[:, :-1]], -1)
            e = e * (before < top_p)
        e = torch.zeros_like(e).scatter_(1, order, e)
    return e / e.sum(-1, keepdim=True)


def _run_verify(state):
    case = state["case"]
    if own:
        from camelid_b200.csrc import ops
        ops.verify_drafts(state["logits"], state["row0_dev"], state["lens_dev"], state["drafts"], state["probs"], state["accept"],
                          state["next"], case["temperature"], case["top_k"], case["top_p"], case["min_p"], state["counts"],
                          state["tokens"], state["err"], state["scratch"])
        return {"counts": state["counts"], "tokens": state["tokens"]}
    p = _target(state["logits"], case)
    n, width = state["drafts"].shape
    row0, lens, drafts = state["row0_dev"].long(), state["lens_dev"].long(), state["drafts"].long()
    seq = torch.arange(n, device="cuda")
    step = torch.arange(width, device="cuda")[None, :]
    there = step < lens[:, None]
    rows = torch.where(there, row0[:, None] + step, row0[:, None])
    px = p[rows, drafts]
    qx = state["probs"][seq[:, None], step, drafts].double() if state["probs"] is not None else torch.ones_like(px)
    accepted = (there & (state["accept"].double() * qx < px)).long().cumprod(1)
    counts = accepted.sum(1)
    last = p[row0 + counts]
    rejected = counts < lens
    at = torch.clamp(counts, max=width - 1)
    if state["probs"] is not None:
        taken = state["probs"][seq, at].double()
    else:
        taken = torch.zeros_like(last).scatter_(1, drafts[seq, at][:, None], 2.0)
    rest = torch.clamp(last - taken * rejected[:, None], min=0.0)
    rest = torch.where((rest.sum(1) > 0.0)[:, None], rest, last)
    total = torch.cumsum(rest, 1)
    over = total > (state["next"].double() * rest.sum(1))[:, None]
    found = torch.argmax(over.long(), 1)
    back = case["vocab"] - 1 - torch.argmax((rest > 0).flip(1).long(), 1)
    found = torch.where(over.any(1), found, back)
    places = torch.arange(width + 1, device="cuda")[None, :]
    padded = torch.cat([drafts, torch.zeros_like(drafts[:, :1])], 1)
    tokens = torch.where(places < counts[:, None], padded, torch.where(places == counts[:, None], found[:, None], -1))
    return {"counts": counts.int(), "tokens": tokens.int()}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "verify":
        n, k, vocab = case["batch"], case["drafts"], case["vocab"]
        rows = sum(max(0, k - (i % 3 if n > 1 else 0)) for i in range(n)) + n
        return {"bytes": 4.0 * vocab * (rows + (n if case["probs"] and k else 0)) + 4.0 * n * (4 * k + 6), "flops": 4.0 * rows * vocab}
    size = 4 if case["dtype"] == "float32" else 2
    lengths, kvh, dim = _lengths(case), case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        kept = sum(min(case["keep"], n) for n in lengths)
        per = case["entries"] * kvh
        return {"bytes": per * (4.0 * sum(lengths) + kept * (2.0 * 2 * dim * size + 12.0)), "flops": per * kept * dim * 3.0 * case["turn"]}
    news = [min(case["new"], n) for n in lengths]
    with_out = case["op"] == "weights"
    keys, pairs = sum(lengths), sum(n * m for n, m in zip(lengths, news))
    return {"bytes": keys * kvh * (dim * size * (2 if with_out else 1) + 8.0) + sum(news) * case["heads"] * dim * size * (2 if with_out else 1),
            "flops": (4.0 if with_out else 2.0) * pairs * case["heads"] * dim}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "verify":
        return _exact_verify(state)
    kvh, dim = case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        return _exact_evict(state)
    scores = state["scores"].double()
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda") if case["op"] == "weights" else None
    group = case["heads"] // kvh
    for i, length in enumerate(state["lengths"]):
        new, row0 = state["news"][i], state["row0"][i]
        blocks = state["table"][i].tolist()[:_pages_of(length)]
        for h in range(kvh):
            keys = torch.cat([state["k"][b, h] for b in blocks])[:length].double()
            values = torch.cat([state["v"][b, h] for b in blocks])[:length].double()
            gained = torch.zeros(length, dtype=torch.float64, device="cuda")
            for j in range(new):
                seen = length - new + j + 1
                q = state["q"][row0 + j].double().view(-1, dim)[h * group:(h + 1) * group]
                w = torch.softmax(q @ keys[:seen].T / math.sqrt(dim), -1)
                gained[:seen] += w.sum(0)
                if out is not None:
                    out[row0 + j].view(-1, dim)[h * group:(h + 1) * group] = w @ values[:seen]
            where = scores[blocks, h].reshape(-1)
            where[:length - new] += gained[:length - new]
            where[length - new:length] = gained[length - new:]
            scores[blocks, h] = where.view(-1, PAGE)
    return {"out": out, "scores": scores}


def _exact_evict(state):
    case = state["case"]
    kept, k, v, scores = state["kept"], state["k"].double(), state["v"].double(), state["scores"].double()
    dim = case["dim"]
    for i, (length, keep) in enumerate(zip(state["lengths"], state["keeps"])):
        table, out_table = state["table"][i].tolist(), state["out_table"][i].tolist()
        blocks, to = table[:_pages_of(length)], out_table[:_pages_of(keep)]
        first = min(case["first"], keep)
        recent = min(case["recent"], keep - first)
        for e in range(case["entries"]):
            for h in range(case["kv_heads"]):
                s = scores[e, blocks, h].reshape(-1)[:length]
                middle = s[first:length - recent]
                # the largest of the middle, the lower place first among equals: a stable ascending sort of the negated scores
                best = torch.sort(-middle, stable=True).indices[:keep - first - recent] + first
                chosen = torch.cat([torch.arange(first, device="cuda"), best.sort().values, torch.arange(length - recent, length, device="cuda")])
                kept[e, i, h, :keep] = chosen.int()
                keys = k[e, blocks, h].reshape(-1, dim)[chosen]
                if case["turn"]:
                    turn = torch.polar(torch.ones(keep, dim // 2, dtype=torch.float64, device="cuda"),
                                       (torch.arange(keep, device="cuda") - chosen).double()[:, None] * state["inv_freq"].double()[None, :])
                    pairs = torch.complex(keys[:, :dim // 2], keys[:, dim // 2:]) * turn
                    keys = torch.cat([pairs.real, pairs.imag], 1)
                moved = (keys, v[e, blocks, h].reshape(-1, dim)[chosen], s[chosen])
                for target, rows in zip((k, v, scores), moved):
                    held = target[e, to, h].reshape(len(to) * PAGE, *rows.shape[1:])
                    held[:keep] = rows
                    target[e, to, h] = held.view(len(to), PAGE, *rows.shape[1:])
    return {"kept": kept, "k": k, "v": v, "scores": scores}


def _exact_verify(state):
    case = state["case"]
    n, width = state["drafts"].shape
    counts, tokens = [], []
    row0, drafts, accept, draws = (state[x].tolist() for x in ("row0_dev", "drafts", "accept", "next"))

    def distribution(row):
        x = state["logits"][row].double()
        if case["temperature"] == 0.0:
            p = torch.zeros_like(x)
            p[int(torch.nonzero(x == x.max())[0])] = 1.0
            return p
        x = x / float(torch.tensor(case["temperature"], dtype=torch.float32))
        values, order = torch.sort(x, descending=True, stable=True)
        p = torch.softmax(values, 0)
        if case["top_k"]:
            p = p[:case["top_k"]] / p[:case["top_k"]].sum()
        if case["min_p"] > 0.0:
            p = p[p >= p[0] * float(torch.tensor(case["min_p"], dtype=torch.float32))]
            p = p / p.sum()
        if case["top_p"] < 1.0:
            stop = int((torch.cumsum(p, 0) < float(torch.tensor(case["top_p"], dtype=torch.float32))).sum()) + 1
            p = p[:stop] / p[:stop].sum()
        full = torch.zeros_like(x)
        full[order[:p.numel()]] = p
        return full

    for i in range(n):
        picked, j = [], 0
        while True:
            p = distribution(row0[i] + j)
            if j == state["lens"][i]:
                break
            x = drafts[i][j]
            q = state["probs"][i, j].double() if state["probs"] is not None else torch.zeros_like(p).index_fill_(0, torch.tensor([x], device="cuda"), 1.0)
            if not accept[i][j] * float(q[x]) < float(p[x]):
                rest = (p - q).clamp(min=0.0)
                p = rest if float(rest.sum()) > 0.0 else p
                break
            picked.append(x)
            j += 1
        walk = torch.cumsum(p, 0)
        over = torch.nonzero(walk > draws[i] * p.sum())
        picked.append(int(over[0]) if over.numel() else int(torch.nonzero(p)[-1]))
        counts.append(j)
        tokens.append(picked + [-1] * (width + 1 - len(picked)))
    return {"counts": torch.tensor(counts, dtype=torch.int32), "tokens": torch.tensor(tokens, dtype=torch.int32)}
