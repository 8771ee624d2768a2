"""Operators of a server that runs many sequences at once on one pool of KV-cache pages.

Three operators, which a serving step calls one after the other:

- ``tables``: the step's block tables, slot map and positions, built on the GPU from the
  requests' lengths (``PageTable.truncate`` takes back what a draft got wrong or a finished
  request held, ``PageTable.extend`` gives each request room for its new tokens);
- ``attention``: the attention of a chunk of new tokens of every request over the paged
  cache, their own keys and values appended first (``PagedKvCache.attention``), from one
  token a request to whole prompts;
- ``attention`` with ``window`` > 0: the same with a sliding window and the first ``sinks``
  tokens always visible.

Head layouts are Llama-2-7B's (32 heads of 128), Mistral-7B's (32 over 8 of 128) and
TinyLlama-1.1B's (32 over 4 of 64), and one of 256 wide heads.  Lengths are ragged and come
from the case alone (``lengths`` seeds them); values come from the seed.

Definitions.  A page holds ``page`` positions of one layer: K pages [pages, kv heads, page,
hd], V pages [pages, kv heads, hd, page] (keys contiguous).  ``free`` is a stack of free
pages, its top at n_free - 1.  ``extend`` pops a page for each that an entry's new length
needs beyond its old one, entries in order; ``truncate`` pushes the pages past the new
length so that it undoes the extend it takes back, and sets their table entries to -1.  A
token at position p sees the keys j <= p with j > p - window (window > 0) or j < sinks.
q and k are rotated (half-split) by the angles p * theta^(-2 i / hd), k and v are rounded
once to the cache's type, and softmax(q k^T / sqrt(hd)) v is f32.
"""
from __future__ import annotations

import math
import random

import torch

own = False

THETA = 10000.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ITEM = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases --------------------------------------------------------------------------
def _tables(name, page, seqs, ctx, new, back, lengths):
    return {"name": name, "op": "tables", "page": page, "seqs": seqs, "ctx_min": ctx[0],
            "ctx_max": ctx[1], "new_min": new[0], "new_max": new[1], "back": back,
            "lengths": lengths}


def _attention(name, dtype, heads, hd, page, seqs, ctx, new, chunks, window=0, sinks=0, lengths=1):
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads[0],
            "kv_heads": heads[1], "hd": hd, "page": page, "seqs": seqs, "ctx_min": ctx[0],
            "ctx_max": ctx[1], "new_min": new[0], "new_max": new[1], "chunks": chunks,
            "window": window, "sinks": sinks, "lengths": lengths}


def listed():
    return [
        # a decode step of a few requests: launch latency
        _tables("tables_step_8", 16, 8, (20, 3000), (1, 1), 0, 1),
        # a busy server with drafted tokens: some rolled back, new ones drafted
        _tables("tables_draft_256", 16, 256, (1, 8000), (1, 9), 5, 2),
        # an offline batch's prompt chunks, over a hundred thousand tokens at once
        _tables("tables_prompts_2048", 32, 2048, (0, 4000), (1, 129), 3, 3),
        # one chat request's next token (Llama-2-7B's heads)
        _attention("decode_1_f16", "f16", (32, 32), 128, 16, 1, (1024, 1024), (1, 1), 0),
        # a continuous batch's decode step, ragged (Mistral-7B's heads)
        _attention("decode_64_bf16", "bf16", (32, 8), 128, 16, 64, (256, 8192), (1, 1), 0, lengths=4),
        # two requests over whole books
        _attention("decode_long_f16", "f16", (32, 8), 128, 128, 2, (90001, 131040), (1, 1), 0, lengths=5),
        # drafted tokens verified (TinyLlama's heads, an f32 cache)
        _attention("verify_16_f32", "f32", (32, 4), 64, 32, 16, (100, 2000), (2, 5), 16, lengths=6),
        # a new prompt
        _attention("prompt_2048_f16", "f16", (32, 32), 128, 16, 1, (0, 0), (2048, 2048), 1),
        # prompt chunks among decoding requests, the step of a chunked prefill
        _attention("mixed_24_bf16", "bf16", (32, 8), 128, 64, 24, (1, 6001), (301, 511), 3, lengths=8),
        # a chunk behind a cached prefix, wide heads, f32
        _attention("chunk_500_f32_hd256", "f32", (8, 1), 256, 32, 1, (777, 777), (500, 500), 1),
        # a decode step of long chats with a sliding window and attention sinks
        _attention("window_decode_48_bf16", "bf16", (32, 8), 128, 32, 48, (4096, 32768), (1, 1), 0,
                   4096, 4, lengths=10),
        # long prompts' chunks under a short window (TinyLlama's heads)
        _attention("window_chunk_2_f16", "f16", (32, 4), 64, 16, 2, (3001, 6007), (2001, 4096), 2,
                   1024, 4, lengths=11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.25:
        page = rng.choice((16, 32, 64, 128))
        while True:
            seqs, ctx, new = _log(rng, 1, 2048), _log(rng, 1, 8000), _log(rng, 1, 129)
            if seqs * new <= 120000 and seqs * (ctx + new) <= 5_000_000:
                break
        return {"op": "tables", "page": page, "seqs": seqs, "ctx_min": rng.randrange(ctx + 1),
                "ctx_max": ctx, "new_min": rng.randint(1, new), "new_max": new,
                "back": rng.randrange(8), "lengths": rng.randrange(1 << 20)}
    while True:
        hd = rng.choice((64, 128, 128, 256))
        kv_heads = _log(rng, 1, 32)
        heads = kv_heads * rng.choice((1, 1, 2, 4, 7, 8, 16))
        if heads > 64:
            continue
        seqs = _log(rng, 1, 128)
        ctx_max = _log(rng, 1, 130000)
        chunked = rng.random() < 0.5
        new_max = _log(rng, 2, 4096) if chunked else 1
        case = {"op": "attention", "dtype": rng.choice(("f32", "f16", "bf16")), "heads": heads,
                "kv_heads": kv_heads, "hd": hd, "page": rng.choice((16, 32, 64, 128, 256)),
                "seqs": seqs, "ctx_min": rng.randrange(ctx_max + 1), "ctx_max": ctx_max,
                "new_min": rng.randint((new_max + 1) // 2, new_max), "new_max": new_max,
                "chunks": rng.randint(1, seqs) if chunked else 0,
                "window": _log(rng, 1, 8192) if rng.random() < 0.4 else 0, "sinks": 0,
                "lengths": rng.randrange(1 << 20)}
        if case["window"]:
            case["sinks"] = rng.choice((0, 1, 4, 4, 37))
        # within the largest listed cases' costs, padded as the plain form pads them
        longest = ctx_max + new_max
        w = work(case)
        if (seqs * longest * kv_heads * hd <= 1_600_000_000
                and seqs * heads * new_max * longest <= 1_100_000_000
                and w["bytes"] <= 1_000_000_000 and w["flops"] <= 56e9):
            return case


def _lengths(case):
    """(cached, new) tokens of each sequence, from the case alone."""
    r = random.Random(case["lengths"])
    n = case["seqs"]
    lo, hi = math.log(case["ctx_min"] + 1), math.log(case["ctx_max"] + 1)
    ctx = [min(case["ctx_max"], int(math.exp(r.uniform(lo, hi)) - 0.5)) for _ in range(n)]
    ctx[r.randrange(n)] = case["ctx_max"]
    if case["op"] == "tables":
        return ctx, [r.randint(case["new_min"], case["new_max"]) for _ in range(n)]
    chunked = set(r.sample(range(n), case["chunks"]))
    return ctx, [r.randint(case["new_min"], case["new_max"]) if i in chunked else 1 for i in range(n)]


def _backs(case, ctx):
    r = random.Random(case["lengths"] + 1)
    return [min(c, r.randint(0, case["back"])) for c in ctx]


def _seen(case, p):
    """Keys that a token at position p sees."""
    w = case["window"]
    return p + 1 if not w or p + 1 <= w else w + min(case["sinks"], p + 1 - w)


def work(case):
    ctx, new = _lengths(case)
    page = case["page"]
    up = lambda n: -(-n // page)  # noqa: E731
    if case["op"] == "tables":
        back = _backs(case, ctx)
        given = sum(up(c - b) for c, b in zip(ctx, back))
        freed = sum(up(c) for c in ctx) - given
        taken = sum(up(c - b + n) for c, b, n in zip(ctx, back, new)) - given
        # ids and lengths of both calls, the lengths' update, a page read and written for each
        # freed and taken, a slot and a position for each token
        return {"bytes": case["seqs"] * 32 + (freed + taken) * 8 + sum(new) * 8, "flops": 0}
    h, g, hd, size = case["heads"], case["kv_heads"], case["hd"], ITEM[case["dtype"]]
    keys = pairs = 0
    for c, n in zip(ctx, new):
        # every key that some new token sees; (key, token) pairs
        w = case["window"]
        low = max(0, c + 1 - w) if w else 0
        keys += c + n - low + min(case["sinks"], low)
        if not w:
            pairs += n * c + n * (n + 1) // 2
        else:
            pairs += sum(_seen(case, c + t) for t in range(n))
    tokens = sum(new)
    # the keys and values read, the new ones written, q, k, v read and the outputs written
    return {"bytes": 2 * g * hd * size * (keys + tokens) + 4 * hd * tokens * (h + 2 * g + h),
            "flops": 4 * hd * h * pairs}


# ---- inputs -----------------------------------------------------------------------------
def _table_of(case, ctx, room, gen):
    """A page table whose sequences hold ctx tokens on pages in no order: its state."""
    page, n = case["page"], case["seqs"]
    lens = torch.tensor(ctx, device="cuda", dtype=torch.int32)
    held = (lens + page - 1) // page
    need = sum(-(-(c + x) // page) for c, x in zip(ctx, room))
    n_pages = need + need // 8 + 3
    max_pages = max(-(-(c + x) // page) for c, x in zip(ctx, room)) + 1
    max_seqs = n + n // 4 + 1
    order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
    ids = torch.randperm(max_seqs, device="cuda", generator=gen)[:n].to(torch.int32)
    first = torch.cumsum(held, 0) - held
    col = torch.arange(max_pages, device="cuda")
    rows = order[(first[:, None] + col).clamp(max=n_pages - 1).long()]
    table = torch.full((max_seqs, max_pages), -1, device="cuda", dtype=torch.int32)
    table[ids.long()] = torch.where(col < held[:, None], rows, -1).to(torch.int32)
    seq_lens = torch.zeros(max_seqs, device="cuda", dtype=torch.int32)
    seq_lens[ids.long()] = lens
    used = sum(-(-c // page) for c in ctx)
    free = torch.cat([order[used:], order[:used]]).contiguous()
    return {"page": page, "table": table, "lens": seq_lens, "free": free, "ids": ids,
            "n_free": torch.tensor([n_pages - used], device="cuda", dtype=torch.int32),
            "n_pages": n_pages, "max_pages": max_pages, "max_seqs": max_seqs}


def _handle_of(t, tokens):
    """The framework's page table in the same state."""
    from unillm_amd import PageTable
    pt = PageTable(t["max_seqs"], t["max_pages"], t["n_pages"], t["page"], tokens)
    pt.block_table.copy_(t["table"])
    pt.seq_lens.copy_(t["lens"])
    pt.free_pages.copy_(t["free"])
    pt.n_free.copy_(t["n_free"])
    return pt


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ctx, new = _lengths(case)
    tokens = sum(new)
    t = _table_of(case, ctx, new, gen)
    state = {"case": case, "tokens": tokens, "t": t,
             "new": torch.tensor(new, device="cuda", dtype=torch.int32)}
    if case["op"] == "tables":
        back = [c - b for c, b in zip(ctx, _backs(case, ctx))]
        state["back"] = torch.tensor(back, device="cuda", dtype=torch.int32)
        if own:
            state["handle"] = _handle_of(t, tokens)
        return state
    g, hd, dtype = case["kv_heads"], case["hd"], DTYPES[case["dtype"]]
    shape = (t["n_pages"], g, t["page"], hd)
    # keys with a few strong channels, as projections have them
    strong = 1 + 3 * (torch.rand(g, 1, hd, device="cuda", generator=gen) > 0.95).to(dtype)
    state["k"] = torch.randn(shape, device="cuda", dtype=dtype, generator=gen) * strong
    state["v"] = torch.randn((t["n_pages"], g, hd, t["page"]), device="cuda", dtype=dtype, generator=gen)
    state["qkv"] = torch.randn(tokens, (case["heads"] + 2 * g) * hd, device="cuda", generator=gen)
    # the step's plan, which all layers share
    if own:
        from unillm_amd import PagedKvCache
        state["handle"] = _handle_of(t, tokens)
        state["handle"].extend(t["ids"], state["new"])
        state["cache"] = PagedKvCache(g, hd, t["n_pages"], t["page"], dtype, THETA,
                                      k=state["k"], v=state["v"])
    else:
        state["longest"] = max(c + n for c, n in zip(ctx, new))
        state["most"] = max(new)
        state["step"] = _extend(t, t["ids"].long(), state["new"], tokens)
    return state


# ---- the plain forms --------------------------------------------------------------------
def _pages(n, page):
    return torch.div(n + page - 1, page, rounding_mode="floor")


def _truncate(t, ids, lens):
    """Sequences `ids` keep their first `lens` tokens; the pages past them are free again."""
    col = torch.arange(t["max_pages"], device="cuda")
    rows = t["table"][ids]
    keep, held = _pages(lens, t["page"]), _pages(t["lens"][ids], t["page"])
    gone = (col >= keep[:, None]) & (col < held[:, None])
    freed = held - keep
    place = torch.cumsum(freed, 0) - freed  # entries and pages in order, undone from the end
    total = freed.sum()
    at = t["n_free"] + total - 1 - (place[:, None] + col - keep[:, None])
    stack = torch.cat([t["free"], t["free"][:1]])  # its last element takes what is kept
    at = torch.where(gone, at, t["n_pages"])
    stack[at.reshape(-1).long()] = rows.reshape(-1)
    t["free"].copy_(stack[:-1])
    t["n_free"] += total.to(torch.int32)
    t["table"][ids] = torch.where(gone, -1, rows).to(torch.int32)
    t["lens"][ids] = lens


def _extend(t, ids, new, tokens):
    """Room for `new` tokens of each sequence: the step's plan."""
    page = t["page"]
    lens = t["lens"][ids]
    held = _pages(lens, page)
    need = _pages(lens + new, page) - held
    place = torch.cumsum(need, 0) - need
    col = torch.arange(t["max_pages"], device="cuda")
    taken = (col >= held[:, None]) & (col < (held + need)[:, None])
    at = t["n_free"] - 1 - (place[:, None] + col - held[:, None])
    rows = torch.where(taken, t["free"][at.clamp(0, t["n_pages"] - 1).long()], t["table"][ids])
    t["table"][ids] = rows
    t["n_free"] -= need.sum().to(torch.int32)
    t["lens"][ids] = lens + new
    ends = torch.cumsum(new, 0).to(torch.int32)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends])
    token = torch.arange(tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(ends, token, right=True)
    pos = lens[seq] + token - cu[seq]
    slots = rows[seq, torch.div(pos, page, rounding_mode="floor").long()] * page + pos % page
    return {"cu": cu, "seq": seq, "positions": pos, "slots": slots, "rows": rows}


def _rotated(x, positions):
    """x [tokens, heads, hd] rotated at its tokens' positions, in f64: far angles lose f32."""
    half = x.shape[-1] // 2
    inv = THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = positions.double()[:, None, None] * inv
    c, s = torch.cos(angle), torch.sin(angle)
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * c - b * s, a * s + b * c], -1).float()


def _attend(state):
    case, t, step = state["case"], state["t"], state["step"]
    h, g, hd, page = case["heads"], case["kv_heads"], case["hd"], t["page"]
    kp, vp, seqs = state["k"], state["v"], case["seqs"]
    x = state["qkv"].view(state["tokens"], h + 2 * g, hd)
    pos, seq, slots = step["positions"], step["seq"], step["slots"].long()
    q, k, v = _rotated(x[:, :h], pos), _rotated(x[:, h:h + g], pos), x[:, h + g:]
    at, off = torch.div(slots, page, rounding_mode="floor"), slots % page
    kp[at, :, off] = k.to(kp.dtype)
    vp[at, :, :, off] = v.to(vp.dtype)
    # every sequence's keys and values, and its queries, padded to the longest
    width = -(-state["longest"] // page)
    pages = step["rows"][:, :width].clamp(min=0).long()
    keys = kp[pages].permute(0, 2, 4, 1, 3).reshape(seqs, g, hd, width * page).float()
    values = vp[pages].permute(0, 2, 1, 4, 3).reshape(seqs, g, width * page, hd).float()
    turn = torch.arange(state["tokens"], device="cuda") - step["cu"][seq]
    rows = torch.zeros(seqs, state["most"], h, hd, device="cuda")
    rows[seq, turn] = q * hd ** -0.5
    at_pos = torch.full((seqs, state["most"]), -1, device="cuda", dtype=pos.dtype)
    at_pos[seq, turn] = pos
    rows = rows.view(seqs, -1, g, h // g, hd).permute(0, 2, 3, 1, 4).reshape(seqs, g, -1, hd)
    scores = torch.matmul(rows, keys).view(seqs, g, h // g, -1, width * page)
    j = torch.arange(width * page, device="cuda")
    p = at_pos[:, :, None]
    seen = j <= p
    if case["window"]:
        seen &= (j > p - case["window"]) | (j < case["sinks"])
    scores = scores.masked_fill(~seen[:, None, None], -torch.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(seqs, g, -1, width * page), values)
    out = out.view(seqs, g, h // g, -1, hd) / total
    out = out.permute(0, 3, 1, 2, 4)[seq, turn]
    return out.reshape(state["tokens"], h * hd), kp, vp


def run(state):
    case, t, n = state["case"], state["t"], state["tokens"]
    if case["op"] == "tables":
        if own:
            pt = state["handle"]
            pt.truncate(t["ids"], state["back"])
            pt.extend(t["ids"], state["new"])
            return {"block_table": pt.block_table, "seq_lens": pt.seq_lens,
                    "free_pages": pt.free_pages, "n_free": pt.n_free,
                    "cu_tokens": pt.cu_tokens[:case["seqs"] + 1], "slots": pt.slots[:n],
                    "positions": pt.positions[:n]}
        ids = t["ids"].long()
        _truncate(t, ids, state["back"])
        step = _extend(t, ids, state["new"], n)
        return {"block_table": t["table"], "seq_lens": t["lens"], "free_pages": t["free"],
                "n_free": t["n_free"], "cu_tokens": step["cu"], "slots": step["slots"],
                "positions": step["positions"]}
    if own:
        out = state["cache"].attention(state["handle"], state["qkv"], case["heads"],
                                       window=case["window"], sinks=case["sinks"])
        k, v = state["cache"].k, state["cache"].v
    else:
        out, k, v = _attend(state)
    return {"out": out, "k": k, "v": v}


# ---- the definition in 64 bits ----------------------------------------------------------
def exact(case, seed):
    if case["op"] == "tables":
        return None
    state = prepare(case, seed)
    t, f64 = state["t"], torch.float64
    h, g, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    kp, vp = state["k"].to(f64), state["v"].to(f64)
    exact_k, exact_v = kp.clone(), vp.clone()
    out = torch.empty(state["tokens"], h, hd, device="cuda", dtype=f64)
    freq = [THETA ** (-2.0 * i / hd) for i in range(hd // 2)]
    ids, first = t["ids"].tolist(), 0
    for i, n in zip(ids, state["new"].tolist()):
        length = int(t["lens"][i])
        pages = t["table"][i, :-(-length // page)].long()
        x = state["qkv"][first:first + n].view(n, -1, hd).to(f64)
        at = torch.arange(length - n, length, device="cuda", dtype=f64)
        turn = torch.polar(torch.ones(n, hd // 2, device="cuda", dtype=f64),
                           at[:, None] * torch.tensor(freq, device="cuda", dtype=f64))[:, None]
        z = torch.complex(x[:, :h + g, :hd // 2], x[:, :h + g, hd // 2:]) * turn
        z = torch.cat([z.real, z.imag], -1)
        # the cache holds the new keys and values in its own type
        where = torch.arange(length - n, length, device="cuda")
        pg, off = pages[where // page], where % page
        for pool, true, new in ((kp, exact_k, z[:, h:].transpose(0, 1)),
                                (vp, exact_v, x[:, h + g:].transpose(0, 1))):
            held = new.float().to(state["k"].dtype).to(f64)
            for head in range(g):
                if pool is kp:
                    pool[pg, head, off], true[pg, head, off] = held[head], new[head]
                else:
                    pool[pg, head, :, off], true[pg, head, :, off] = held[head], new[head]
        few = max(1, min(n, (1 << 28) // length))
        for head in range(h):
            k = kp[pages, head // (h // g)].reshape(-1, hd)[:length]
            v = vp[pages, head // (h // g)].transpose(1, 2).reshape(-1, hd)[:length]
            for a in range(0, n, few):
                s = z[a:a + few, head] @ k.T / math.sqrt(hd)
                p = where[a:a + few, None]
                j = torch.arange(length, device="cuda")
                hidden = j > p
                if case["window"]:
                    hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
                s[hidden] = -math.inf
                out[first + a:first + a + few, head] = torch.softmax(s, -1) @ v
        first += n
    return {"out": out.view(-1, h * hd), "k": exact_k, "v": exact_v}
