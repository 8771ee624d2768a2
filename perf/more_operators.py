"""Operators of a server whose paged KV cache is held in 8 bits.

- ``rope``: rotary positions of q or k rows (``Rope.apply``): half-split or interleaved
  pairs, all of a head or its first ``rot`` dimensions, frequencies scaled for long contexts;
- ``write``: a step's new keys and values, rotated and quantised into the pages
  (``PagedKvCache8.append``), and what that changed read back (``PagedKvCache8.read``);
- ``read``: whole cached sequences read back, to be moved to another server;
- ``attention``: a step's tokens over the 8-bit pages (``PagedKvCache8.attention``), from one
  token a request to whole prompts; with ``append`` their keys and values are written first
  and what that changed is read back.

Head layouts are Llama-2-7B's (32 heads of 128), Mistral-7B's (32 over 8 of 128) and
TinyLlama-1.1B's (32 over 4 of 64), and one of 256 wide heads.  Lengths are ragged and come
from the case alone (``lengths`` seeds them); values come from the seed.

Definitions.  A pair (x, y) of a row at position p is turned by the angle p f_i, times the
magnitude: m (x cos - y sin), m (x sin + y cos), i the pair, rows rounded once to their type.
f_i = theta^(-2 i / rot), and
  linear:  f_i / factor;
  llama3:  with t = original f_i / 2 pi turns over the original context, r the ramp of t from
           low to high cut to [0, 1]: f_i (r + (1 - r) / factor);
  yarn:    the dimensions that make `high` and `low` turns, rot log(original / (2 pi t)) /
           (2 log theta), rounded down and up, cut to [0, rot - 1]: r falls from 1 at the
           first to 0 at the second, m = 0.1 log(factor) + 1.

A page holds ``page`` positions of one layer: K codes [pages, kv heads, page, hd], V codes
[pages, kv heads, hd, page], and for each 16 positions and kv head an exponent e (held as e +
127 in a byte): a code c stands for c 2^e.  Codes are int8 (up to 127) or e4m3 (up to 448).
Writing new positions of such a block (keys rotated first, an f32 row): e is the least, at least
-126, with which the new values' largest magnitude fits, and no less than the block's own if it holds
positions before them (whose codes are rounded anew when it grows); new values are rounded to
nearest even.  A token at position p sees the keys j <= p with j > p - window (window > 0) or j < sinks;
softmax(q k^T / sqrt(hd)) v is f32.
"""
from __future__ import annotations

import math
import random

import torch

own = False

THETA = 10000.0
BLOCK = 16
TOP = {"int8": 127.0, "e4m3": 448.0}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
FLOATS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ITEM = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases --------------------------------------------------------------------------
def _rope(name, dtype, n, heads, hd, rot, layout, scaling, far, pad=0):
    return {"name": name, "op": "rope", "dtype": dtype, "n": n, "heads": heads, "hd": hd, "rot": rot,
            "layout": layout, "scaling": scaling, "far": far, "pad": pad}


def _cache(name, op, kind, heads, hd, page, seqs, ctx, new, chunks, append=True, out="bf16",
           window=0, sinks=0, rot=0, layout="half", lengths=1):
    return {"name": name, "op": op, "kind": kind, "heads": heads[0], "kv_heads": heads[1], "hd": hd,
            "page": page, "seqs": seqs, "ctx_min": ctx[0], "ctx_max": ctx[1], "new_min": new[0],
            "new_max": new[1], "chunks": chunks, "append": append, "out": out, "window": window,
            "sinks": sinks, "rot": rot or hd, "layout": layout, "lengths": lengths}


def listed():
    return [
        # one chat request's next token: q and k of a layer (Llama-2-7B's heads)
        _rope("rope_1_bf16", "bf16", 1, 64, 128, 128, "half", "none", 4000),
        # a chunk's queries inside the fused projections, part of each head, a stretched context
        _rope("rope_777_f16_part", "f16", 777, 32, 128, 64, "interleaved", "yarn", 60000, 2048),
        # a long prompt's queries (Llama-2-7B's heads)
        _rope("rope_20001_f32", "f32", 20001, 32, 128, 128, "half", "llama3", 120000),
        # a continuous batch's decode step (Mistral-7B's heads)
        _cache("write_96_int8", "write", "int8", (32, 8), 128, 16, 96, (1, 9000), (1, 1), 0, lengths=3),
        # a new prompt behind a cached prefix (Llama-2-7B's heads)
        _cache("write_4000_e4m3", "write", "e4m3", (32, 32), 128, 64, 1, (333, 333), (4000, 4000), 1),
        # two requests handed to another server
        _cache("read_2_int8", "read", "int8", (32, 8), 128, 128, 2, (30001, 60000), (1, 1), 0, out="f16", lengths=4),
        # one chat request's next token (Llama-2-7B's heads)
        _cache("decode_1_int8", "attention", "int8", (32, 32), 128, 16, 1, (1500, 1500), (1, 1), 0, append=False),
        # a continuous batch's decode step, ragged (Mistral-7B's heads)
        _cache("decode_80_e4m3", "attention", "e4m3", (32, 8), 128, 32, 80, (200, 9000), (1, 1), 0, append=False,
               layout="interleaved", lengths=5),
        # three requests over whole books
        _cache("decode_long_int8", "attention", "int8", (32, 8), 128, 128, 3, (70001, 100000), (1, 1), 0,
               append=False, lengths=6),
        # drafted tokens verified (TinyLlama's heads)
        _cache("verify_12_e4m3", "attention", "e4m3", (32, 4), 64, 32, 12, (100, 3500), (2, 6), 12, lengths=7),
        # a new prompt (Mistral-7B's heads)
        _cache("prompt_3001_int8", "attention", "int8", (32, 8), 128, 16, 1, (0, 0), (3001, 3001), 1),
        # prompt chunks among decoding requests, wide heads, a sliding window with attention sinks
        _cache("mixed_20_e4m3", "attention", "e4m3", (16, 2), 256, 64, 20, (1, 7001), (201, 400), 4,
               window=4096, sinks=4, rot=64, lengths=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.2:
        while True:
            n, heads, hd = _log(rng, 1, 40000), _log(rng, 1, 64), rng.choice((64, 80, 96, 128, 128, 256))
            rot = hd if rng.random() < 0.5 else 2 * rng.randint(1, hd // 2)
            case = {"op": "rope", "dtype": rng.choice(("f32", "f16", "bf16")), "n": n, "heads": heads, "hd": hd,
                    "rot": rot, "layout": rng.choice(("half", "interleaved")),
                    "scaling": rng.choice(("none", "linear", "llama3", "yarn")), "far": _log(rng, n, 1 << 20),
                    "pad": rng.choice((0, 0, 1, 64, 1000))}
            if work(case)["bytes"] <= 650_000_000:
                return case
    op = rng.choice(("write", "write", "read", "attention", "attention", "attention", "attention", "attention"))
    while True:
        hd = rng.choice((64, 128, 128, 256))
        kv_heads = _log(rng, 1, 32)
        heads = kv_heads * rng.choice((1, 1, 2, 4, 7, 8, 16))
        if heads > 64:
            continue
        seqs = _log(rng, 1, 128)
        ctx_max = _log(rng, 1, 100000)
        chunked = rng.random() < 0.5
        new_max = _log(rng, 2, 4096) if chunked else 1
        case = {"op": op, "kind": rng.choice(("int8", "e4m3")), "heads": heads, "kv_heads": kv_heads, "hd": hd,
                "page": rng.choice((16, 32, 64, 128, 256)), "seqs": seqs, "ctx_min": rng.randrange(ctx_max + 1),
                "ctx_max": ctx_max, "new_min": rng.randint((new_max + 1) // 2, new_max), "new_max": new_max,
                "chunks": rng.randint(1, seqs) if chunked else 0, "append": op == "write" or rng.random() < 0.5,
                "out": rng.choice(("f32", "f16", "bf16")) if op == "read" else "bf16",
                "window": _log(rng, 1, 8192) if op == "attention" and rng.random() < 0.4 else 0, "sinks": 0,
                "rot": hd if rng.random() < 0.6 else 8 * rng.randint(1, hd // 8),
                "layout": rng.choice(("half", "interleaved")), "lengths": rng.randrange(1 << 20)}
        if case["window"]:
            case["sinks"] = rng.choice((0, 1, 4, 4, 37))
        # within the largest listed cases' costs, padded as the plain form pads them
        longest = ctx_max + new_max
        w = work(case)
        if (seqs * longest * kv_heads * hd <= 1_000_000_000 and w["bytes"] <= 600_000_000 and w["flops"] <= 70e9
                and (op != "attention" or seqs * heads * new_max * longest <= 500_000_000)):
            return case


def _lengths(case):
    """(cached, new) tokens of each sequence, from the case alone."""
    r = random.Random(case["lengths"])
    n = case["seqs"]
    lo, hi = math.log(case["ctx_min"] + 1), math.log(case["ctx_max"] + 1)
    ctx = [min(case["ctx_max"], int(math.exp(r.uniform(lo, hi)) - 0.5)) for _ in range(n)]
    ctx[r.randrange(n)] = case["ctx_max"]
    chunked = set(r.sample(range(n), case["chunks"]))
    return ctx, [r.randint(case["new_min"], case["new_max"]) if i in chunked else 1 for i in range(n)]


def _back(case, ctx, new):
    """Positions that are read back: (first, count) of each sequence."""
    if case["op"] == "read":
        return [(0, c + n) for c, n in zip(ctx, new)]
    return [(c // BLOCK * BLOCK, c % BLOCK + n) for c, n in zip(ctx, new)]


def work(case):
    if case["op"] == "rope":
        size = ITEM[case["dtype"]]
        return {"bytes": case["n"] * (2 * case["heads"] * case["hd"] * size + 4),
                "flops": 3 * case["n"] * case["heads"] * case["rot"]}
    ctx, new = _lengths(case)
    h, g, hd = case["heads"], case["kv_heads"], case["hd"]
    tokens, each = sum(new), 2 * g * hd + 2 * g / BLOCK  # of a position: K and V codes and exponents
    back = sum(n for _, n in _back(case, ctx, new))
    bytes_, flops = 0, 0
    if case["append"] and case["op"] != "read":
        bytes_ += tokens * (2 * g * hd * 4 + each)
        flops += 3 * tokens * g * case["rot"]
    if case["append"] or case["op"] == "read":
        bytes_ += back * (each + 2 * g * hd * ITEM[case["out"]])
    if case["op"] == "attention":
        w, sinks = case["window"], case["sinks"]
        for c, n in zip(ctx, new):
            low = max(0, c + 1 - w) if w else 0
            bytes_ += each * (c + n - low + min(sinks, low))
            if not w:
                pairs = n * c + n * (n + 1) // 2
            else:
                pairs = sum(p + 1 if p < w else w + min(sinks, p + 1 - w) for p in range(c, c + n))
            flops += 4 * hd * h * pairs
        bytes_ += 2 * tokens * h * hd * 4
    return {"bytes": bytes_, "flops": flops}


# ---- inputs -----------------------------------------------------------------------------
SCALED = {"none": {}, "linear": {"factor": 4.0},
          "llama3": {"factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
          "yarn": {"factor": 16.0, "low": 1.0, "high": 32.0, "original": 4096}}


def _rope_handle(hd, rot, layout, scaling="none"):
    from unillm_amd import Rope
    return Rope(hd, rotary_dim=rot, theta=THETA, interleaved=layout == "interleaved",
                scaling=None if scaling == "none" else scaling, **SCALED[scaling])


def _prepare_rope(case, gen):
    n, heads, hd = case["n"], case["heads"], case["hd"]
    rows = torch.randn(n, heads * hd + case["pad"], device="cuda", generator=gen).to(FLOATS[case["dtype"]])
    state = {"case": case, "x": rows[:, :heads * hd].unflatten(1, (heads, hd)),
             "positions": torch.randint(case["far"], (n,), device="cuda", generator=gen, dtype=torch.int32)}
    if own:
        state["rope"] = _rope_handle(hd, case["rot"], case["layout"], case["scaling"])
    return state


def _exponent(top, kind):
    """The least e >= -126 with top <= TOP 2^e, of magnitudes `top`."""
    m, x = torch.frexp(top)
    room = TOP[kind] / 2.0 ** math.ceil(math.log2(TOP[kind]))  # TOP = room 2^ceil
    e = x - math.ceil(math.log2(TOP[kind])) + (m > room).to(x.dtype)
    return torch.where(top > 0, e, -126).clamp(min=-126)


def _codes(scaled, kind):
    return scaled.round().to(torch.int8) if kind == "int8" else scaled.to(torch.float8_e4m3fn)


def _pow2(e):
    """2^e of whole numbers e in [-126, 127], exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _filled(shape, across, kind, gen):
    """Codes of a pool and its exponents, the values a few strong channels along the dimensions."""
    pages, g = shape[:2]
    keys = 2 if across == 3 else 3  # the dimension of positions; `across` that of channels
    wide = [1, g, 1, 1]
    wide[across] = shape[across]
    strong = 1 + 3 * (torch.rand(wide, device="cuda", generator=gen) > 0.95).float()
    x = torch.randn(shape, device="cuda", generator=gen) * strong
    blocks = x.unflatten(keys, (shape[keys] // BLOCK, BLOCK))
    e = _exponent(blocks.abs().amax((keys + 1, 4 if keys == 2 else 2)), kind)
    per = e[:, :, :, None, None] if keys == 2 else e[:, :, None, :, None]
    codes = _codes(blocks * _pow2(-per), kind).reshape(shape)
    return codes, (e + 127).to(torch.uint8).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "rope":
        return _prepare_rope(case, gen)
    ctx, new = _lengths(case)
    page, n, g, hd, kind = case["page"], case["seqs"], case["kv_heads"], case["hd"], case["kind"]
    up = lambda x: -(-x // page)  # noqa: E731
    total = [c + x for c, x in zip(ctx, new)]
    n_pages = sum(map(up, total)) + 5
    max_pages = max(map(up, total)) + 1
    max_seqs = n + n // 4 + 1
    tokens = sum(new)
    whole = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)  # noqa: E731
    # pages in no order: each sequence's, one after the other, off the end of this list
    order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
    ids = torch.randperm(max_seqs, device="cuda", generator=gen)[:n].to(torch.int32)
    lens, news = whole(ctx), whole(new)
    held = whole([up(t) for t in total])
    col = torch.arange(max_pages, device="cuda")
    at = (torch.cumsum(held, 0) - held)[:, None] + col
    rows = torch.where(col < held[:, None], order[at.clamp(max=n_pages - 1).long()], -1).to(torch.int32)
    back = _back(case, ctx, new)
    counts = [x for _, x in back]
    state = {"case": case, "tokens": tokens, "ids": ids, "rows": rows, "lens": whole(total), "page": page,
             "longest": max(total), "most": max(new), "n_back": sum(counts),
             "blocks": sum((c + x - 1) // BLOCK - c // BLOCK + 1 for c, x in zip(ctx, new)),
             "starts": whole([s for s, _ in back]),
             "cu_back": whole([sum(counts[:i]) for i in range(n + 1)])}
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), news.long(), output_size=tokens)
    first = torch.cumsum(news, 0) - news
    state["seq"], state["turn"] = seq, torch.arange(tokens, device="cuda") - first[seq]
    state["positions"] = lens[seq] + state["turn"].to(torch.int32)
    state["k"], state["k_exp"] = _filled((n_pages, g, page, hd), 3, kind, gen)
    state["v"], state["v_exp"] = _filled((n_pages, g, hd, page), 2, kind, gen)
    width = (case["heads"] if case["op"] == "attention" else 0) + (2 * g if case["append"] else 0)
    state["x"] = torch.randn(tokens, width * hd, device="cuda", generator=gen)
    if own:
        from unillm_amd import PagedKvCache8, PageTable
        pt = PageTable(max_seqs, max_pages, n_pages, page, tokens)
        had = whole([up(c) for c in ctx])
        pt.block_table[ids.long()] = torch.where(col < had[:, None], rows, -1).to(torch.int32)
        pt.seq_lens[ids.long()] = lens
        # the step takes each sequence's further pages, in order, from the top of the free stack
        extra = rows[(col >= had[:, None]) & (col < held[:, None])]
        spare = order[int(held.sum()):]
        stack = torch.cat([spare, extra.flip(0)])
        pt.free_pages[:stack.numel()] = stack
        pt.n_free.fill_(stack.numel())
        pt.extend(ids, news)
        state["table"] = pt
        state["cache"] = PagedKvCache8(g, hd, n_pages, page, CODES[kind], _rope_handle(hd, case["rot"], case["layout"]),
                                       k=state["k"], v=state["v"], k_exp=state["k_exp"], v_exp=state["v_exp"])
    return state


# ---- the plain forms --------------------------------------------------------------------
def _frequencies(rot, scaling):
    """(radians a position of each pair, magnitude)"""
    s = SCALED[scaling]
    f = THETA ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    if scaling == "linear":
        return f / s["factor"], 1.0
    if scaling == "llama3":
        r = ((s["original"] * f / (2 * math.pi) - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        return f * (r + (1 - r) / s["factor"]), 1.0
    if scaling == "yarn":
        dim = lambda t: rot * math.log(s["original"] / (2 * math.pi * t)) / (2 * math.log(THETA))  # noqa: E731
        a, b = max(0, math.floor(dim(s["high"]))), min(rot - 1, math.ceil(dim(s["low"])))
        i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
        r = 1 - ((i - a) / max(b - a, 0.001)).clamp(0, 1)
        return f * (r + (1 - r) / s["factor"]), 0.1 * math.log(s["factor"]) + 1
    return f, 1.0


def _rotated(x, positions, rot, layout, scaling="none"):
    """x [n, heads, hd] rotated at its rows' positions, in f64: far angles lose f32."""
    f, m = _frequencies(rot, scaling)
    angle = positions.double()[:, None, None] * f
    c, s = m * torch.cos(angle), m * torch.sin(angle)
    y, rest = x[..., :rot].double(), x[..., rot:]
    if layout == "half":
        a, b = y.chunk(2, -1)
        y = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([y.to(x.dtype), rest], -1)


def _slots(state, seq, positions):
    page = state["page"]
    at = state["rows"][seq, torch.div(positions, page, rounding_mode="floor").long()]
    return at.long(), (positions % page).long()


def _write(state, k, v):
    """The step's keys and values [tokens, kv heads, hd] into their blocks of 16 positions."""
    kind, n, u = state["case"]["kind"], state["blocks"], torch.uint8
    at, off = _slots(state, state["seq"], state["positions"])
    block = at * (state["page"] // BLOCK) + off // BLOCK
    begins = torch.cat([torch.ones_like(block[:1]), (block[1:] != block[:-1]).to(block.dtype)])
    which, place = torch.cumsum(begins, 0) - 1, off % BLOCK
    pg, part, from_ = (torch.zeros(n, device="cuda", dtype=torch.int64) for _ in range(3))
    pg[which], part[which] = at, off // BLOCK
    from_[which[begins == 1]] = place[begins == 1]
    fresh = torch.zeros(n, BLOCK, device="cuda", dtype=torch.bool)
    fresh[which, place] = True
    old = torch.arange(BLOCK, device="cuda") < from_[:, None]
    for pool, exps, x, keys in ((state["k"], state["k_exp"], k, 2), (state["v"], state["v_exp"], v, 3)):
        x16 = torch.zeros(n, BLOCK, *x.shape[1:], device="cuda")
        x16[which, place] = x
        e = _exponent(x16.abs().amax((1, 3)), kind)
        had = exps[pg, :, part].to(torch.int32) - 127
        e = torch.where(from_[:, None] > 0, torch.maximum(e, had), e)
        split = pool.view(u).unflatten(keys, (-1, BLOCK))  # (bytes: what 8-bit floats are taken and put by)
        codes = split[pg, :, part] if keys == 2 else split[pg, :, :, part]  # [n, g, 16, hd] or [n, g, hd, 16]
        codes = codes.transpose(1, 2) if keys == 2 else codes.permute(0, 3, 1, 2)
        held = codes.contiguous().view(CODES[kind]).float()
        again = _codes(held * _pow2((had - e).clamp(-126, 0))[:, None, :, None], kind)
        put = _codes(x16 * _pow2(-e)[:, None, :, None], kind)
        got = torch.where(fresh[:, :, None, None], put.view(u),
                          torch.where(old[:, :, None, None], again.view(u), codes))
        if keys == 2:
            split[pg, :, part] = got.transpose(1, 2)
        else:
            split[pg, :, :, part] = got.permute(0, 2, 3, 1)
        exps[pg, :, part] = (e + 127).to(u)


def _values(state, pages):
    """(k, v) [..., kv heads, positions, hd] f32 that the codes of whole pages stand for."""
    codes = lambda pool: pool.view(torch.uint8)[pages].view(pool.dtype).float()  # noqa: E731
    k = codes(state["k"]).unflatten(-2, (-1, BLOCK))
    k = (k * _pow2(state["k_exp"][pages].int() - 127)[..., None, None]).flatten(-3, -2)
    v = codes(state["v"]).unflatten(-1, (-1, BLOCK))
    v = (v * _pow2(state["v_exp"][pages].int() - 127)[..., None, :, None]).flatten(-2)
    return k, v.transpose(-1, -2)


def _read(state):
    cu, n = state["cu_back"], state["n_back"]
    row = torch.arange(n, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(cu[1:], row, right=True)
    at, off = _slots(state, seq, state["starts"][seq] + row - cu[seq])
    dtype, part = FLOATS[state["case"]["out"]], torch.div(off, BLOCK, rounding_mode="floor")
    k = state["k"].view(torch.uint8)[at, :, off].view(state["k"].dtype).float()
    v = state["v"].view(torch.uint8)[at, :, :, off].view(state["v"].dtype).float()
    ke, ve = (_pow2(state[x][at, :, part].int() - 127)[..., None] for x in ("k_exp", "v_exp"))
    return (k * ke).to(dtype), (v * ve).to(dtype)


def _attend(state, q):
    case, seqs = state["case"], state["case"]["seqs"]
    h, g, hd, page = case["heads"], case["kv_heads"], case["hd"], state["page"]
    width = -(-state["longest"] // page)
    keys, values = _values(state, state["rows"][:, :width].clamp(min=0).long())  # [seqs, pages, g, page, hd]
    keys = keys.permute(0, 2, 4, 1, 3).reshape(seqs, g, hd, width * page)
    values = values.permute(0, 2, 1, 3, 4).reshape(seqs, g, width * page, hd)
    # every sequence's queries, padded to the most
    rows = torch.zeros(seqs, state["most"], h, hd, device="cuda")
    rows[state["seq"], state["turn"]] = q * hd ** -0.5
    p = torch.full((seqs, state["most"]), -1, device="cuda", dtype=torch.int32)
    p[state["seq"], state["turn"]] = state["positions"]
    rows = rows.view(seqs, -1, g, h // g, hd).permute(0, 2, 3, 1, 4).reshape(seqs, g, -1, hd)
    scores = torch.matmul(rows, keys).view(seqs, g, h // g, -1, width * page)
    j, p = torch.arange(width * page, device="cuda"), p[:, :, None]
    seen = j <= p
    if case["window"]:
        seen &= (j > p - case["window"]) | (j < case["sinks"])
    scores = scores.masked_fill(~seen[:, None, None], -torch.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(seqs, g, -1, width * page), values)
    out = out.view(seqs, g, h // g, -1, hd) / total
    return out.permute(0, 3, 1, 2, 4)[state["seq"], state["turn"]].reshape(state["tokens"], h * hd)


def _run_own(state):
    case, op = state["case"], state["case"]["op"]
    if op == "rope":
        return {"out": state["rope"].apply(state["x"], state["positions"])}
    cache, table, got = state["cache"], state["table"], {}
    if op == "write":
        cache.append(table, state["x"])
    if op == "attention":
        got["out"] = cache.attention(table, state["x"], case["heads"], window=case["window"], sinks=case["sinks"])
    if op != "attention" or case["append"]:
        got["k"], got["v"] = cache.read(table, state["ids"], state["starts"], state["cu_back"], state["n_back"],
                                        dtype=FLOATS[case["out"]])
    return got


def run(state):
    if own:
        return _run_own(state)
    case, op = state["case"], state["case"]["op"]
    if op == "rope":
        return {"out": _rotated(state["x"], state["positions"], case["rot"], case["layout"], case["scaling"])}
    g, hd, got = case["kv_heads"], case["hd"], {}
    x = state["x"].unflatten(1, (-1, hd))
    turned = lambda y: _rotated(y, state["positions"], case["rot"], case["layout"])  # noqa: E731
    if case["append"] and op != "read":
        _write(state, turned(x[:, -2 * g:-g]), x[:, -g:])
    if op == "attention":
        got["out"] = _attend(state, turned(x[:, :case["heads"]]))
    if op != "attention" or case["append"]:
        got["k"], got["v"] = _read(state)
    return got


# ---- the definition in 64 bits ----------------------------------------------------------
def _turns(rot, scaling):
    """Each pair's angle a position and its magnitude, by the definition, as plain numbers."""
    s, got = SCALED[scaling], []
    for i in range(rot // 2):
        f = THETA ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= s["factor"]
        if scaling == "llama3":
            turns = s["original"] * f / (2 * math.pi)
            part = min(1.0, max(0.0, (turns - s["low"]) / (s["high"] - s["low"])))
            f = part * f + (1 - part) * f / s["factor"]
        if scaling == "yarn":
            ends = [rot * math.log(s["original"] / (2 * math.pi * t)) / (2 * math.log(THETA))
                    for t in (s["high"], s["low"])]
            a, b = max(0, math.floor(ends[0])), min(rot - 1, math.ceil(ends[1]))
            part = min(1.0, max(0.0, (i - a) / max(b - a, 0.001)))
            f = (1 - part) * f + part * f / s["factor"]
        got.append(f)
    return got, 0.1 * math.log(s["factor"]) + 1 if scaling == "yarn" else 1.0


def _turned(x, positions, rot, layout, scaling="none"):
    f, m = _turns(rot, scaling)
    f64, half = torch.float64, rot // 2
    angle = positions.to(f64)[:, None] * torch.tensor(f, device="cuda", dtype=f64)
    turn = torch.polar(torch.full_like(angle, m), angle)[:, None]
    y = x.to(f64).clone()
    if layout == "half":
        z = torch.complex(y[..., :half], y[..., half:rot]) * turn
        y[..., :half], y[..., half:rot] = z.real, z.imag
    else:
        z = torch.complex(y[..., 0:rot:2], y[..., 1:rot:2]) * turn
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


def _held(values, least, kind):
    """(values of a block [16 or fewer, hd] as 8 bits hold them with one exponent, it)"""
    top, e = float(values.abs().max()), -126
    if top > 0:
        e = max(e, math.ceil(math.log2(top / TOP[kind])) - 1)
        while top > TOP[kind] * 2.0 ** e:
            e += 1
    e = max(e, least)
    return _rounded(values, e, kind), e


def _rounded(values, e, kind):
    y = values * 2.0 ** -e
    if kind == "int8":
        return y.round() * 2.0 ** e
    # e4m3: 4 significant bits, down to multiples of 2^-9
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6) - 3)
    return (y / step).round() * step * 2.0 ** e


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rope":
        return {"out": _turned(state["x"], state["positions"], case["rot"], case["layout"], case["scaling"])}
    ctx, new = _lengths(case)
    kind, g, hd, h, page = case["kind"], case["kv_heads"], case["hd"], case["heads"], case["page"]
    f64, blocks = torch.float64, state["blocks"] * g
    if case["append"] and blocks > 25000:  # (a block and head at a time)
        return None
    out, ks, vs, first = [], [], [], 0
    for i, (c, n, (start, count)) in enumerate(zip(ctx, new, _back(case, ctx, new))):
        pages = state["rows"][i, :-(-(c + n) // page)].long()
        k, v = (y.transpose(0, 1).reshape(g, -1, hd)[:, :c + n].to(f64) for y in _values(state, pages))
        at = torch.arange(c, c + n, device="cuda")
        x = state["x"][first:first + n].unflatten(1, (-1, hd)).to(f64)
        if case["append"] and case["op"] != "read":
            new_k = _turned(x[:, -2 * g:-g], at, case["rot"], case["layout"]).float().to(f64)  # (rows' own rounding)
            for held, fresh, exps in ((k, new_k, state["k_exp"]), (v, x[:, -g:], state["v_exp"])):
                for b in range(c // BLOCK, (c + n - 1) // BLOCK + 1):
                    a, z = max(c, b * BLOCK), min(c + n, (b + 1) * BLOCK)
                    had = exps[pages[b * BLOCK // page], :, b * BLOCK % page // BLOCK].tolist()
                    for head in range(g):
                        least = had[head] - 127 if a % BLOCK else -126
                        held[head, a:z], e = _held(fresh[a - c:z - c, head], least, kind)
                        if e > least and a % BLOCK:
                            held[head, b * BLOCK:a] = _rounded(held[head, b * BLOCK:a], e, kind)
        ks.append(k[:, start:start + count].transpose(0, 1))
        vs.append(v[:, start:start + count].transpose(0, 1))
        if case["op"] == "attention":
            q = _turned(x[:, :h], at, case["rot"], case["layout"])
            o = torch.empty(n, h, hd, device="cuda", dtype=f64)
            few = max(1, min(n, (1 << 28) // (c + n)))
            j = torch.arange(c + n, device="cuda")
            for head in range(h):
                for a in range(0, n, few):
                    s = q[a:a + few, head] @ k[head // (h // g)].T / math.sqrt(hd)
                    p = at[a:a + few, None]
                    hidden = j > p
                    if case["window"]:
                        hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
                    s[hidden] = -math.inf
                    o[a:a + few, head] = torch.softmax(s, -1) @ v[head // (h // g)]
            out.append(o.view(n, h * hd))
        first += n
    got = {"out": torch.cat(out)} if out else {}
    if case["op"] != "attention" or case["append"]:
        got["k"], got["v"] = torch.cat(ks), torch.cat(vs)
    return got
