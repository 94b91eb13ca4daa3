"""Cases of the paged-cache and beam-search operators, each with its plain form in torch.

Five operators that a batched decoding program calls together: attention of one new token over a
paged cache (`paged_decode`), of a chunk of new tokens (`paged_prefill`), the write of new keys and
values into the pages (`paged_append`), the bookkeeping of pages (`page_update`, `page_compact`,
`page_copy`) and the selection of beams (`beam_select`, `beam_reorder`).

`run` computes a case in elementary torch operations, or, where `own` is true, with the calls that a
user makes of the library.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # The smallest decode step: one sequence of a Llama-shaped layer, pages of 16, latency counts.
        dict(name="decode_one_sequence", op="decode", batch=1, heads=32, kv_heads=8, dim=128,
             page=16, longest=1001, ragged=False, window=0, sinks=0),
        # A serving batch at mixed lengths, some of its slots empty.
        dict(name="decode_ragged_batch", op="decode", batch=64, heads=32, kv_heads=8, dim=128,
             page=32, longest=8192, ragged=True, window=0, sinks=0),
        # Long chats behind a sliding window with sinks, six query heads to a key head, head size 64.
        dict(name="decode_window_d64", op="decode", batch=48, heads=24, kv_heads=4, dim=64,
             page=64, longest=32768, ragged=True, window=4096, sinks=4),
        # Short pieces of prompts behind cached prefixes of several sequences.
        dict(name="prefill_ragged_chunk", op="prefill", batch=4, heads=32, kv_heads=8, dim=128,
             page=16, chunk=40, prefix=500, ragged=True, window=0, sinks=0),
        # One whole prompt.
        dict(name="prefill_prompt", op="prefill", batch=1, heads=32, kv_heads=8, dim=128,
             page=64, chunk=4096, prefix=0, ragged=False, window=0, sinks=0),
        # Long pieces behind a sliding window, odd lengths, head size 64.
        dict(name="prefill_window_d64", op="prefill", batch=2, heads=16, kv_heads=4, dim=64,
             page=32, chunk=2999, prefix=2500, ragged=True, window=1024, sinks=8),
        # One decode step's new key and value of each sequence.
        dict(name="append_step", op="append", batch=64, kv_heads=8, dim=128, page=32, chunk=1,
             prefix=4096, ragged=False),
        # The keys and values of ragged prompts.
        dict(name="append_prompts", op="append", batch=8, kv_heads=8, dim=128, page=16, chunk=2047,
             prefix=100, ragged=True),
        # One reordering step of beam search: 32 prompts with 8 beams each, copy on write over 8 layers.
        dict(name="pages_beam_step", op="update", groups=32, beams=8, longest=1500, page=16,
             pages=12000, slabs=16, row=512),
        # Defragmentation of a half-filled pool of 8 layers.
        dict(name="pages_compact", op="compact", rows=64, longest=2048, page=64, pages=4099,
             slabs=16, row=512, live=0.5),
        # Beam search over one sequence at a small vocabulary.
        dict(name="beam_one_prompt", op="beam", batch=1, beams=4, width=4, vocab=32000,
             f32=False, done=False, tokens=512),
        # A batch of beams at a large vocabulary, some of them finished.
        dict(name="beam_batch", op="beam", batch=64, beams=8, width=8, vocab=128256,
             f32=False, done=True, tokens=2048),
    ]


def _spread(rng, low, high):
    """A whole number, spread evenly over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prefill", "prefill", "append", "update", "compact", "beam"])
    if op in ("decode", "prefill"):
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
        dim = rng.choice([64, 128])
        page = rng.choice([8, 16, 24, 32, 64, 128])
        window = rng.choice([0, _spread(rng, 1, 4096)])
        case = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=page, ragged=rng.random() < 0.7,
                    window=window, sinks=rng.choice([0, 1, 4, 37]) if window else 0)
        if op == "decode":
            batch = _spread(rng, 1, 128)
            most = max(64, min(131072, (64 * 8192 * 8 * 128) // (batch * kv_heads * dim)))
            return dict(case, batch=batch, longest=_spread(rng, 1, most))
        batch = _spread(rng, 1, 8)
        pairs = 4096 * 2048 * 32 * 128 // (batch * heads * dim)  # of queries and keys a head
        chunk = _spread(rng, 1, min(4096 // batch, math.isqrt(pairs)))
        most = max(1, min(16384, pairs // chunk - chunk // 2 - 1))
        return dict(case, batch=batch, chunk=chunk, prefix=_spread(rng, 1, most) - 1)
    if op == "append":
        batch = _spread(rng, 1, 128)
        return dict(op=op, batch=batch, kv_heads=rng.choice([1, 2, 5, 8]), dim=rng.choice([64, 128]),
                    page=rng.choice([8, 16, 24, 32, 64, 128]), chunk=_spread(rng, 1, 16384 // batch),
                    prefix=_spread(rng, 1, 4096) - 1, ragged=rng.random() < 0.5)
    if op == "update":
        groups, beams = _spread(rng, 1, 32), rng.choice([1, 2, 3, 4, 8])
        longest, page = _spread(rng, 1, 1500), rng.choice([8, 16, 24, 32, 64])
        pages = groups * (beams + 1) * (2 + longest // page) + rng.randrange(1, 2000)
        return dict(op=op, groups=groups, beams=beams, longest=longest, page=page,
                    pages=min(pages, 12000), slabs=rng.choice([2, 6, 16]), row=rng.choice([256, 512]))
    if op == "compact":
        return dict(op=op, rows=_spread(rng, 1, 64), longest=_spread(rng, 1, 2048),
                    page=rng.choice([16, 24, 32, 64]), pages=_spread(rng, 40, 4099),
                    slabs=rng.choice([2, 4, 16]), row=rng.choice([128, 256, 512]), live=rng.uniform(0.1, 0.95))
    beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
    return dict(op=op, batch=_spread(rng, 1, 512 // beams), beams=beams,
                width=max(1, min(32, beams * rng.choice([1, 1, 2]))), vocab=_spread(rng, 50, 128256),
                f32=rng.random() < 0.4, done=rng.random() < 0.5, tokens=_spread(rng, 1, 2048))


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _normal(gen, *shape, dtype=torch.float16):
    return torch.randn(shape, dtype=dtype, device=DEV, generator=gen)


def _scattered_table(rs, lengths, page, pool=0):
    """Pages of a pool in no order, one row a sequence; (table, pages of the pool)."""
    need = (lengths + page - 1) // page
    entries = max(1, int(need.max()))
    pool = max(pool, int(need.sum()) + 7)
    free = rs.permutation(pool)
    table = np.full((len(lengths), entries), -1)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = free[at:at + n]
        at += n
    return table, pool


def _prepare_attention(c, rs, gen):
    batch, chunk = c["batch"], c.get("chunk", 1)
    if c["op"] == "decode":
        lengths = np.full(batch, c["longest"])
        if c["ragged"]:  # lengths between nothing and the longest, every eighth slot empty
            lengths = rs.randint(1, c["longest"] + 1, batch)
            lengths[0] = c["longest"]
            lengths[7::8] = 0
        news = np.ones(batch, dtype=np.int64)
    else:
        news = np.full(batch, chunk)
        prefix = np.full(batch, c["prefix"])
        if c["ragged"]:
            news = rs.randint(1, chunk + 1, batch)
            news[0] = chunk
            prefix = rs.randint(0, c["prefix"] + 1, batch)
            prefix[0] = c["prefix"]
        lengths = prefix + news
    table, pool = _scattered_table(rs, lengths, c["page"])
    shape = (pool, c["kv_heads"], c["page"], c["dim"])
    q = (batch, c["heads"], c["dim"]) if c["op"] == "decode" else (batch, c["heads"], chunk, c["dim"])
    return dict(case=c, q=_normal(gen, *q), k=_normal(gen, *shape), v=_normal(gen, *shape),
                table=_ints(table), lens=_ints(lengths), news=_ints(news))


def _prepare_append(c, rs, gen):
    news = np.full(c["batch"], c["chunk"])
    starts = np.full(c["batch"], c["prefix"])
    if c["ragged"]:
        news = rs.randint(0, c["chunk"] + 1, c["batch"])
        starts = rs.randint(0, c["prefix"] + 1, c["batch"])
    most = c["batch"] * ((c["prefix"] + c["chunk"] + c["page"] - 1) // c["page"]) + 7
    table, pool = _scattered_table(rs, starts + news, c["page"], most)
    shape = (pool, c["kv_heads"], c["page"], c["dim"])
    new = (c["batch"], c["kv_heads"], c["chunk"], c["dim"])
    return dict(case=c, new_k=_normal(gen, *new), new_v=_normal(gen, *new), k=_normal(gen, *shape),
                v=_normal(gen, *shape), table=_ints(table), starts=_ints(starts), news=_ints(news))


def _prepare_update(c, rs, gen):
    """Beams that share their prompt's full pages and own what follows."""
    groups, beams, page, pages = c["groups"], c["beams"], c["page"], c["pages"]
    entries = (c["longest"] + 1 + page - 1) // page + 1
    free, at = rs.permutation(pages), 0
    refs = np.zeros(pages, dtype=np.int64)
    table, lens = np.full((groups * beams, entries), -1), np.zeros(groups * beams, dtype=np.int64)
    parents = np.zeros(groups * beams, dtype=np.int64)
    for g in range(groups):
        length = rs.randint(1, c["longest"] + 1)
        held = (length + page - 1) // page
        common = rs.randint(0, length // page + 1)
        if at + common + beams * (held - common) > pages:
            common = held = length = 0
        for w in range(beams):
            r = g * beams + w
            if w:
                table[r, :common] = table[g * beams, :common]
            else:
                table[r, :common] = free[at:at + common]
                at += common
            table[r, common:held] = free[at:at + held - common]
            at += held - common
            lens[r] = length
            refs[table[r, :held]] += 1
            parents[r] = g * beams + rs.randint(0, beams)
    other = rs.randint(0, (pages - at) // 4 + 1)  # pages of sequences that are not in this table
    refs[free[at:at + other]] = 1
    pool = _normal(gen, c["slabs"], pages, page, c["row"])
    return dict(case=c, table=_ints(table), lens=_ints(lens), parents=_ints(parents),
                capacity=_ints(lens[parents] + 1), refs=_ints(refs), pool=pool)


def _prepare_compact(c, rs, gen):
    pages = c["pages"]
    live = rs.permutation(pages)[:max(1, int(pages * c["live"]))]
    entries = (c["longest"] + c["page"] - 1) // c["page"]
    table, at, refs = np.full((c["rows"], entries), -1), 0, np.zeros(pages, dtype=np.int64)
    refs[live] = 1
    for r in range(c["rows"]):
        n = min(rs.randint(0, entries + 1), len(live) - at)
        table[r, :n] = live[at:at + n]
        at += n
    refs[live[:at // 3]] += 1
    pool = _normal(gen, c["slabs"], pages, c["page"], c["row"])
    return dict(case=c, table=_ints(table), refs=_ints(refs), pool=pool)


def _prepare_beam(c, rs, gen):
    batch, beams = c["batch"], c["beams"]
    logits = _normal(gen, batch, beams, c["vocab"], dtype=torch.float32) * 3
    logits = logits if c["f32"] else logits.half()
    logits[:, :, ::97] = -math.inf  # tokens that the program bans
    scores = -5 * torch.rand(batch, beams, device=DEV, generator=gen)
    done = torch.zeros(batch, beams, dtype=torch.bool, device=DEV)
    if c["done"]:
        done = torch.rand(batch, beams, device=DEV, generator=gen) < 0.2
    history = torch.randint(0, c["vocab"], (batch * beams, c["tokens"]), dtype=torch.int32,
                            device=DEV, generator=gen)
    return dict(case=c, logits=logits, scores=scores, done=done, eos=2, history=history)


def prepare(case, seed):
    rs, gen = np.random.RandomState(seed % (1 << 32)), torch.Generator(device=DEV).manual_seed(seed)
    kind = {"decode": _prepare_attention, "prefill": _prepare_attention, "append": _prepare_append,
            "update": _prepare_update, "compact": _prepare_compact, "beam": _prepare_beam}
    return kind[case["op"]](dict(case), rs, gen)


# ---------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------
def _gathered(pages, table, positions):
    """[B, kv heads, n, D] in 32 bits: the rows at `positions` [B, n] of each sequence."""
    page = pages.shape[2]
    where = torch.gather(table.long(), 1, positions // page).clamp(min=0)
    return pages[where, :, positions % page].transpose(1, 2).float()


def _attention(q, k, v, visible, dim):
    """softmax(q k^T / sqrt(D)) v over the visible keys; zero where there is none."""
    s = torch.matmul(q, k.transpose(-1, -2)) * dim ** -0.5
    s = torch.where(visible, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0)


def _plain_decode(s):
    c = s["case"]
    batch, heads, dim = s["q"].shape
    reach = s["table"].shape[1] * c["page"]
    lens = s["lens"].long()[:, None]
    if c["window"] and c["window"] + c["sinks"] < reach:
        first = torch.clamp(lens - c["window"], min=c["sinks"])
        positions = torch.cat([torch.arange(c["sinks"], device=DEV).expand(batch, -1),
                               first + torch.arange(c["window"], device=DEV)], 1)
    else:
        positions = torch.arange(reach, device=DEV).expand(batch, -1)
    visible = positions < lens
    if c["window"]:
        visible = visible & ((positions >= lens - c["window"]) | (positions < c["sinks"]))
    positions = positions.clamp(max=reach - 1)
    k, v = _gathered(s["k"], s["table"], positions), _gathered(s["v"], s["table"], positions)
    q = s["q"].float().view(batch, c["kv_heads"], -1, dim)
    return _attention(q, k, v, visible[:, None, None], dim).reshape(batch, heads, dim).half()


def _plain_prefill(s):
    c = s["case"]
    batch, heads, chunk, dim = s["q"].shape
    keys = torch.arange(s["table"].shape[1] * c["page"], device=DEV)
    k = _gathered(s["k"], s["table"], keys.expand(batch, -1))
    v = _gathered(s["v"], s["table"], keys.expand(batch, -1))
    i = torch.arange(chunk, device=DEV)
    at = (s["lens"].long() - s["news"].long())[:, None, None] + i[:, None]
    visible = keys <= at
    if c["window"]:
        visible = visible & ((keys > at - c["window"]) | (keys < c["sinks"]))
    visible = visible & (i[:, None] < s["news"][:, None, None])
    q = s["q"].float().view(batch, c["kv_heads"], -1, chunk, dim)
    out = _attention(q, k[:, :, None], v[:, :, None], visible[:, None, None], dim)
    return out.reshape(batch, heads, chunk, dim).half()


def _plain_append(s):
    page, chunk = s["case"]["page"], s["case"]["chunk"]
    i = torch.arange(chunk, device=DEV)
    at = s["starts"].long()[:, None] + i
    b, i = torch.nonzero(i < s["news"][:, None], as_tuple=True)
    at = at[b, i]
    where = s["table"].long()[b, at // page]
    s["k"][where, :, at % page] = s["new_k"][b, :, i]
    s["v"][where, :, at % page] = s["new_v"][b, :, i]
    return s["k"], s["v"]


def _dense(mask, values):
    """The values where the mask holds, at the front and in order; -1 after them."""
    n = mask.numel()
    at = torch.where(mask, torch.cumsum(mask, 0) - 1, n)
    return torch.full((n + 1,), -1, device=DEV, dtype=torch.long).scatter(0, at, values)[:n]


def _plain_update(s):
    table, refs, page = s["table"].long(), s["refs"].long(), s["case"]["page"]
    rows, entries = table.shape
    count = refs.numel()
    parents = s["parents"].long()
    known = (parents >= 0) & (parents < rows)
    parent = torch.where(known, parents, 0)
    lens = torch.where(known, s["lens"].long()[parent], 0).clamp(0, entries * page)
    capacity = torch.maximum(s["capacity"].long().clamp(0, entries * page), lens)
    full, partial, held = lens // page, lens % page > 0, (capacity + page - 1) // page
    e = torch.arange(entries, device=DEV)
    old = table[parent]
    valid = (old >= 0) & (old < count)
    shared = (e < full[:, None]) & valid
    last = torch.gather(old, 1, full.clamp(max=entries - 1)[:, None])[:, 0]
    last_ok = partial & (last >= 0) & (last < count)
    b = torch.arange(len(parents), device=DEV)
    first = torch.full((rows,), len(parents), device=DEV).scatter_reduce(
        0, parent, torch.where(known, b, len(parents)), "amin")
    keeps = last_ok & (first[parent] == b) & (refs[last.clamp(0, count - 1)] == 1)
    copies = last_ok & ~keeps
    at_last = e == full[:, None]
    fresh = (e >= (full + partial)[:, None]) & (e < held[:, None]) | at_last & copies[:, None]
    new = torch.where(shared | at_last & keeps[:, None], old, -1)

    def holds(t):
        ok = (t >= 0) & (t < count)
        return torch.zeros(count, dtype=torch.long, device=DEV).scatter_add(
            0, t.clamp(0, count - 1).view(-1), ok.long().view(-1))

    left = (refs - holds(table) + holds(new)).clamp(min=0)
    free = _dense(left == 0, torch.arange(count, device=DEV))
    rank = (torch.cumsum(fresh.view(-1), 0) - 1).view_as(fresh)
    got = torch.where(fresh & (rank < count), free[rank.clamp(0, count - 1)], -1)
    new = torch.where(fresh, got, new)
    left = left + holds(got)
    to = torch.gather(new, 1, full.clamp(max=entries - 1)[:, None])[:, 0]
    copied = copies & (to >= 0)
    moves = torch.stack([_dense(copied, last), _dense(copied, to)]).int()
    info = torch.stack([(left == 0).sum(), (fresh & (got < 0)).sum(), copied.sum()]).int()
    pool = s["pool"]
    src, dst = last[copied], to[copied]
    pool[:, dst] = pool[:, src]
    return dict(table=new.int(), lens=lens.int(), refs=left.int(), copies=moves, info=info, pool=pool)


def _plain_compact(s):
    table, refs = s["table"].long(), s["refs"].long().clamp(min=0)
    count = refs.numel()
    live = refs > 0
    n = live.sum()
    at = torch.arange(count, device=DEV)
    holes, high = _dense(~live & (at < n), at), live & (at >= n)
    rank = (torch.cumsum(high, 0) - 1).clamp(min=0)
    index = torch.where(high, holes[rank], torch.where(live, at, -1))
    moves = torch.stack([_dense(high, at), holes])[:, :max(1, count // 2)].int()
    ok = (table >= 0) & (table < count)
    new = torch.where(ok, index[table.clamp(0, count - 1)], -1)
    left = torch.zeros(count + 1, dtype=torch.long, device=DEV).scatter(
        0, torch.where(live, index, count), refs)[:count]
    pool = s["pool"]
    src, dst = at[high], holes[:count][rank[high]]
    pool[:, dst] = pool[:, src]
    return dict(table=new.int(), refs=left.int(), moves=moves, index=index.int(),
                info=torch.stack([n, high.sum()]).int(), pool=pool)


def _plain_beam(s):
    """In 64 bits: which of two near candidates is the larger must not hang on a rounding."""
    batch, beams, vocab = s["logits"].shape
    width = s["case"]["width"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    x = x - torch.where(top == -math.inf, 0.0, top)
    x = x - torch.log(torch.exp(x).sum(-1, keepdim=True))
    x = x + s["scores"].double()[..., None]
    ended = torch.full((vocab,), -math.inf, device=DEV, dtype=torch.double)
    ended[s["eos"]] = 0
    x = torch.where(s["done"][..., None], s["scores"].double()[..., None] + ended, x)
    best, at = torch.sort(x.view(batch, -1), dim=-1, descending=True, stable=True)
    best, at = best[:, :width], at[:, :width]
    rows = torch.arange(batch, device=DEV)[:, None]
    none = best == -math.inf
    tokens = torch.where(none, -1, at % vocab)
    parents = torch.where(none, -1, rows * beams + at // vocab)
    done = ~none & (s["done"].view(-1)[parents.clamp(min=0)] | (tokens == s["eos"]))
    history = torch.where(parents.view(-1, 1) >= 0, s["history"][parents.clamp(min=0).view(-1)], 0)
    return dict(scores=best.float(), tokens=tokens.int(), parents=parents.int(), done=done,
                history=history)


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------
def _library(s):
    from llm_compiler_3_b200 import ops
    c = s["case"]
    op = c["op"]
    if op == "decode":
        return ops.paged_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], window=c["window"],
                                sinks=c["sinks"])
    if op == "prefill":
        return ops.paged_prefill(s["q"], s["k"], s["v"], s["table"], s["lens"], s["news"],
                                 window=c["window"], sinks=c["sinks"])
    if op == "append":
        ops.paged_append(s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["starts"], s["news"])
        return s["k"], s["v"]
    if op == "update":
        table, lens, refs, copies, info = ops.page_update(
            s["table"], s["lens"], s["parents"], s["capacity"], s["refs"], c["page"])
        ops.page_copy(s["pool"], copies, info[2:])
        return dict(table=table, lens=lens, refs=refs, copies=copies, info=info, pool=s["pool"])
    if op == "compact":
        table, refs, moves, index, info = ops.page_compact(s["table"], s["refs"])
        ops.page_copy(s["pool"], moves, info[1:])
        return dict(table=table, refs=refs, moves=moves, index=index, info=info, pool=s["pool"])
    scores, tokens, parents, done = ops.beam_select(s["logits"], s["scores"], c["width"], s["done"],
                                                    s["eos"])
    return dict(scores=scores, tokens=tokens, parents=parents, done=done,
                history=ops.beam_reorder(s["history"], parents))


def run(state):
    if own:
        return _library(state)
    plain = {"decode": _plain_decode, "prefill": _plain_prefill, "append": _plain_append,
             "update": _plain_update, "compact": _plain_compact, "beam": _plain_beam}
    return plain[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without (lengths at their expectation where they are drawn)
# ---------------------------------------------------------------------------------------------
def _visible(at, window, sinks):
    """Keys that the query at position `at` sees."""
    if not window or at + 1 <= window:
        return at + 1
    return window + min(sinks, at + 1 - window)


def work(case):
    c, op = case, case["op"]
    if op == "decode":
        rng = np.random.RandomState(0)
        lengths = np.full(c["batch"], c["longest"])
        if c["ragged"]:
            lengths = rng.randint(1, c["longest"] + 1, c["batch"])
            lengths[0] = c["longest"]
            lengths[7::8] = 0
        keys = sum(_visible(int(n) - 1, c["window"], c["sinks"]) for n in lengths if n)
        return dict(bytes=4 * c["dim"] * (c["kv_heads"] * keys + c["heads"] * c["batch"]),
                    flops=4 * c["dim"] * c["heads"] * keys)
    if op == "prefill":
        half = 0.5 if c["ragged"] else 1.0
        pairs = keys = news = 0
        for b in range(c["batch"]):
            n = c["chunk"] if b == 0 else max(1, int(c["chunk"] * half))
            p = c["prefix"] if b == 0 else int(c["prefix"] * half)
            pairs += sum(_visible(p + i, c["window"], c["sinks"]) for i in range(n))
            keys += _visible(p + n - 1, c["window"] and c["window"] + n - 1, c["sinks"])
            news += n
        return dict(bytes=2 * c["dim"] * (c["heads"] * (news + c["batch"] * c["chunk"]) + 2 * c["kv_heads"] * keys),
                    flops=4 * c["dim"] * c["heads"] * pairs)
    if op == "append":
        rows = c["batch"] * c["chunk"] * (0.5 if c["ragged"] else 1.0)
        return dict(bytes=8 * rows * c["kv_heads"] * c["dim"], flops=0)
    if op == "update":
        rows = c["groups"] * c["beams"]
        entries = c["longest"] // c["page"] + 2
        alone = (1 - 1 / c["beams"]) ** c["beams"]  # a parent without children; the others keep a page
        copies = rows * alone * (1 - 1 / c["page"]) if c["beams"] > 1 else 0
        return dict(bytes=8 * rows * entries + 8 * c["pages"] + copies * c["slabs"] * c["page"] * c["row"] * 4,
                    flops=0)
    if op == "compact":
        entries = (c["longest"] + c["page"] - 1) // c["page"]
        moves = c["pages"] * c["live"] * (1 - c["live"])
        return dict(bytes=8 * c["rows"] * entries + 12 * c["pages"] + moves * c["slabs"] * c["page"] * c["row"] * 4,
                    flops=0)
    rows = c["batch"] * c["beams"] * (0.8 if c["done"] else 1.0)
    return dict(bytes=rows * c["vocab"] * (4 if c["f32"] else 2) + 4 * c["batch"] * c["tokens"] * (c["beams"] + c["width"]),
                flops=3 * rows * c["vocab"])


# ---------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c, op = s["case"], case["op"]
    if op in ("decode", "prefill"):
        q = s["q"].double()
        q = q[:, :, None] if op == "decode" else q
        out = torch.zeros_like(q)
        page, group = c["page"], c["heads"] // c["kv_heads"]
        for b in range(c["batch"]):
            n, m = int(s["lens"][b]), int(s["news"][b])
            if n == 0:
                continue
            held = s["table"][b, :(n + page - 1) // page].long()
            k, v = (t[held].transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :n].double()
                    for t in (s["k"], s["v"]))
            at, j = torch.arange(n - m, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
            hidden = j > at
            if c["window"]:
                hidden = hidden | ((at - j >= c["window"]) & (j >= c["sinks"]))
            for h in range(c["heads"]):
                w = (q[b, h, :m] @ k[h // group].T / math.sqrt(c["dim"])).masked_fill(hidden, -math.inf)
                out[b, h, :m] = torch.softmax(w, -1) @ v[h // group]
        return out[:, :, 0] if op == "decode" else out
    if op == "beam":
        x = s["logits"].double()
        x = x - torch.logsumexp(x, -1, keepdim=True) + s["scores"].double()[..., None]
        x[s["done"]] = -math.inf
        ended = torch.where(s["done"], s["scores"].double(), -math.inf)
        every = torch.cat([x.flatten(1), ended], 1)
        return dict(scores=torch.topk(every, c["width"], -1).values, tokens=None, parents=None,
                    done=None, history=None)
    return None
