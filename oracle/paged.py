"""64-bit CPU restatement of the paged-cache operators (test infrastructure only).

Written from the definitions in ``include/npu_b200.h``: sequences are rebuilt
from their pages one by one, every key is shown or hidden by the written rule,
and softmax is taken in FP64.  ``attention_paged`` also returns, per output
element, how far a kernel may be off that rounds only where the kernels do:

  * each softmax weight to FP16 before the second product, relative to a number
    2^7 or more below the largest weight: a relative 2^-11 (below 2^-21 of the
    largest, where FP16 is subnormal, an absolute 2^-32 of it);
  * scores in FP32: a dot product of D terms is off by at most (D + 4) 2^-23
    times the sum of the terms' magnitudes (tensor cores may cut instead of
    round, hence 2^-23), which moves each weight by that relative amount, and
    the exponential by 2^-21;
  * sums of n weights and n products in FP32: n 2^-23 each, relative to the
    sum of the magnitudes;
  * the output to FP16: 2^-11 of it (2^-25 below the normal numbers).
"""
from __future__ import annotations

import torch

__all__ = ["rows_of_pages", "attention_paged", "append_paged", "page_update", "page_compact",
           "page_copy"]


def rows_of_pages(pages: torch.Tensor, row: torch.Tensor, n: int) -> torch.Tensor:
    """Positions [0, n) of one sequence: [Hkv, n, D].  Entries that are no page
    (their positions must be hidden) give NaN."""
    page_size = pages.shape[2]
    parts = []
    for e in range((n + page_size - 1) // page_size):
        page = int(row[e])
        ok = 0 <= page < pages.shape[0]
        parts.append(pages[page] if ok else torch.full_like(pages[0], float("nan")))
    if not parts:
        return pages[0][:, :0]
    return torch.cat(parts, 1)[:, :n]


def attention_paged(q, k_pages, v_pages, table, seq_lens, q_lens=None, window=0, sinks=0,
                    scale=None):
    """q [B, Hq, M, D]; query i < q_lens[b] (default M) of sequence b is at position
    seq_lens[b] - q_lens[b] + i; later rows are zero.  Returns (out, bound) in FP64."""
    batch, heads, chunk, dim = q.shape
    kv_heads = k_pages.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(batch):
        n = int(seq_lens[b])
        m = chunk if q_lens is None else int(q_lens[b])
        k = rows_of_pages(k_pages, table[b], n).double()
        v = rows_of_pages(v_pages, table[b], n).double()
        for i in range(m):
            p = n - m + i
            see = [j for j in range(n)
                   if 0 <= j <= p and (window == 0 or j > p - window or j < sinks)]
            if not see:
                continue
            for h in range(heads):
                kk, vv = k[h * kv_heads // heads][see], v[h * kv_heads // heads][see]
                qq = q[b, h, i].double()
                w = torch.softmax(kk @ qq * scale, 0)
                out[b, h, i] = w @ vv
                mass = w @ vv.abs()
                off = float((kk.abs() @ qq.abs()).max()) * abs(scale) * (dim + 4) * 2.0 ** -23
                rel = 2.0 ** -11 + 2 * off + 2.0 ** -20 + 2 * len(see) * 2.0 ** -23
                bound[b, h, i] = (2.0 ** -11 * out[b, h, i].abs() + 2.0 ** -25 + rel * mass
                                  + len(see) * 2.0 ** -32 * vv.abs().max())
    return out, bound


def append_paged(k, k_pages, table, starts, lens=None):
    """k [B, Hkv, M, D] into a copy of the pages; rows without a page are dropped."""
    pages = k_pages.clone()
    page_size = pages.shape[2]
    for b in range(k.shape[0]):
        for i in range(k.shape[2] if lens is None else int(lens[b])):
            at = int(starts[b]) + i
            if not 0 <= at < table.shape[1] * page_size:
                continue
            page = int(table[b, at // page_size])
            if 0 <= page < pages.shape[0]:
                pages[page, :, at % page_size] = k[b, :, i]
    return pages


def page_update(table, lens, parents, capacity, refs, page_size):
    """The next step's page table, row by row on Python numbers; returns the lists
    (table, lens, refs, copies, info) of npu_b200_page_update."""
    old = [[int(x) for x in row] for row in table]
    rows, entries, n = len(old), len(old[0]), len(refs)
    page = lambda x: 0 <= x < n  # noqa: E731
    left = [int(x) for x in refs]
    for row in old:
        for x in row:
            if page(x):
                left[x] -= 1
    new, new_lens, wants, seen = [], [], [], set()
    for b, parent in enumerate(int(x) for x in parents):
        row = [-1] * entries
        length = 0
        if 0 <= parent < rows:
            length = min(max(int(lens[parent]), 0), entries * page_size)
        cap = max(min(max(int(capacity[b]), 0), entries * page_size), length)
        full, part = divmod(length, page_size)
        for e in range(full):
            if page(old[parent][e]):
                row[e] = old[parent][e]
                left[row[e]] += 1
        start = full
        if part:
            start += 1
            last = old[parent][full]
            if page(last):
                if parent not in seen and int(refs[last]) == 1:
                    row[full] = last
                    left[last] += 1
                else:
                    wants.append((b, full, last))
        if 0 <= parent < rows:
            seen.add(parent)
        wants += [(b, e, None) for e in range(start, -(-cap // page_size))]
        new.append(row)
        new_lens.append(length)
    left = [max(x, 0) for x in left]
    sources = {s for _, _, s in wants if s is not None}
    free = [p for p in range(n) if left[p] == 0 and p not in sources]
    copies, short = [], 0
    for b, e, source in wants:
        if not free:
            short += 1
            continue
        new[b][e] = free.pop(0)
        left[new[b][e]] = 1
        if source is not None:
            copies.append((source, new[b][e]))
    pad = len(new) - len(copies)
    moves = [[s for s, _ in copies] + [-1] * pad, [d for _, d in copies] + [-1] * pad]
    return new, new_lens, left, moves, [len(free) + sum(left[p] == 0 for p in sources), short,
                                        len(copies)]


def page_compact(table, refs):
    """The lists (table, refs, moves, index, info) of npu_b200_page_compact."""
    n = len(refs)
    live = [p for p in range(n) if int(refs[p]) > 0]
    count = len(live)
    holes = [p for p in range(count) if int(refs[p]) <= 0]
    high = [p for p in live if p >= count]
    index = [-1] * n
    for p in live:
        index[p] = p
    for p, to in zip(high, holes):
        index[p] = to
    left = [0] * n
    for p in live:
        left[index[p]] = int(refs[p])
    new = [[index[int(x)] if 0 <= int(x) < n else -1 for x in row] for row in table]
    pad = [-1] * (max(1, n // 2) - len(high))
    return new, left, [high + pad, holes + pad], index, [count, len(high)]


def page_copy(pool, pages, count=None):
    """pool [slabs, N, ...] with pages[0][i] copied to pages[1][i], as a new tensor."""
    out = pool.clone()
    n = len(pages[0]) if count is None else min(max(int(count), 0), len(pages[0]))
    for i in range(n):
        s, d = int(pages[0][i]), int(pages[1][i])
        if 0 <= s < pool.shape[1] and 0 <= d < pool.shape[1]:
            out[:, d] = pool[:, s]
    return out
