"""Attention of a chunk of new tokens over a paged cache, against the 64-bit oracle
(oracle/paged.py, which derives each element's bound; a weight's rounding is
relative to a maximum that may lag by 2^8, so its absolute part, 2^-25 of the
largest weight, only shrinks)."""
import pytest
import torch

import oracle
from conftest import seeded
from test_paged import INF, NAN, check, check_with_nan, far_below, ints, paged_cache, steep


def _prefill(q, k, v, table, lens, q_lens=None, **kw):
    from llm_compiler_3_b200 import _native, ops
    out = torch.full(q.shape, NAN, dtype=torch.float16, device="cuda")
    ops.paged_prefill(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ints(lens).cuda(),
                      None if q_lens is None else ints(q_lens).cuda(), out=out, **kw)
    torch.cuda.synchronize()
    assert _native.device_status() == 0
    return out.cpu()


def check_prefill(q, k, v, table, lens, q_lens=None, **kw):
    got = _prefill(q, k, v, table, lens, q_lens, **kw)
    check(got, *oracle.attention_paged(q, k, v, table, lens, q_lens, **kw))
    return got


PREFILL_ARGS = dict(batch=2, q_heads=8, kv_heads=2, head_dim=128, queries=5, num_pages=9, page_size=16,
                    entries=4, window=0, sinks=0, scale=0.1)


@pytest.mark.parametrize("change,message", [
    (dict(head_dim=96), "head_dim 96"), (dict(q_heads=7), "multiple of kv_heads"),
    (dict(kv_heads=0), "kv_heads 0"), (dict(page_size=12), "page_size 12"),
    (dict(num_pages=0), "0 pages"), (dict(num_pages=1 << 26), "too many rows"),
    (dict(entries=0), "0 table entries"), (dict(batch=0), "batch 0"), (dict(queries=0), "queries 0"),
    (dict(queries=1 << 26), "too many query blocks"),
    (dict(window=-1), "window -1"), (dict(sinks=-1), "sinks -1"), (dict(scale=INF), "scale"),
    (dict(scale=NAN), "scale"),
])
def test_refusals(change, message):
    """Refused on the host, before any CUDA call."""
    from llm_compiler_3_b200 import _native
    a = dict(PREFILL_ARGS, **change)
    p = 1 << 20

    def call(ptrs):
        return _native.lib().npu_b200_paged_prefill(
            *ptrs, a["batch"], a["q_heads"], a["kv_heads"], a["head_dim"], a["queries"], a["num_pages"],
            a["page_size"], a["entries"], a["window"], a["sinks"], a["scale"], None)

    assert call([p] * 7) == -1
    assert message.encode() in _native.lib().npu_b200_last_error()
    a = dict(PREFILL_ARGS)
    for i in (0, 1, 2, 3, 4, 6):
        assert call([None if j == i else p for j in range(7)]) == -1
    for i in (0, 1, 2, 6):
        assert call([p + 8 if j == i else p for j in range(7)]) == -1


# ---- on the GPU ------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("page", [8, 16, 24, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_page_sizes(cuda, page, dim):
    """Pages smaller and larger than the 128-key tile; ragged chunks after ragged prefixes."""
    lens, q_lens = [130, 40, 257, 7, 0], [17, 40, 1, 3, 0]
    k, v, table = paged_cache(lens, 2, dim, page, seed=page)
    check_prefill(seeded((5, 4, 40, dim), 3), k, v, table, lens, q_lens)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (6, 2), (7, 1), (8, 1), (16, 1), (24, 2), (40, 1)])
@pytest.mark.parametrize("queries", [1, 5, 33])
def test_groups_and_few_queries(cuda, heads, kv_heads, queries):
    """Any number of query heads to a key head, stacked in a tile or over several."""
    lens = [70, queries]
    k, v, table = paged_cache(lens, kv_heads, 64, 16, seed=heads)
    check_prefill(seeded((2, heads, queries, 64), 4), k, v, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [127, 128, 129, 256, 300])
@pytest.mark.parametrize("dim", [64, 128])
def test_query_tiles(cuda, queries, dim):
    """Chunks around one and two query tiles, some rows at negative positions."""
    lens = [queries + 5, queries // 2]
    k, v, table = paged_cache(lens, 1, dim, 32, seed=queries)
    check_prefill(seeded((2, 2, queries, dim), 5), k, v, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (50, 33), (64, 100), (100, 3), (128, 128),
                                          (129, 140), (200, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_window(cuda, window, sinks):
    """Windows and sinks on, inside and across tile borders; keys that no query sees hold
    NaN, and the entries of pages without a visible key are no pages."""
    lens, q_lens = [700, 64, 300, 1, 0, 133], [100, 64, 30, 1, 0, 5]
    k, v, table = paged_cache(lens, 1, 64, 16, seed=window % 1000 + sinks % 1000)
    shown = table.clone()
    for b, (n, m) in enumerate(zip(lens, q_lens)):
        seen = [j > n - m - window or j < sinks for j in range(n)]
        for j in range(n):
            if not seen[j]:
                k[table[b, j // 16], :, j % 16] = NAN
                v[table[b, j // 16], :, j % 16] = INF
        for e in range((n + 15) // 16):
            if not any(seen[e * 16:e * 16 + 16]):
                shown[b, e] = -1
    check_prefill(seeded((6, 2, 100, 64), 6), k, v, shown, lens, q_lens, window=window, sinks=sinks)


@pytest.mark.gpu
def test_window_of_a_long_chunk(cuda):
    """Query tiles far apart: each reads its own tiles and the sinks'."""
    lens, q_lens = [900], [700]
    k, v, table = paged_cache(lens, 1, 128, 64, seed=31)
    check_prefill(seeded((1, 1, 700, 128), 7), k, v, table, lens, q_lens, window=150, sinks=20)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_of_any_size(cuda, dim):
    """Scores far apart (maxima that move), all equal, and negative scales."""
    lens = [400, 300]
    k, v, table = paged_cache(lens, 1, dim, 16, seed=9)
    q = seeded((2, 4, 20, dim), 8, std=20.0)
    check_prefill(q, k, v, table, lens)
    check_prefill(q, k, v, table, lens, scale=-0.125)
    check_prefill(q, k, v, table, lens, scale=0.0)
    order = torch.arange(400).float()
    for b, n in enumerate(lens):  # rising scores: the maximum moves at every tile
        for j in range(n):
            k[table[b, j // 16], :, j % 16] = order[j] / 100
    check_prefill(torch.ones(2, 4, 20, dim).half(), k, v, table, lens, scale=0.5)


@pytest.mark.gpu
def test_agrees_with_the_contiguous_operator_and_with_decode(cuda):
    """A prompt in pages is the prompt in a flat cache; its last row is a decode step."""
    from llm_compiler_3_b200 import ops
    n = 517
    k, v, table = paged_cache([n], 2, 128, 32, seed=12)
    q = seeded((1, 8, n, 128), 9)
    got = _prefill(q, k, v, table, [n])
    flat = [oracle.rows_of_pages(t, table[0], n)[None].contiguous().cuda() for t in (k, v)]
    want = ops.prefill_attention(q.cuda(), *flat, causal=True).cpu()
    assert float((got.float() - want.float()).abs().max()) < 1e-2
    one = ops.paged_decode(q[:, :, -1].contiguous().cuda(), k.cuda(), v.cuda(), table.cuda(), ints([n]).cuda()).cpu()
    check(got[:, :, -1:], *oracle.attention_paged(q[:, :, -1:], k, v, table, [n]))
    check(one[:, :, None], *oracle.attention_paged(q[:, :, -1:], k, v, table, [n]))


@pytest.mark.gpu
def test_clamps_lengths_and_reports_bad_pages(cuda):
    from llm_compiler_3_b200 import _native, ops
    k, v, table = paged_cache([48, 48], 1, 64, 16, seed=10)
    q = seeded((2, 2, 9, 64), 9)
    assert torch.equal(_prefill(q, k, v, table, [1 << 30, -5], [100, 4]), _prefill(q, k, v, table, [48, 0], [9, 4]))
    assert torch.count_nonzero(_prefill(q, k, v, table, [48, 48], [0, -3])) == 0
    for page in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        bad = table.clone()
        bad[1, 1] = page
        out = ops.paged_prefill(q.cuda(), k.cuda(), v.cuda(), bad.cuda(), ints([48, 48]).cuda())
        with pytest.raises(_native.NpuError, match="0x8"):
            _native.device_status()
        assert torch.equal(out[0].cpu(), _prefill(q, k, v, table, [48, 48])[0])


@pytest.mark.gpu
def test_on_streams_and_in_graphs(cuda):
    from llm_compiler_3_b200 import ops
    lens = [300, 200]
    k, v, table = (t.cuda() for t in paged_cache(lens, 1, 128, 16, seed=13))
    q, n = seeded((2, 4, 90, 128), 11).cuda(), ints(lens).cuda()
    want = ops.paged_prefill(q, k, v, table, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_prefill(q, k, v, table, n)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.paged_prefill(q, k, v, table, n))
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and all(torch.equal(g, want) for g in got)
    n.copy_(ints([95, 90]))
    graph.replay()
    assert torch.equal(out, ops.paged_prefill(q, k, v, table, n))


@pytest.mark.gpu
def test_checks_of_the_wrapper(cuda):
    from llm_compiler_3_b200 import ops
    k, v, table = (t.cuda() for t in paged_cache([20, 20], 2, 64, 16))
    q, n = seeded((2, 4, 3, 64), 1).cuda(), ints([20, 20]).cuda()
    good = dict(q=q, k_pages=k, v_pages=v, page_table=table, seq_lens=n)
    for change in (dict(q=q.float()), dict(q=q[:, :, :, ::2]), dict(q=q[:1]), dict(q=q[:, :, 0]),
                   dict(seq_lens=n[:1]), dict(q_lens=n[:1]), dict(q_lens=n.long()), dict(v_pages=v[:1]),
                   dict(out=torch.empty_like(q)[:1]), dict(q_lens=n.cpu())):
        with pytest.raises(ValueError):
            ops.paged_prefill(**dict(good, **change))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dim,window,sinks", [(2, 64, 0, 0), (4, 128, 0, 0), (4, 64, 20, 3), (2, 128, 9, 0)])
def test_values_that_are_no_numbers_stay_with_the_queries_that_see_them(cuda, heads, dim, window, sinks):
    """Infinite and NaN values of some tokens reach exactly the queries and dimensions that see
    them: not the queries before, though they share a tile, nor those whose window has passed."""
    lens, q_lens = [150, 300], [150, 140]
    k, v, table = paged_cache(lens, 2, dim, 16, seed=dim + window)
    for b, j, d, x in ((0, 40, 3, NAN), (0, 120, 7, INF), (1, 170, 1, -INF), (1, 290, 0, NAN)):
        v[int(table[b, j // 16]), :, j % 16, d] = x
    q = seeded((2, heads, 150, dim), 6)
    got = _prefill(q, k, v, table, lens, q_lens, window=window, sinks=sinks)
    want = oracle.attention_paged(q, k, v, table, lens, q_lens, window=window, sinks=sinks)[0]
    odd = ~want.isfinite()
    assert odd.any() and torch.equal(got.double().nan_to_num(1e9, 2e9, 3e9)[odd], want.nan_to_num(1e9, 2e9, 3e9)[odd])
    # The other elements do not depend on them: as with zeros in their places.
    want, bound = oracle.attention_paged(q, k, v.nan_to_num(0, 0, 0), table, lens, q_lens, window=window, sinks=sinks)
    check(torch.where(odd, want.half(), got), want, torch.where(odd, want.abs(), bound))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim,queries", [(4, 1, 64, 7), (4, 1, 128, 7), (2, 2, 128, 130), (8, 4, 64, 40),
                                                        (16, 16, 128, 3), (8, 8, 128, 300)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 9)])
def test_keys_shared_by_a_cluster(cuda, heads, kv_heads, dim, queries, window, sinks):
    """Few query tiles behind long prefixes: CTAs that share the keys of a tile, some of them
    without any; all of a row's keys in one CTA's share; empty sequences; the same bits twice."""
    lens, q_lens = [1400, queries, 129, 0], [queries, queries, 1, 0]
    k, v, table = paged_cache(lens, kv_heads, dim, 16, seed=dim + queries)
    q = seeded((4, heads, queries, dim), 8)
    got = check_prefill(q, k, v, table, lens, q_lens, window=window, sinks=sinks)
    assert torch.equal(got, _prefill(q, k, v, table, lens, q_lens, window=window, sinks=sinks))
    check_prefill(q[:1], k, v, table[:1], lens[:1], q_lens[:1], window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [8, 24, 40, 64, 128])
@pytest.mark.parametrize("dim,window,sinks", [(64, 150, 33), (128, 95, 8), (64, 1, 200), (128, 257, 0), (64, 32, 32)])
def test_windows_over_units_of_keys(cuda, page, dim, window, sinks):
    """Sinks, gap and window in one tile, in units of 32 keys that pages of other sizes cut across;
    sinks that run into the window; chunks that begin anywhere."""
    lens, q_lens = [700, 333, 65, 20], [140, 33, 65, 7]
    k, v, table = paged_cache(lens, 1, dim, page, seed=page + sinks)
    check_prefill(seeded((4, 2, 140, dim), 9), k, v, table, lens, q_lens, window=window, sinks=sinks)


@pytest.mark.gpu
def test_captured_and_overlapping_calls(cuda):
    """A captured call follows the lengths and tables it finds; calls on two streams, of clusters and
    of many CTAs, keep apart."""
    from llm_compiler_3_b200 import _native, ops
    lens, q_lens = [500, 61], [33, 20]
    k, v, table = paged_cache(lens, 2, 128, 16, seed=5)
    q = seeded((2, 8, 33, 128), 12)
    state = [t.cuda() for t in (q, k, v, table, ints(lens), ints(q_lens))]
    ops.paged_prefill(*state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_prefill(*state)
    for new_lens, new_q in (([500, 61], [33, 20]), ([61, 7], [1, 0]), ([300, 60], [0, 33])):
        state[4].copy_(ints(new_lens))
        state[5].copy_(ints(new_q))
        graph.replay()
        torch.cuda.synchronize()
        check(out.cpu(), *oracle.attention_paged(q, k, v, table, new_lens, new_q))
    other = seeded((2, 8, 700, 128), 13).cuda()
    long = ints([500, 61]).cuda()
    want = [ops.paged_prefill(*state), ops.paged_prefill(other, *state[1:4], long, long)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(8):
        with torch.cuda.stream(streams[0]):
            got[0].append(ops.paged_prefill(*state))
        with torch.cuda.stream(streams[1]):
            got[1].append(ops.paged_prefill(other, *state[1:4], long, long))
    torch.cuda.synchronize()
    assert _native.device_status() == 0
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [1, 4, 9, 20])
@pytest.mark.parametrize("dim,queries", [(64, 3), (128, 3), (128, 40), (64, 200)])
def test_queries_and_keys_that_are_no_numbers(cuda, dim, queries, copies):
    """NaN in a query, in the newest key alone in its tile (and in its CTA's share), in every key of a
    tile, in one key of a tile whose other keys weigh nothing: the rows that see it are NaN, whether
    clusters of 8, 4 or 2 CTAs join their parts or one CTA has them all."""
    lens = [897, 897, 897, 897] * copies
    k, v, table = paged_cache(lens, 1, dim, 16, seed=dim + queries)
    q = seeded((len(lens), 2, queries, dim), 14)

    def key(row, j):
        return k[int(table[row, j // 16]), 0, j % 16]

    for c in range(0, len(lens), 4):
        q[c, 1, queries // 2, 5] = NAN
        key(c + 1, 896)[7] = NAN
        for j in range(256, 384):
            key(c + 2, j)[0] = NAN
            key(c + 3, j)[:] = -30
        q[c + 3] = q[c + 3].abs() + 1  # the scores of tile 2 lie 240 and more below the others
        key(c + 3, 300)[9] = NAN
    got = _prefill(q, k, v, table, lens, [queries] * len(lens))
    want, bound = oracle.attention_paged(q[:4], k, v, table[:4], lens[:4], [queries] * 4)
    for c in range(0, len(lens), 4):
        if c:  # the same tokens, other pages and values: only where NaN is
            assert torch.equal(got[c:c + 4].isnan(), want.isnan())
        else:
            check_with_nan(got[:4], want, bound)


@pytest.mark.gpu
def test_numbers_that_are_none_cost_no_second_pass(cuda):
    """A prompt with NaN in all queries, in one key, in one early or late value or in all values
    takes about what it takes without (rows done again one by one took 400 times as long)."""
    from llm_compiler_3_b200 import ops
    n = 2048
    k, v, table = paged_cache([n], 2, 128, 64, seed=3)
    q = seeded((1, 8, n, 128), 5)

    def took(q, k, v):
        state = [t.cuda() for t in (q, k, v, table, ints([n]))]
        ops.paged_prefill(*state)
        times = []
        for _ in range(5):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            ops.paged_prefill(*state)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return sorted(times)[2]

    bad_q, bad_k, bad_v, late_v, all_v = q.clone(), k.clone(), v.clone(), v.clone(), v.clone()
    bad_q[..., 3] = NAN
    bad_k[int(table[0, 0]), :, 0, 3] = NAN
    bad_v[int(table[0, 0]), :, 0, 3] = NAN
    late_v[int(table[0, -1]), :, 40] = NAN
    all_v[:, :, :, 3] = NAN
    plain = took(q, k, v)
    for case in ((bad_q, k, v), (q, bad_k, v), (q, k, bad_v), (q, k, late_v), (q, k, all_v)):
        assert took(*case) < 4 * plain + 0.1, (took(*case), plain)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dim,window,sinks", [(2, 64, 0, 0), (8, 128, 0, 0), (2, 128, 100, 0), (8, 64, 300, 9),
                                                    (1, 64, 40, 600), (4, 128, 1, 0), (4, 64, 64, 32)])
@pytest.mark.parametrize("batch,queries", [(1, 7), (3, 70), (16, 150), (2, 333)])
def test_values_that_are_no_numbers_behind_long_prefixes(cuda, heads, dim, window, sinks, batch, queries):
    """The same where clusters share the keys and where one CTA has them: single tokens with infinite
    or NaN values in the prefix, in the chunk, beside one another in one dimension; chunks that are
    shorter than the call's."""
    lens, q_lens = ([900, 450, 641, 70] * 4)[:batch], [queries, 65, 1, 70] * 4
    q_lens = [min(a, b, queries) for a, b in zip(lens, q_lens)]
    k, v, table = paged_cache(lens, 1, dim, 16, seed=dim + window)
    for b, (n, m) in enumerate(zip(lens, q_lens)):
        for j, d, x in ((n - 1, 0, NAN), (n - m, 9, INF), (n - m + 3, 9, -INF), (n - m + 5, 17, INF), (n // 2, 33, -INF),
                        (n - 40, 63, NAN), (max(0, n - m - 20), 40, INF), (3, 41, NAN)):
            if 0 <= j < n:
                v[int(table[b, j // 16]), :, j % 16, d] = x
    q = seeded((batch, heads, queries, dim), 6)
    got = _prefill(q, k, v, table, lens, q_lens, window=window, sinks=sinks)
    rows = slice(0, 3)  # of 64 bits; the others are as many more of the same
    args = (q[rows], k, v, table[rows], lens[rows], q_lens[rows])
    want = oracle.attention_paged(*args, window=window, sinks=sinks)[0]
    odd = ~want.isfinite()
    some = got[rows].double()
    assert odd.any() and torch.equal(some.nan_to_num(1e9, 2e9, 3e9)[odd], want.nan_to_num(1e9, 2e9, 3e9)[odd])
    args = (q[rows], k, v.nan_to_num(0, 0, 0), *args[3:])
    want, bound = oracle.attention_paged(*args, window=window, sinks=sinks)
    check(torch.where(odd, want.half(), got[rows]), want, torch.where(odd, want.abs(), bound))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,queries", [(20, 3), (900, 7), (900, 300)])
def test_keeps_weights_far_below_the_largest(cuda, dim, n, queries):
    """As in decode, for every query that sees some of them."""
    q, k, v, table = far_below(dim, 16, n)
    q = q[:, :, None].expand(1, 2, queries, dim).contiguous()
    got = _prefill(q, k, v, table, [n], scale=1.0)
    want, _ = oracle.attention_paged(q, k, v, table, [n], scale=1.0)
    check(got, want, 3 * 2.0 ** -11 * want + 2.0 ** -25 + 64 * n * 2.0 ** -32)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("base", [0, 10, 20, 23, 24, 25, 26])
def test_steep_and_large_scores(cuda, dim, base):
    """As in decode."""
    for n, queries, scale in ((300, 300, 1.0), (700, 5, -1.0), (3000, 130, 1.0)):
        q, k, v, table = steep(dim, 16, n, base)
        q = q[:, :, None].expand(1, 2, queries, dim).contiguous() * scale
        got = _prefill(q, k, v, table, [n], scale=scale)
        assert float((got.double() - 1).abs().max()) <= 2.0 ** -10 + n * 2.0 ** -23
