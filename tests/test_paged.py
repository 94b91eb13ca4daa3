"""Paged key-value cache: attention of one new token and the append, against the
64-bit oracle (oracle/paged.py, which derives each element's bound)."""
import ctypes

import pytest
import torch

import oracle
from conftest import seeded

NAN, INF = float("nan"), float("inf")


def paged_cache(lens, kv_heads, dim, page, seed=0, spare=3, reserve=0):
    """(k_pages, v_pages, table) with the sequences' pages in no order; rows past
    each length and every unused page hold NaN (K) and infinity (V)."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + reserve + page - 1) // page for n in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g).tolist()
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    k = torch.full((pool, kv_heads, page, dim), NAN).half()
    v = torch.full((pool, kv_heads, page, dim), INF).half()
    at = 0
    for b, n in enumerate(lens):
        for e in range(need[b]):
            table[b, e] = order[at]
            rows = max(0, min(page, n - e * page))
            k[order[at], :, :rows] = seeded((kv_heads, rows, dim), seed + 1000 + at)
            v[order[at], :, :rows] = seeded((kv_heads, rows, dim), seed + 9000 + at)
            at += 1
    return k, v, table


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def _decode(q, k, v, table, lens, **kw):
    from llm_compiler_3_b200 import _native, ops
    dev = torch.device("cuda", 0)
    out = ops.paged_decode(q.to(dev), k.to(dev), v.to(dev), table.to(dev), ints(lens).to(dev), **kw)
    torch.cuda.synchronize()
    assert _native.device_status() == 0
    return out.cpu()


def check(got, want, bound):
    assert torch.isfinite(got).all()
    off = (got.double() - want).abs() - bound
    assert float(off.max()) <= 0, f"off by {float((got.double() - want).abs().max())}, past its bound by {float(off.max())}"


def check_decode(q, k, v, table, lens, **kw):
    got = _decode(q, k, v, table, lens, **kw)
    want, bound = oracle.attention_paged(q[:, :, None], k, v, table, lens, q_lens=[min(1, n) for n in lens], **kw)
    check(got, want[:, :, 0], bound[:, :, 0])
    return got


# ---- on the CPU: the oracle and the refusals -------------------------------------------------
def test_oracle_agrees_with_the_flat_oracle():
    lens = [37, 1, 16]
    k, v, table = paged_cache(lens, 2, 64, 16)
    q = seeded((3, 6, 64), 1)
    got, bound = oracle.attention_paged(q[:, :, None], k, v, table, lens, q_lens=[1, 1, 1])
    for b, n in enumerate(lens):
        flat = [oracle.rows_of_pages(t, table[b], n)[None] for t in (k, v)]
        want = oracle.attention_decode(q[b:b + 1], flat[0], flat[1], [n], 64 ** -0.5)
        torch.testing.assert_close(got[b, :, 0].float(), want[0], atol=1e-5, rtol=1e-5)
    assert float(bound.max()) < 1e-2


def test_oracle_window_and_sinks():
    """window 4 and 2 sinks at position 9 of 10: keys 0, 1, 6, 7, 8, 9."""
    k, v, table = paged_cache([10], 1, 64, 8)
    q = seeded((1, 1, 1, 64), 2)
    got, _ = oracle.attention_paged(q, k, v, table, [10], window=4, sinks=2)
    kk, vv = (oracle.rows_of_pages(t, table[0], 10)[0, [0, 1, 6, 7, 8, 9]].double() for t in (k, v))
    want = torch.softmax(kk @ q[0, 0, 0].double() / 8, 0) @ vv
    torch.testing.assert_close(got[0, 0, 0], want)


DECODE_ARGS = dict(batch=2, q_heads=8, kv_heads=2, head_dim=128, num_pages=9, page_size=16, entries=4,
                   window=0, sinks=0, scale=0.1)


@pytest.mark.parametrize("change,message", [
    (dict(head_dim=96), "head_dim 96"), (dict(head_dim=32), "head_dim 32"),
    (dict(q_heads=7), "multiple of kv_heads"), (dict(q_heads=0), "multiple of kv_heads"),
    (dict(kv_heads=0), "kv_heads 0"), (dict(page_size=12), "page_size 12"),
    (dict(page_size=0), "page_size 0"), (dict(page_size=65544), "page_size 65544"),
    (dict(num_pages=0), "0 pages"), (dict(num_pages=1 << 26), "too many rows"),
    (dict(entries=0), "0 table entries"), (dict(entries=1 << 27), "too many positions"),
    (dict(batch=0), "batch 0"), (dict(window=-1), "window -1"), (dict(sinks=-1), "sinks -1"),
    (dict(scale=INF), "scale"), (dict(scale=NAN), "scale"),
])
def test_decode_refusals(change, message):
    """Refused on the host, before any CUDA call."""
    from llm_compiler_3_b200 import _native
    a = dict(DECODE_ARGS, **change)
    p = ctypes.c_void_p(1 << 20)
    rc = _native.lib().npu_b200_paged_decode(
        p, p, p, p, p, p, a["batch"], a["q_heads"], a["kv_heads"], a["head_dim"], a["num_pages"],
        a["page_size"], a["entries"], a["window"], a["sinks"], a["scale"], p, 1 << 30, None)
    assert rc == -1
    assert message.encode() in _native.lib().npu_b200_last_error()


def test_decode_refuses_pointers():
    from llm_compiler_3_b200 import _native
    a = DECODE_ARGS
    p = 1 << 20

    def call(ptrs, ws=p, ws_bytes=1 << 30):
        return _native.lib().npu_b200_paged_decode(
            *ptrs, a["batch"], a["q_heads"], a["kv_heads"], a["head_dim"], a["num_pages"],
            a["page_size"], a["entries"], 0, 0, 0.1, ws, ws_bytes, None)

    for i in range(6):
        assert call([None if j == i else p for j in range(6)]) == -1
        assert b"null" in _native.lib().npu_b200_last_error()
    for i in (0, 1, 2, 5):
        assert call([p + 8 if j == i else p for j in range(6)]) == -1
        assert b"aligned" in _native.lib().npu_b200_last_error()
    need = _native.lib().npu_b200_paged_decode_workspace_size(8, 2, 128)
    assert call([p] * 6, p, need - 1) == -1 and call([p] * 6, None, need) == -1
    assert b"workspace" in _native.lib().npu_b200_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(head_dim=100), "head_dim 100"), (dict(page_size=4), "page_size 4"),
    (dict(rows=0), "0 rows"), (dict(batch=0), "batch 0"), (dict(batch=65536), "batch 65536"),
    (dict(num_pages=0), "0 pages"), (dict(entries=0), "0 table entries"),
])
def test_append_refusals(change, message):
    from llm_compiler_3_b200 import _native
    a = dict(batch=2, kv_heads=2, rows=3, head_dim=64, num_pages=9, page_size=16, entries=4, **{})
    a.update(change)
    p = 1 << 20
    rc = _native.lib().npu_b200_paged_append(p, p, p, p, p, p, p, a["batch"], a["kv_heads"],
                                             a["rows"], a["head_dim"], a["num_pages"],
                                             a["page_size"], a["entries"], None)
    assert rc == -1
    assert message.encode() in _native.lib().npu_b200_last_error()


def test_outputs_over_inputs_are_refused():
    """On the host, before any CUDA call: the kernels read what they would overwrite."""
    from llm_compiler_3_b200 import _native
    lib = _native.lib()
    p = [(i + 1) << 28 for i in range(9)]

    def refused(rc):
        return rc == -1 and b"overlap" in lib.npu_b200_last_error()

    q_bytes = 3 * 8 * 128 * 2
    for shift in (0, 16, q_bytes - 16, 16 - q_bytes):
        assert refused(lib.npu_b200_paged_decode(*p[:5], p[0] + shift, 3, 8, 2, 128, 9, 16, 4, 0, 0, 0.1, p[6],
                                                 1 << 26, None))
        assert refused(lib.npu_b200_paged_prefill(p[0], p[1], p[2], p[3], p[4], None, p[0] + 5 * shift, 3, 8, 2, 128,
                                                  5, 9, 16, 4, 0, 0, 0.1, None))
    for k, v in ((p[2], p[1]), (p[0], p[3] + 16), (p[3], p[1]), (p[0], p[2] + 9 * 2 * 16 * 128 * 2 - 16)):
        assert refused(lib.npu_b200_paged_append(k, v, p[2], p[3], p[4], p[5], None, 3, 2, 5, 128, 9, 16, 4, None))
    for scores, done in ((p[1], p[7]), (p[3], p[2])):
        assert refused(lib.npu_b200_beam_select(p[0], 0, p[1], p[2], scores, p[4], p[5], done, 2, 4, 50, 4, 1, p[8],
                                                1 << 26, None))


def test_outputs_over_pages_are_refused():
    """An output in the pool that the call reads, or over the parents it goes by."""
    from llm_compiler_3_b200 import _native
    lib = _native.lib()
    p = [(i + 1) << 28 for i in range(7)]
    pool = 9 * 2 * 16 * 128 * 2
    for pages in p[1:3]:
        for shift in (0, 16, pool - 16):
            assert lib.npu_b200_paged_decode(*p[:5], pages + shift, 3, 8, 2, 128, 9, 16, 4, 0, 0, 0.1, p[6], 1 << 26,
                                             None) == -1
            assert b"overlap" in lib.npu_b200_last_error()
            assert lib.npu_b200_paged_prefill(*p[:5], None, pages + shift, 3, 8, 2, 128, 5, 9, 16, 4, 0, 0, 0.1,
                                              None) == -1
            assert b"overlap" in lib.npu_b200_last_error()
    for out in (p[1], p[1] + 12, p[1] - 60):
        assert lib.npu_b200_beam_reorder(p[0], p[1], out, 3, 4, 16, None) == -1
        assert b"overlap" in lib.npu_b200_last_error()


def test_operators_refuse_cpu_tensors():
    from llm_compiler_3_b200 import ops
    k, v, table = paged_cache([5], 1, 64, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_decode(seeded((1, 2, 64), 1), k, v, table, ints([5]))
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_append(seeded((1, 1, 1, 64), 1), seeded((1, 1, 1, 64), 1), k, v, table, ints([5]))


# ---- on the GPU: attention of one token ------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("page", [8, 16, 24, 32, 40, 64, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_page_sizes(cuda, page, dim):
    """Pages smaller and larger than the 32-key tile, and sizes that no tile divides."""
    lens = [1, 31, 32, 33, 0, 100, 257]
    k, v, table = paged_cache(lens, 2, dim, page, seed=page)
    check_decode(seeded((len(lens), 8, dim), 3), k, v, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (5, 5), (6, 2), (7, 1), (8, 1), (9, 1),
                                            (16, 1), (24, 2), (17, 1), (40, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_groups(cuda, heads, kv_heads, dim):
    """Any number of query heads to a key head, past one block of 8 or 16 too."""
    lens = [70, 5]
    k, v, table = paged_cache(lens, kv_heads, dim, 16, seed=heads)
    check_decode(seeded((2, heads, dim), 4), k, v, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (32, 4), (33, 32), (50, 33), (64, 100),
                                          (100, 3), (500, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_decode_window(cuda, window, sinks):
    """Windows and sinks on, inside and across tile and page borders; hidden keys may
    hold NaN, and the entries of pages without a visible key are no pages."""
    lens = [300, 64, 33, 1, 0, 129]
    k, v, table = paged_cache(lens, 2, 128, 16, seed=window % 1000 + sinks % 1000)
    shown, kk, vv = table.clone(), k.clone(), v.clone()
    for b, n in enumerate(lens):
        for j in range(n):
            if not (j > n - 1 - window or j < sinks):
                kk[table[b, j // 16], :, j % 16] = NAN
                vv[table[b, j // 16], :, j % 16] = INF
        for e in range((n + 15) // 16):
            if not any(j < n and (j > n - 1 - window or j < sinks) for j in range(e * 16, e * 16 + 16)):
                shown[b, e] = -1
    q = seeded((len(lens), 4, 128), 5)
    got = check_decode(q, kk, vv, shown, lens, window=window, sinks=sinks)
    assert torch.count_nonzero(got[4]) == 0


@pytest.mark.gpu
def test_decode_splits_and_joins(cuda):
    """One long sequence beside short and empty ones: units that span many stretches."""
    lens = [20000, 3, 0, 777]
    k, v, table = paged_cache(lens, 1, 128, 64, seed=8)
    q = seeded((4, 2, 128), 6)
    first = check_decode(q, k, v, table, lens)
    for _ in range(3):
        assert torch.equal(_decode(q, k, v, table, lens), first)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 127, 128, 129, 700])
def test_decode_batches(cuda, batch):
    """More sequences than the threads that lay the line out."""
    lens = [(7 * b) % 50 for b in range(batch)]
    lens[0] = 40
    k, v, table = paged_cache(lens, 1, 64, 8, seed=batch)
    check_decode(seeded((batch, 2, 64), 7), k, v, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,heads,kv_heads,dim", [(1, 4, 1, 64), (1, 20, 2, 128), (3, 12, 4, 64), (9, 5, 5, 128),
                                                      (18, 8, 8, 64), (40, 6, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 20)])
def test_decode_of_few_units(cuda, batch, heads, kv_heads, dim, window, sinks):
    """Units that clusters of 8, 4, 2 and single CTAs take, some of the CTAs without a tile, and the
    same sequences under tables too wide for them, over the line; each the same bits twice."""
    lens = [(i * 353 + 1) % 900 for i in range(batch)]
    lens[-1] = max(lens[-1], 777)
    k, v, table = paged_cache(lens, kv_heads, dim, 16, seed=batch)
    q = seeded((batch, heads, dim), 11)
    wide = torch.full((batch, 4096), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    for entries in (table, wide):
        got = check_decode(q, k, v, entries, lens, window=window, sinks=sinks)
        assert torch.equal(got, _decode(q, k, v, entries, lens, window=window, sinks=sinks))


@pytest.mark.gpu
def test_decode_scores_of_any_size(cuda):
    """Scores far apart, all equal, a negative scale, and -inf keys' weights."""
    lens = [200, 200]
    k, v, table = paged_cache(lens, 1, 64, 16, seed=9)
    q = seeded((2, 4, 64), 8, std=20.0)
    check_decode(q, k, v, table, lens)
    check_decode(q, k, v, table, lens, scale=-0.125)
    check_decode(q, k, v, table, lens, scale=0.0)


@pytest.mark.gpu
def test_decode_clamps_lengths_and_reports_bad_pages(cuda):
    from llm_compiler_3_b200 import _native, ops
    k, v, table = paged_cache([48, 48], 1, 64, 16, seed=10)
    q = seeded((2, 2, 64), 9)
    want = _decode(q, k, v, table, [48, 0])
    assert torch.equal(_decode(q, k, v, table, [1 << 30, -5]), want)
    dev = torch.device("cuda", 0)
    for page in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        bad = table.clone()
        bad[1, 1] = page
        out = ops.paged_decode(q.to(dev), k.to(dev), v.to(dev), bad.to(dev), ints([48, 48]).to(dev))
        with pytest.raises(_native.NpuError, match="0x8"):
            _native.device_status()
        assert torch.equal(out[0].cpu(), _decode(q, k, v, table, [48, 48])[0])


@pytest.mark.gpu
def test_decode_of_shared_pages_and_pool_slices(cuda):
    """Two rows that name the same pages, in slices of one pool of several layers."""
    k, v, table = paged_cache([40], 2, 64, 16, seed=11)
    pool = torch.stack([torch.zeros_like(k), k, v, torch.zeros_like(k)]).cuda()
    rows = table.repeat(2, 1)
    q = seeded((2, 4, 64), 10)
    want = check_decode(q, k, v, rows, [40, 33])
    assert torch.equal(_decode(q, pool[1], pool[2], rows, [40, 33]), want)


@pytest.mark.gpu
def test_decode_on_streams_and_in_graphs(cuda):
    """Calls in flight on two streams, and two captured graphs replayed at once: each
    has scratch of its own.  A replay follows the lengths it finds."""
    from llm_compiler_3_b200 import ops
    lens = [3000, 3000]
    k, v, table = (t.cuda() for t in paged_cache(lens, 1, 128, 16, seed=12))
    qs = [seeded((2, 8, 128), 20 + i).cuda() for i in range(2)]
    n = ints(lens).cuda()
    want = [ops.paged_decode(q, k, v, table, n) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_decode(qs[i], k, v, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for q, g in zip(qs, graphs):
        with torch.cuda.graph(g):
            outs.append(ops.paged_decode(q, k, v, table, n))
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    n.copy_(ints([17, 0]))
    later = ops.paged_decode(qs[0], k, v, table, n)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], later) and torch.count_nonzero(later[1]) == 0


@pytest.mark.gpu
def test_decode_checks_of_the_wrapper(cuda):
    from llm_compiler_3_b200 import ops
    k, v, table = (t.cuda() for t in paged_cache([20, 20], 2, 64, 16))
    q, n = seeded((2, 4, 64), 1).cuda(), ints([20, 20]).cuda()
    bad = [dict(q=q.float()), dict(q=q[:, :, ::2]), dict(q=q[:1]), dict(seq_lens=n[:1]), dict(seq_lens=n.long()),
           dict(page_table=table.long()), dict(page_table=table[:1]), dict(v_pages=v[:1]),
           dict(k_pages=k.transpose(1, 2)), dict(out=torch.empty_like(q)[:1]), dict(out=torch.empty_like(q).float()),
           dict(seq_lens=n.cpu())]
    good = dict(q=q, k_pages=k, v_pages=v, page_table=table, seq_lens=n)
    for change in bad:
        with pytest.raises(ValueError):
            ops.paged_decode(**dict(good, **change))
    out = torch.empty_like(q)
    assert ops.paged_decode(**good, out=out) is out


# ---- on the GPU: the append ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dim,page,rows,lens", [(64, 8, 1, None), (128, 16, 1, [1, 0, 1]),
                                                (64, 24, 50, [50, 0, 13]), (128, 32, 33, None)])
def test_append(cuda, dim, page, rows, lens):
    """Rows that begin inside a page and run over several; every other row stays."""
    from llm_compiler_3_b200 import _native, ops
    starts = [0, 5, page]
    k, v, table = paged_cache([s + rows for s in starts], 2, dim, page, seed=rows)
    new_k, new_v = seeded((3, 2, rows, dim), 1), seeded((3, 2, rows, dim), 2)
    kg, vg = k.cuda(), v.cuda()
    ops.paged_append(new_k.cuda(), new_v.cuda(), kg, vg, table.cuda(), ints(starts).cuda(),
                     None if lens is None else ints(lens).cuda())
    assert _native.device_status() == 0
    for got, new, old in ((kg, new_k, k), (vg, new_v, v)):
        want = oracle.append_paged(new, old, table, starts, lens)
        assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))


@pytest.mark.gpu
def test_append_drops_rows_without_a_page(cuda):
    from llm_compiler_3_b200 import _native, ops
    k, v, table = paged_cache([32, 32], 1, 64, 16, seed=3)
    table[1, 1] = -1
    new = seeded((2, 1, 20, 64), 4)
    starts = [-3, 10]  # positions -3..-1 and 16..29 of sequence 1 have none
    kg, vg = k.cuda(), v.cuda()
    ops.paged_append(new.cuda(), new.cuda(), kg, vg, table.cuda(), ints(starts).cuda())
    with pytest.raises(_native.NpuError, match="0x8"):
        _native.device_status()
    want = oracle.append_paged(new, k, table, starts)
    assert torch.equal(kg.cpu().view(torch.int16), want.view(torch.int16))


@pytest.mark.gpu
def test_calls_from_threads_and_streams(cuda):
    """Two host threads, each with a stream of its own, at once."""
    import threading
    from llm_compiler_3_b200 import ops
    lens = [900, 300]
    k, v, table = (t.cuda() for t in paged_cache(lens, 2, 64, 32, seed=14))
    n, qs = ints(lens).cuda(), [seeded((2, 8, 64), 70 + i).cuda() for i in range(2)]
    want = [ops.paged_decode(q, k, v, table, n) for q in qs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [ops.paged_decode(qs[i], k, v, table, n) for _ in range(200)]
            torch.cuda.current_stream().synchronize()
            bad.extend(1 for g in got if not torch.equal(g, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.gpu
@pytest.mark.parametrize("dim,heads,kv_heads,lens,window", [
    (128, 2, 1, [60000, 5, 0, 9000], 0), (64, 3, 1, [50000, 20000], 0), (64, 9, 1, [30000, 1], 0),
    (128, 16, 1, [20000, 300, 7000], 0), (64, 2, 2, [1000, 0, 31, 400], 0), (128, 1, 1, [3], 0),
    (64, 2, 1, [40000, 39000, 12], 9000)])
def test_decode_of_wide_tables(cuda, dim, heads, kv_heads, lens, window):
    """Tables with room for many more keys than there are: part of the work is dealt out
    on the way, whatever there turns out to be.  The same bits each time."""
    k, v, table = paged_cache(lens, kv_heads, dim, 16, seed=len(lens))
    wide = torch.full((len(lens), 80000), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    q = seeded((len(lens), heads, dim), 12)
    kw = dict(window=window, sinks=3) if window else {}
    if window:  # a window narrows what a table can hold: widen it in sequences instead
        wide, q = wide.repeat(60, 1), q.repeat(60, 1, 1)
        lens = lens * 60
    first = _decode(q, k, v, wide, lens, **kw)
    n = 3 if window else len(lens)
    want, bound = oracle.attention_paged(q[:n, :, None], k, v, wide[:n], lens[:n],
                                         q_lens=[min(1, x) for x in lens[:n]], **kw)
    check(first[:n], want[:, :, 0], bound[:, :, 0])
    if window:
        # Every copy of a sequence is split at other places: near, not equal.
        for c in range(1, 60):
            check(first[3 * c:3 * c + 3], want[:, :, 0], bound[:, :, 0])
    for _ in range(5):
        assert torch.equal(_decode(q, k, v, wide, lens, **kw), first)


def check_with_nan(got, want, bound):
    """NaN exactly where the definition has it; the rest within its bound."""
    odd = want.isnan()
    assert odd.any() and torch.equal(got.isnan(), odd)
    check(torch.where(odd, 0, got), torch.where(odd, 0, want), torch.where(odd, 0, bound))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,heads,kv_heads,copies,reach", [
    (128, 4, 1, 1, 1000),   # clusters of 8 CTAs
    (64, 4, 1, 1, 2100),
    (64, 20, 2, 1, 2100),
    (128, 4, 1, 4, 1000),   # of 4
    (128, 4, 1, 9, 1000),   # of 2
    (128, 4, 1, 20, 1000),  # one CTA to a unit
    (64, 4, 1, 1, 80000),   # the line of tiles
    (128, 4, 1, 20, 80000),
])
def test_decode_of_queries_and_keys_that_are_no_numbers(cuda, dim, heads, kv_heads, copies, reach):
    """NaN in a query, in the newest key alone in its tile (and in its CTA's share), in every key of a
    tile, in one key among others: the rows that see it are NaN, whoever joins their parts."""
    lens = [225, 225, 225, 225, 33] * copies
    k, v, table = paged_cache(lens, kv_heads, dim, 16, seed=dim + copies)
    wide = torch.full((len(lens), (reach + 15) // 16), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    q = seeded((len(lens), heads, dim), 13)
    for c in range(0, len(lens), 5):
        q[c, 1, 5] = NAN
        for row, keys in ((c + 1, [224]), (c + 2, range(64, 96)), (c + 3, [100])):
            for j in keys:
                k[int(wide[row, j // 16]), kv_heads - 1, j % 16, 7] = NAN
    got = _decode(q, k, v, wide, lens)
    want, bound = oracle.attention_paged(q[:, :, None], k, v, wide, lens, q_lens=[1] * len(lens))
    check_with_nan(got, want[:, :, 0], bound[:, :, 0])


def far_below(dim, page, n):
    """(q [1, 2, D], k, v, table): one key whose weight is 2^25 times that of each of the others, whose
    values alone are not 0."""
    k, v, table = paged_cache([n], 1, dim, page, seed=n)
    for j in range(n):
        at = int(table[0, j // page]), 0, j % page
        k[at], v[at] = 0.0, 64.0
    k[int(table[0, 0]), 0, 0] = 17.68 / dim
    v[int(table[0, 0]), 0, 0] = 0.0
    return torch.ones(1, 2, dim).half(), k, v, table


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,reach", [(20, 20), (900, 900), (3000, 80000)])
def test_decode_keeps_weights_far_below_the_largest(cuda, dim, n, reach):
    """Weights of 2^-25 of the largest: each is rounded by 2^-11 of itself (2^-32 of the largest), like
    the output (by 2^-25 at least), and the sums by less than 2^-11 together."""
    q, k, v, table = far_below(dim, 16, n)
    wide = torch.full((1, (reach + 15) // 16), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    got = _decode(q, k, v, wide, [n], scale=1.0)
    want, _ = oracle.attention_paged(q[:, :, None], k, v, wide, [n], [1], scale=1.0)
    bound = 3 * 2.0 ** -11 * want + 2.0 ** -25 + 64 * n * 2.0 ** -32
    check(got, want[:, :, 0], bound[:, :, 0])


def steep(dim, page, n, base):
    """(q [1, 2, D], k, v, table): scores of `base` and up to 40 more, rising and falling, and values of 1,
    so that attention is 1 whatever the weights are."""
    k, v, table = paged_cache([n], 1, dim, page, seed=n)
    r = torch.Generator().manual_seed(n)
    step = torch.rand(n, generator=r) * 40
    step[:n // 3] = torch.linspace(0, 40, n // 3)
    q = torch.zeros(1, 2, dim).half()
    q[..., 0] = 2.0 ** (base // 2)
    q[..., 1] = 1.0
    for j in range(n):
        at = int(table[0, j // page]), 0, j % page
        k[at], v[at] = 0.0, 1.0
        k[at][0], k[at][1] = 2.0 ** (base - base // 2), step[j]
    return q, k, v, table


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("base", [0, 10, 20, 23, 24, 25, 26])
def test_decode_of_steep_and_large_scores(cuda, dim, base):
    """No weight passes FP16's range, however large the scores and their steps: the output is the sum of
    rounded weights over the sum of the weights, 2^-11 and the output's own rounding off 1."""
    for n, scale in ((300, 1.0), (700, -1.0), (5000, 1.0)):
        q, k, v, table = steep(dim, 16, n, base)
        got = _decode(q * scale, k, v, table, [n], scale=scale)
        assert float((got.double() - 1).abs().max()) <= 2.0 ** -10 + n * 2.0 ** -23
