"""Page tables of the next step, compaction and page copies: whole numbers, compared
exactly with the row-by-row oracle (oracle/paged.py)."""
import random

import pytest
import torch

import oracle
from conftest import seeded


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def beams(seed, groups, width, longest, page, pages, entries, shared=True):
    """(table, lens, refs): rows of `groups` prompts whose beams share full pages."""
    r = random.Random(seed)
    free = r.sample(range(pages), pages)
    refs = [0] * pages
    table, lens = [], []
    for _ in range(groups):
        n = r.randint(0, longest)
        common = [free.pop() for _ in range(r.randint(0, n // page) if shared else 0)]
        for _ in range(width):
            row = common + [free.pop() for _ in range(-(-n // page) - len(common))]
            for p in row:
                refs[p] += 1
            table.append(row + [-1] * (entries - len(row)))
            lens.append(n)
    for _ in range(r.randint(0, len(free) // 2)):  # pages that another table holds
        refs[free.pop()] = r.randint(1, 3)
    return table, lens, refs


# ---- on the CPU ------------------------------------------------------------------------------
def test_oracle_update_by_hand():
    """Row 0 (6 tokens, pages 4 and 1 of 4) forks into rows 0 and 2; row 1 is freed; a new
    prompt of 5 tokens comes in: the lowest free pages, the copy's first."""
    table, lens, refs, copies, info = oracle.page_update(
        [[4, 1, -1], [0, -1, -1]], [6, 2], [0, -1, 0], [9, 5, 7], [1, 1, 0, 0, 1, 2], 4)
    assert table == [[4, 1, 0], [2, 3, -1], [4, -1, -1]]
    assert lens == [6, 0, 6] and info == [0, 1, 0] and refs == [1, 1, 1, 1, 2, 2]
    table, lens, refs, copies, info = oracle.page_update(
        [[4, 1, -1], [0, -1, -1]], [6, 2], [0, 0], [6, 9], [1, 1, 0, 0, 1, 2], 4)
    assert table == [[4, 1, -1], [4, 0, 2]] and copies == [[1, -1], [0, -1]] and info == [1, 0, 1]
    assert refs == [1, 1, 1, 0, 2, 2]


def test_oracle_compact_by_hand():
    table, refs, moves, index, info = oracle.page_compact([[5, 1, -1], [3, 9, 2]], [0, 2, 0, 1, 0, 1])
    assert info == [3, 2] and moves == [[3, 5, -1], [0, 2, -1]]
    assert table == [[2, 1, -1], [0, -1, -1]] and refs == [1, 2, 1, 0, 0, 0]
    assert index == [-1, 1, -1, 0, -1, 2]


def test_oracle_pages_to_copy_from_are_not_handed_out():
    """Rows 0 and 1 share page 0 and rows 2 and 3 page 1, rolled back to 5 of 8 tokens: every
    child copies, nobody holds pages 0 and 1 any more, and they are free after the step only."""
    table, lens, refs, copies, info = oracle.page_update(
        [[0], [0], [1], [1]], [5, 5, 5, 5], [2, 3, 0, 1], [6, 6, 6, 6], [2, 2, 0, 0, 0, 0, 0], 8)
    assert table == [[2], [3], [4], [5]] and copies == [[1, 1, 0, 0], [2, 3, 4, 5]]
    assert refs == [0, 0, 1, 1, 1, 1, 0] and info == [3, 0, 4]


def test_clusters_have_started_before_their_shared_memory_is_written():
    """By reading: a CTA of a cluster may start after another has counted, so each kernel passes a
    cluster barrier before its first write to the others."""
    from llm_compiler_3_b200 import build
    kernels = (build.CSRC / "pages.cu").read_text().split("__global__")[1:]
    writes = [k for k in kernels if "cluster_share(" in k]
    assert len(writes) == 2
    for k in writes:
        before = k[:k.index("cluster_share(")]
        assert "cluster_wait();" in before or "cluster_sync_all();" in before


@pytest.mark.parametrize("change,message", [
    (dict(rows=0), "0 rows"), (dict(rows=8193), "8193 rows"), (dict(new_rows=0), "to 0"),
    (dict(new_rows=8193), "to 8193"), (dict(entries=0), "0 table entries"), (dict(page=12), "page_size 12"),
    (dict(pages=0), "0 pages"), (dict(entries=1 << 27), "positions"),
])
def test_update_refusals(change, message):
    from llm_compiler_3_b200 import _native
    a = dict(rows=2, new_rows=2, entries=4, page=16, pages=8, **{})
    a.update(change)
    p = [(i + 1) << 24 for i in range(10)]
    lib = _native.lib()
    assert lib.npu_b200_page_update(*p, a["rows"], a["new_rows"], a["entries"], a["page"], a["pages"], None) == -1
    assert message.encode() in lib.npu_b200_last_error()


def test_refusals_of_pointers():
    from llm_compiler_3_b200 import _native
    lib = _native.lib()
    p = [(i + 1) << 24 for i in range(10)]
    for i in range(10):
        assert lib.npu_b200_page_update(*p[:i], None, *p[i + 1:], 2, 2, 4, 16, 8, None) == -1
        assert b"null" in lib.npu_b200_last_error()
    for i, j in ((5, 0), (6, 1), (7, 4)):  # a result over the input it comes from
        q = list(p)
        q[i] = p[j] + 4
        assert lib.npu_b200_page_update(*q, 2, 2, 4, 16, 8, None) == -1
        assert b"overlap" in lib.npu_b200_last_error()
    for i in range(7):
        assert lib.npu_b200_page_compact(*p[:i], None, *p[i + 1:7], 2, 4, 8, None) == -1
        assert b"null" in lib.npu_b200_last_error()
    for i, j in ((2, 0), (3, 1)):
        q = list(p)
        q[i] = p[j]
        assert lib.npu_b200_page_compact(*q[:7], 2, 4, 8, None) == -1
        assert b"overlap" in lib.npu_b200_last_error()
    assert lib.npu_b200_page_compact(*p[:7], 0, 4, 8, None) == -1
    assert lib.npu_b200_page_compact(*p[:7], 2, 4, 0, None) == -1
    for args in ((None, p[0], None, 1, 1, 1, 16), (p[0], None, None, 1, 1, 1, 16),
                 (p[0], p[1], None, 0, 1, 1, 16), (p[0], p[1], None, 1, 0, 1, 16),
                 (p[0], p[1], None, 1, 1, 0, 16), (p[0], p[1], None, 1, 1, 1, 24),
                 (p[0], p[1], None, 1, 1, 1, 0), (p[0] + 8, p[1], None, 1, 1, 1, 16)):
        assert lib.npu_b200_page_copy(*args, None) == -1


# ---- on the GPU ------------------------------------------------------------------------------
def run_update(table, lens, parents, capacity, refs, page):
    from llm_compiler_3_b200 import ops
    got = ops.page_update(ints(table).cuda(), ints(lens).cuda(), ints(parents).cuda(),
                          ints(capacity).cuda(), ints(refs).cuda(), page)
    return [g.cpu().tolist() for g in got]


def check_update(*args):
    got, want = run_update(*args), oracle.page_update(*args)
    for name, g, w in zip(("table", "lens", "refs", "copies", "info"), got, want):
        assert g == w, name
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("page", [8, 24, 64])
def test_update_of_beams(cuda, seed, page):
    """Random beams: forks, frees, growth, admissions; what the pool holds may run short."""
    r = random.Random(100 * seed + page)
    groups, width, longest = r.randint(1, 6), r.randint(1, 5), r.choice([5, 60, 300])
    entries = -(-longest // page) + r.randint(1, 3)
    pages = groups * width * entries + r.randint(1, 40)
    table, lens, refs = beams(seed, groups, width, longest, page, pages, entries)
    rows = groups * width
    parents = [r.choice([-1, r.randrange(rows), r.randrange(rows)]) for _ in range(r.randint(1, 2 * rows))]
    capacity = [r.randint(0, entries * page + 20) if q < 0 else lens[q] + r.choice([0, 1, 1, page]) for q in parents]
    check_update(table, lens, parents, capacity, refs, page)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(8))
def test_update_of_rows_rolled_back(cuda, seed):
    """Rows cut back into pages that others share, with and without holds outside the table: each
    child copies, and no page is copied from and to in one step."""
    r = random.Random(seed)
    page, groups, width = r.choice([8, 16]), r.randint(2, 5), r.randint(2, 4)
    table, _, refs, pages = [], [], [], groups * (1 + width) + 6
    for g in range(groups):
        table += [[2 * g, 2 * g + 1, -1]] * width
        refs += [width, width + r.choice([0, 0, 1])]
    refs += [0] * (pages + width * groups)
    rows = groups * width
    lens = [r.choice([page + 1, page + r.randrange(1, page), 3, page]) for _ in range(rows)]
    parents = [r.randrange(rows) for _ in range(rows)]
    got = check_update(table, lens, parents, [lens[q] + 1 for q in parents], refs, page)
    n = got[4][2]
    assert not set(got[3][0][:n]) & set(got[3][1][:n]) and got[4][1] == 0


@pytest.mark.gpu
def test_update_identity_and_free(cuda):
    table, lens, refs = beams(3, 4, 3, 100, 16, 200, 9)
    rows = list(range(12))
    got = check_update(table, lens, rows, lens, refs, 16)
    assert got[0] == table and got[2] == refs and got[4][1:] == [0, 0]
    got = check_update(table, lens, [-1], [0], refs, 16)  # every row freed
    held = {p for row in table for p in row if p >= 0}
    assert all(got[2][p] == 0 for p in held)


@pytest.mark.gpu
def test_update_corner_rows(cuda):
    """Parents that are no rows, lengths and capacities out of range, entries that are no
    pages, a partly filled page that another table holds too, negative counts."""
    table = [[0, 1, -1, -1], [7, 99, 2, -1], [3, -1, 4, 5], [6, 8, -1, -1]]
    lens = [12, 24, 1 << 30, -4]
    refs = [1, 2, 1, 1, 1, 1, 1, 1, -3, 0, 0, 5]
    parents = [0, 0, 1, 2, 3, 4, -7, 1]
    capacity = [12, 13, 1 << 30, 0, 9, 8, -1, 24]
    check_update(table, lens, parents, capacity, refs, 8)
    check_update([[-1]], [0], [0], [0], [0], 8)
    check_update([[-1]], [0], [0], [8], [0], 8)
    check_update([[0]], [8], [0, 0], [8, 8], [1], 8)


@pytest.mark.gpu
def test_update_of_many_rows_and_pages(cuda):
    """Thousands of rows, more pages than the cluster has threads, few rows of long tables."""
    table, lens, refs = beams(5, 800, 4, 40, 8, 40000, 7)
    r = random.Random(1)
    parents = [r.randrange(3200) for _ in range(3200)]
    check_update(table, lens, parents, [lens[q] + 1 for q in parents], refs, 8)
    table, lens, refs = beams(6, 1, 2, 30000, 8, 70000, 4000)
    check_update(table, lens, [1, 0, 0], [lens[0] + 1] * 3, refs, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("pages,live,rows", [(1, 0, 1), (1, 1, 1), (2, 1, 1), (37, 20, 3), (64, 64, 2),
                                             (300, 0, 2), (5000, 2500, 40), (40001, 30000, 9)])
def test_compact(cuda, pages, live, rows):
    from llm_compiler_3_b200 import ops
    r = random.Random(pages + live)
    refs = [0] * pages
    for p in r.sample(range(pages), live):
        refs[p] = r.randint(1, 4)
    if pages == 300:
        refs[7] = -2
    table = [[r.randint(-2, pages + 1) for _ in range(11)] for _ in range(rows)]
    got = [g.cpu().tolist() for g in ops.page_compact(ints(table).cuda(), ints(refs).cuda())]
    for name, g, w in zip(("table", "refs", "moves", "index", "info"), got, oracle.page_compact(table, refs)):
        assert g == w, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,page", [(torch.float16, (3, 16, 64)), (torch.uint8, (16,)),
                                        (torch.float32, (1028,)), (torch.float16, (8, 16, 200))])
def test_copy(cuda, dtype, page):
    """Every slab's pages, bit for bit; skipped, counted and refused pairs."""
    from llm_compiler_3_b200 import _native, ops
    pool = seeded((3, 11, *page), 4, std=50.0).to(dtype)
    pages = [[0, 5, -1, 10, 2], [1, 7, -1, 3, 9]]
    for count in (None, 4, 0, 99, -3):
        got = pool.cuda()
        ops.page_copy(got, ints(pages).cuda(), None if count is None else ints([count]).cuda())
        assert _native.device_status() == 0
        want = oracle.page_copy(pool, pages, count)
        assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))
    got = pool.cuda()
    ops.page_copy(got, ints([[0, 11, 3, -1], [1, 2, -5, 4]]).cuda())
    with pytest.raises(_native.NpuError, match="0x8"):
        _native.device_status()
    want = oracle.page_copy(pool, [[0], [1]])
    assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.gpu
def test_wrapper_checks(cuda):
    from llm_compiler_3_b200 import ops
    table, lens, refs = (ints(x).cuda() for x in beams(1, 2, 2, 30, 8, 40, 6))
    rows = ints([0, 1]).cuda()
    for args in ((table.long(), lens, rows, rows, refs), (table, lens[:2], rows, rows, refs),
                 (table, lens, rows, rows[:1], refs), (table, lens, rows, rows, refs.float()),
                 (table[:, ::2], lens, rows, rows, refs), (table, lens.cpu(), rows, rows, refs)):
        with pytest.raises(ValueError):
            ops.page_update(*args, 8)
    pool = torch.zeros(2, 40, 16, device="cuda")
    pages = ints([[0], [1]]).cuda()
    for args in ((pool[:, ::2], pages), (pool[0], pages), (pool, pages[:1]), (pool, pages, rows[:0]),
                 (pool, pages, rows.long())):
        with pytest.raises(ValueError):
            ops.page_copy(*args)


@pytest.mark.gpu
def test_update_and_copy_in_a_graph(cuda):
    """A captured step follows the tables it finds."""
    from llm_compiler_3_b200 import ops
    table, lens, refs = beams(8, 3, 4, 100, 16, 150, 8)
    state = [ints(x).cuda() for x in (table, lens, list(range(12)), lens, refs)]
    pool = seeded((2, 150, 16, 8), 3).cuda()
    ops.page_update(*state, 16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.page_update(*state, 16)
        ops.page_copy(pool, got[3], got[4][2:])
    r = random.Random(2)
    for _ in range(3):
        parents = [r.randrange(12) for _ in range(12)]
        capacity = [lens[p] + 1 for p in parents]
        state[2].copy_(ints(parents))
        state[3].copy_(ints(capacity))
        before = pool.cpu()
        graph.replay()
        torch.cuda.synchronize()
        want = oracle.page_update(table, lens, parents, capacity, refs, 16)
        for g, w in zip(got, want):
            assert g.cpu().tolist() == w
        assert torch.equal(pool.cpu(), oracle.page_copy(before, want[3], want[4][2]))


@pytest.mark.gpu
def test_compactions_beside_other_work(cuda):
    """Many compactions in a row while another stream keeps the SMs busy, so that a cluster's CTAs
    start apart: the same results each time."""
    from llm_compiler_3_b200 import ops
    r = random.Random(9)
    refs = [r.choice([0, 0, 1, 2]) for _ in range(3000)]
    table = [[r.randint(-1, 2999) for _ in range(40)] for _ in range(20)]
    state = ints(table).cuda(), ints(refs).cuda()
    pool = torch.zeros(2, 4000, 8192, dtype=torch.float16, device="cuda")
    pages = torch.stack([torch.arange(2000), torch.arange(2000, 4000)]).int().cuda()
    busy, got = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for _ in range(50):
        with torch.cuda.stream(busy):
            ops.page_copy(pool, pages)
        got.append(ops.page_compact(*state))
    torch.cuda.synchronize()
    want = [ints(w) for w in oracle.page_compact(table, refs)]
    for g in got:
        assert all(torch.equal(x.cpu(), w) for x, w in zip(g, want))
