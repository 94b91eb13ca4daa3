"""Beam search's selection and the reordering of states, against the 64-bit oracle.

How near two candidates may be before the kernel may take the other: M and x - M are
exact or rounded once in FP32; each exponential is off by at most 2^-22 and by its
argument's rounding, |x - M| log2 e 2^-24 (ln 2 of it), which is weighted by the
exponential itself: y 2^-y 2^-24 < 2^-24.  The FP32 sums of a warp's stretch add at
most 64 terms' roundings in a chain (2^-24 each: 2^-18), so ln S is off by less than
2^-17.  The rest is FP64.  Scores come back rounded to FP32."""
import pytest
import torch

import oracle
from conftest import seeded

NEAR = 2.0 ** -17
INF, NAN = float("inf"), float("nan")


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def _select(logits, scores, width, done=None, eos=-1):
    from llm_compiler_3_b200 import _native, ops
    got = ops.beam_select(logits.cuda(), scores.cuda(), width, None if done is None else done.cuda(), eos)
    torch.cuda.synchronize()
    assert _native.device_status() == 0
    return [g.cpu() for g in got]


def check(logits, scores, width, done=None, eos=-1):
    """Every chosen candidate is worth what the oracle's of that rank is, within NEAR, and is
    the oracle's own wherever its neighbours are further than that."""
    got = _select(logits, scores, width, done, eos)
    want = oracle.beam_select(logits, scores, width, done, eos)
    worth = oracle.beam_worths(logits, scores, done, eos)
    batch, beams, vocab = logits.shape
    ranked = worth.sort(-1, descending=True).values
    for b in range(batch):
        chosen = set()
        for k in range(width):
            if want[0][b, k] == -INF:
                assert got[0][b, k] == -INF and int(got[1][b, k]) == -1 and int(got[2][b, k]) == -1
                assert not bool(got[3][b, k])
                continue
            token, parent = int(got[1][b, k]), int(got[2][b, k])
            assert 0 <= parent - b * beams < beams and 0 <= token < vocab
            at = (parent - b * beams) * vocab + token
            assert at not in chosen
            chosen.add(at)
            size = 2.0 ** -23 * (1 + abs(float(want[0][b, k])))
            assert abs(float(worth[b, at] - want[0][b, k])) <= 2 * NEAR
            assert abs(float(got[0][b, k].double() - worth[b, at])) <= NEAR + size
            gaps = [abs(float(ranked[b, j] - ranked[b, k])) for j in (k - 1, k + 1) if 0 <= j < ranked.shape[1]]
            if all(g > 2 * NEAR or g == 0 for g in gaps):
                assert (token, parent) == (int(want[1][b, k]), int(want[2][b, k]))
                assert bool(got[3][b, k]) == bool(want[3][b, k])
    return got


# ---- on the CPU ------------------------------------------------------------------------------
def test_oracle_by_hand():
    logits = torch.tensor([[[0.0, 0.0, -INF], [1.0, 0.0, NAN]]])
    scores = torch.tensor([[-1.0, -1.5]])
    s, t, p, d = oracle.beam_select(logits, scores, 4)
    assert t.tolist() == [[0, 1, 0, 1]] and p.tolist() == [[0, 0, 1, 1]]
    torch.testing.assert_close(s[0, 0], torch.tensor(-1 - 0.6931471805599453, dtype=torch.float64))
    s, t, p, d = oracle.beam_select(logits, scores, 3, torch.tensor([[True, False]]), 2)
    assert t.tolist() == [[2, 0, 1]] and p.tolist() == [[0, 1, 1]] and d.tolist() == [[True, False, False]]


@pytest.mark.parametrize("change,message", [
    (dict(beams=0), "beams 0"), (dict(beams=33), "beams 33"), (dict(width=0), "width 0"),
    (dict(width=33), "width 33"), (dict(vocab=0), "vocab 0"), (dict(vocab=(1 << 26) + 1), "vocab"),
    (dict(batch=0), "batch 0"), (dict(batch=20000), "batch 20000"), (dict(eos=50), "end token"),
    (dict(eos=-2), "end token"), (dict(eos=-1), "finished beams"),
])
def test_refusals(change, message):
    from llm_compiler_3_b200 import _native
    lib = _native.lib()
    a = dict(batch=2, beams=4, vocab=50, width=4, eos=1)
    a.update(change)
    p = 1 << 24

    def call(logits=p, scores=p, ws=p, ws_bytes=1 << 30):
        return lib.npu_b200_beam_select(logits, 0, scores, p, p, p, p, p, a["batch"], a["beams"],
                                        a["vocab"], a["width"], a["eos"], ws, ws_bytes, None)

    assert call() == -1
    assert message.encode() in lib.npu_b200_last_error()
    a.update(dict(batch=2, beams=4, vocab=50, width=4, eos=1))
    for kw in (dict(logits=None), dict(scores=None), dict(ws=None), dict(ws_bytes=8), dict(logits=p + 8), dict(ws=p + 8)):
        assert call(**kw) == -1


def test_reorder_refusals():
    from llm_compiler_3_b200 import _native
    lib = _native.lib()
    p, q, r = 1 << 24, 1 << 25, 1 << 26
    for args in ((None, q, r, 2, 2, 16), (p, None, r, 2, 2, 16), (p, q, None, 2, 2, 16), (p, q, r, 0, 2, 16),
                 (p, q, r, 2, 0, 16), (p, q, r, 2, 2, 0), (p, q, p, 2, 2, 16), (p, q, p + 16, 2, 2, 16)):
        assert lib.npu_b200_beam_reorder(*args, None) == -1


# ---- on the GPU ------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("batch,beams,vocab,width", [
    (1, 1, 1, 1), (1, 1, 1, 4), (2, 3, 2, 32), (1, 4, 7, 4), (3, 2, 8, 5), (2, 5, 255, 5), (1, 32, 513, 32),
    (3, 4, 1001, 8), (2, 3, 8191, 6), (1, 2, 8193, 16), (1, 1, 50257, 1), (2, 8, 32000, 8), (40, 3, 999, 3)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_select(cuda, batch, beams, vocab, width, dtype):
    """Vocabularies around a lane's, a warp's and a stretch's share, rows off every alignment."""
    logits = (seeded((batch, beams, vocab), vocab + width, std=3.0).float()
              + 0.001 * seeded((batch, beams, vocab), 5).float()).to(dtype)
    scores = -3 * torch.rand(batch, beams, generator=torch.Generator().manual_seed(width))
    check(logits, scores, width)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("finished", [False, True])
def test_select_of_many_rows(cuda, dtype, finished):
    """More rows than three CTAs an SM hold at once, with and without finished beams."""
    logits = seeded((151, 4, 1300), 31, std=3.0).to(dtype)
    scores = -3 * torch.rand(151, 4, generator=torch.Generator().manual_seed(7))
    done = torch.rand(151, 4, generator=torch.Generator().manual_seed(8)) < 0.3
    check(logits, scores, 4, *((done, 17) if finished else ()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_ties_go_to_the_lowest_index(cuda, dtype):
    """All logits equal, in one and in several beams; steps of equal values."""
    logits = torch.zeros(2, 3, 9001, dtype=dtype)
    scores = torch.tensor([[0.0, 0.0, 0.0], [-1.0, 0.0, -1.0]])
    got = _select(logits, scores, 8)
    assert got[1].tolist() == [list(range(8))] * 2 and got[2].tolist() == [[0] * 8, [4] * 8]
    logits = (torch.arange(9001) % 100 / 8).to(dtype).expand(1, 2, -1).contiguous()
    got = _select(logits, torch.zeros(1, 2), 32)
    assert got[1].tolist() == [list(range(99, 3300, 100))[:32]] and got[2].tolist() == [[0] * 32]
    logits[0, 1, 5] = 13.0  # the second beam's best token, and so a larger sum: all its others fall behind
    got = _select(logits, torch.tensor([[0.0, 0.5]]), 3)
    assert got[1][0, 0] == 5 and got[2][0, 0] == 1


@pytest.mark.gpu
@pytest.mark.parametrize("order", [1, -1])
def test_sorted_logits(cuda, order):
    """Rising logits: every word passes the kept ones; falling: none after the first."""
    x = torch.arange(20000).float() * 1e-3
    logits = (x if order > 0 else x.flip(0)).expand(1, 2, -1).contiguous()
    check(logits, torch.tensor([[0.0, -0.00037]]), 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_masked_and_special_logits(cuda, dtype):
    """Banned tokens, whole rows banned, NaN, infinities, beams that are out, fewer
    candidates than the width."""
    logits = seeded((4, 3, 700), 3, std=2.0).to(dtype)
    logits[0, :, ::2] = -INF
    logits[0, 1] = -INF
    logits[1, :, 3:] = -INF          # 9 candidates in all
    logits[2, 0, 10] = NAN
    logits[2, 1, 20:23] = INF
    logits[2, 2, 5] = -torch.finfo(dtype).max
    logits[3] = -INF
    scores = -torch.rand(4, 3, generator=torch.Generator().manual_seed(1))
    check(logits, scores, 12)
    scores[0, 0], scores[1, 1], scores[2, 2] = -INF, NAN, -1e9
    check(logits, scores, 12)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_masked_with_the_lowest_number(cuda, dtype):
    """A mask of the type's lowest value leaves its tokens equal candidates: over a whole row, over
    all but a few tokens, over the rest of a row of -inf, over one stretch of a longer row."""
    low = torch.finfo(dtype).min
    logits = seeded((5, 2, 20000), 8, std=2.0).to(dtype)
    logits[0] = low
    logits[1, 0] = low
    logits[1, 1, 300:] = low
    logits[2] = -INF
    logits[2, :, 5:9] = low
    logits[3, :, 3000:9000] = low
    logits[4, 0, :19999] = low
    check(logits, -torch.rand(5, 2, generator=torch.Generator().manual_seed(3)), 7)
    check(logits[:, :, :50].contiguous(), torch.zeros(5, 2), 7)


@pytest.mark.gpu
def test_largest_logits(cuda):
    """Differences up to the type's range, and -1e9 as the scores of a first step's copies."""
    logits = seeded((2, 4, 3001), 9).float() * 1e37
    check(logits, torch.tensor([[0.0, -1e9, -1e9, -1e9], [-5.0, -5.0, -6.0, -7.0]]), 4)
    check(seeded((2, 4, 3001), 10, std=2.0).float(), torch.tensor([[0.0, -1e9, -1e9, -1e9]] * 2), 4)


@pytest.mark.gpu
def test_finished_beams(cuda):
    logits = seeded((5, 4, 1500), 21, std=3.0)
    scores = -4 * torch.rand(5, 4, generator=torch.Generator().manual_seed(4))
    done = torch.rand(5, 4, generator=torch.Generator().manual_seed(5)) < 0.5
    done[0], done[1] = True, False
    logits[2, :, 7] = 30.0  # the end token wins
    check(logits, scores, 6, done, 7)
    got = check(logits[:1], scores[:1], 6, done[:1], 7)
    assert got[1].tolist() == [[7, 7, 7, 7, -1, -1]] and got[3].tolist() == [[True] * 4 + [False] * 2]
    check(logits, scores, 6, None, 7)


@pytest.mark.gpu
def test_large_batch_is_its_rows(cuda):
    """A batch over a large vocabulary: the same bits as its sequences alone, each time."""
    logits = seeded((24, 4, 128256), 30, std=3.0)
    scores = -torch.rand(24, 4, generator=torch.Generator().manual_seed(6))
    got = check(logits, scores, 4)
    again = _select(logits, scores, 4)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((6,), torch.uint8), ((6, 3), torch.uint8), ((6, 5), torch.float16),
                                         ((6, 4), torch.int32), ((6, 7, 9), torch.float32), ((6, 4096), torch.int64),
                                         ((6, 33000), torch.float16)])
def test_reorder(cuda, shape, dtype):
    """Rows of 1-, 4- and 16-byte words; a row twice, a row dropped, -1, no such row."""
    from llm_compiler_3_b200 import _native, ops
    state = torch.randint(0, 200, shape, generator=torch.Generator().manual_seed(2)).to(dtype)
    parents = ints([[3, 3, 0], [-1, 5, 2]])
    got = ops.beam_reorder(state.cuda(), parents.cuda())
    assert _native.device_status() == 0
    want = torch.stack([state[p] if p >= 0 else torch.zeros_like(state[0]) for p in parents.view(-1).tolist()])
    assert torch.equal(got.cpu(), want)
    got = ops.beam_reorder(state.cuda(), ints([6, 1, -2]).cuda())
    with pytest.raises(_native.NpuError, match="0x8"):
        _native.device_status()
    assert torch.equal(got.cpu(), torch.stack([torch.zeros_like(state[0]), state[1], torch.zeros_like(state[0])]))


@pytest.mark.gpu
def test_reorder_of_unaligned_slices(cuda):
    from llm_compiler_3_b200 import ops
    whole = torch.arange(400, dtype=torch.float16).cuda()
    state = whole[3:387].view(6, 64)
    got = ops.beam_reorder(state, ints([5, 0, 1]).cuda())
    assert torch.equal(got, state[[5, 0, 1]])


@pytest.mark.gpu
def test_wrapper_checks_and_graphs(cuda):
    from llm_compiler_3_b200 import _native, ops
    logits, scores = seeded((2, 3, 500), 1).cuda(), torch.zeros(2, 3).cuda()
    done = torch.zeros(2, 3, dtype=torch.bool).cuda()
    for args in ((logits.bfloat16(), scores, 3), (logits[:, :, ::2], scores, 3), (logits, scores.half(), 3),
                 (logits, scores[:1], 3), (logits, scores, 0), (logits, scores, 3, done.int(), 1),
                 (logits, scores, 3, done[:1], 1), (logits, scores.cpu(), 3)):
        with pytest.raises(ValueError):
            ops.beam_select(*args)
    with pytest.raises(_native.NpuError, match="end token"):
        ops.beam_select(logits, scores, 3, done)
    with pytest.raises(_native.NpuError, match="aligned"):
        ops.beam_select(torch.zeros(1510).half().cuda()[1:1501].view(1, 3, 500), scores[:1], 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.beam_select(logits, scores, 4, done, 2)
        rows = ops.beam_reorder(logits.view(6, 500), got[2])
    for seed in range(3):
        logits.copy_(seeded((2, 3, 500), 40 + seed))
        graph.replay()
        want = ops.beam_select(logits, scores, 4, done, 2)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(rows, logits.view(6, 500)[want[2].view(-1).long()])


@pytest.mark.gpu
def test_zeros_of_both_signs_tie(cuda):
    logits = torch.full((1, 2, 600), -1.0, dtype=torch.float16)
    logits[0, :, 5::90] = -0.0
    logits[0, :, 7::90] = 0.0
    got = _select(logits, torch.zeros(1, 2), 14)
    assert got[1].tolist() == [sorted(list(range(5, 600, 90)) + list(range(7, 600, 90)))]
    assert got[2].tolist() == [[0] * 14]
