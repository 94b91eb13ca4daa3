"""The paged and beam operators together, as a decoding program uses them: prompts through
paged_append and paged_prefill, then beam search over them with page_update, page_copy,
paged_append, paged_decode, beam_select and beam_reorder, and a compaction on the way.

The model is an embedding per token (query, key and value, FP16) and an FP32 output
matrix.  The check knows no pages: it rebuilds each beam's keys and values from the
tokens that the beam holds, and takes attention over them in 64 bits."""
import random

import pytest
import torch

import oracle
from conftest import seeded
from test_paged import check, ints

VOCAB, HEADS, KV, DIM, PAGE, LAYERS = 53, 6, 2, 64, 8, 2
EOS = 3


class Model:
    def __init__(self):
        self.q = seeded((VOCAB, HEADS, DIM), 1)
        self.k = seeded((LAYERS, VOCAB, KV, DIM), 2)
        self.v = seeded((LAYERS, VOCAB, KV, DIM), 3)
        self.out = torch.randn(HEADS * DIM, VOCAB, generator=torch.Generator().manual_seed(4))

    def expected(self, tokens, layer, window, sinks):
        """Attention of the last token of `tokens` over all of them: (out, bound) [Hq, D]."""
        n = len(tokens)
        pages = [t[layer][tokens].transpose(0, 1).contiguous()[None] for t in (self.k, self.v)]
        table = torch.zeros(1, 1, dtype=torch.int32)
        want, bound = oracle.attention_paged(self.q[tokens[-1:]][:, :, None], *pages, table, [n], [1],
                                             window=window, sinks=sinks)
        return want[0, :, 0], bound[0, :, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks,seed", [(0, 0, 1), (20, 3, 2), (5, 0, 3)])
def test_beam_search_over_a_paged_cache(cuda, window, sinks, seed):
    from llm_compiler_3_b200 import _native, ops
    r = random.Random(seed)
    model, batch, width, steps, pool_pages = Model(), 3, 4, 14, 160
    entries = 8
    dev = torch.device("cuda", 0)
    pool = torch.full((2 * LAYERS, pool_pages, KV, PAGE, DIM), float("nan"), dtype=torch.float16, device=dev)
    mk, mv, mq = model.k.to(dev), model.v.to(dev), model.q.to(dev)
    out_w = model.out.to(dev)
    options = dict(window=window, sinks=sinks)

    # Admission: rows without a parent, pages for the prompts.
    prompts = [[r.randrange(VOCAB) for _ in range(n)] for n in (1, 17, 30)]
    longest = max(map(len, prompts))
    lens = ints([len(p) for p in prompts]).to(dev)
    refs = torch.zeros(pool_pages, dtype=torch.int32, device=dev)
    none = torch.full((1, entries), -1, dtype=torch.int32, device=dev)
    table, kept, refs, copies, info = ops.page_update(none, ints([0]).to(dev), ints([-1] * batch).to(dev),
                                                      lens, refs, PAGE)
    assert info.tolist()[1:] == [0, 0] and kept.tolist() == [0] * batch
    padded = torch.tensor([p + [0] * (longest - len(p)) for p in prompts], device=dev)
    for layer in range(LAYERS):
        ops.paged_append(mk[layer][padded].transpose(1, 2).contiguous(), mv[layer][padded].transpose(1, 2).contiguous(),
                         pool[2 * layer], pool[2 * layer + 1], table, ints([0] * batch).to(dev), lens)
    q = mq[padded].transpose(1, 2).contiguous()
    hidden = ops.paged_prefill(q, pool[0], pool[1], table, lens, lens, **options)
    for b, p in enumerate(prompts):
        for i in range(longest):
            got = hidden[b, :, i].cpu()
            if i < len(p):
                check(got, *model.expected(p[:i + 1], 0, window, sinks))
            else:
                assert torch.count_nonzero(got) == 0
    last = torch.stack([hidden[b, :, len(p) - 1] for b, p in enumerate(prompts)])

    # The first step makes `width` beams of each prompt.
    logits = (last.float().view(batch, 1, -1) @ out_w).contiguous()
    scores = torch.zeros(batch, 1, device=dev)
    done = torch.zeros(batch, 1, dtype=torch.bool, device=dev)
    history = torch.zeros(batch, steps, dtype=torch.int32, device=dev)
    beams = [list(p) for p in prompts]  # what each row of the table holds, on the host
    for step in range(steps):
        before = logits.cpu(), scores.cpu(), done.cpu()
        scores, tokens, parents, done = ops.beam_select(logits, scores, width, done, EOS)
        want = oracle.beam_select(*before[:2], width, before[2], EOS)
        assert tokens.cpu().tolist() == want[1].tolist() and parents.cpu().tolist() == want[2].tolist()
        assert done.cpu().tolist() == want[3].tolist()
        flat = parents.view(-1)
        history = ops.beam_reorder(history, flat)
        history[:, step] = tokens.view(-1)
        beams = [beams[p] + [t] for p, t in zip(flat.tolist(), tokens.view(-1).tolist())]

        # Their pages: forked, grown by the new token's.
        table, kept, refs, copies, info = ops.page_update(table, lens, flat, lens[flat.long()] + 1, refs, PAGE)
        assert info.tolist()[1] == 0
        ops.page_copy(pool, copies, info[2:])
        if step in (4, 9):  # the pool defragmented between two steps
            table, refs, moves, _, info = ops.page_compact(table, refs)
            ops.page_copy(pool, moves, info[1:])
        rows = table.cpu()
        held = rows[rows >= 0]
        assert torch.equal(torch.bincount(held.long(), minlength=pool_pages).int(), refs.cpu())
        lens = kept + 1
        assert lens.tolist() == [len(b) for b in beams]
        now = tokens.view(-1).long()
        for layer in range(LAYERS):
            ops.paged_append(mk[layer][now][:, :, None].contiguous(), mv[layer][now][:, :, None].contiguous(),
                             pool[2 * layer], pool[2 * layer + 1], table, kept)
            got = ops.paged_decode(mq[now], pool[2 * layer], pool[2 * layer + 1], table, lens, **options).cpu()
            for w, b in enumerate(beams):
                check(got[w], *model.expected(b, layer, window, sinks))
            if layer == 0:
                logits = (got.to(dev).float().view(batch, width, -1) @ out_w).contiguous()
    lengths = [len(p) for p in prompts for _ in range(width)]
    assert history.tolist() == [b[n:] for b, n in zip(beams, lengths)]

    # Every row freed: every page is.
    _, _, refs, _, info = ops.page_update(table, lens, ints([-1]).to(dev), ints([0]).to(dev), refs, PAGE)
    assert info.tolist() == [pool_pages, 0, 0] and torch.count_nonzero(refs) == 0
    assert _native.device_status() == 0


@pytest.mark.gpu
def test_the_documented_step_with_beams_that_end(cuda):
    """The README's step, run as it stands, where most tokens are banned: beams without a
    continuation take no pages, write no rows and give zeros, and their places fill again."""
    import re
    from conftest import ROOT
    from llm_compiler_3_b200 import _native
    blocks = re.findall(r"```python\n(.*?)```", (ROOT / "README.md").read_text(), re.S)
    step, = [b for b in blocks if "ops.page_update(" in b]
    batch, width, kv, page, pages, entries, vocab = 3, 2, 2, 8, 50, 45, 40
    dev = torch.device("cuda", 0)
    lens, at = [9, 9, 20, 20, 300, 300], 0
    table, refs = torch.full((batch * width, entries), -1, dtype=torch.int32), torch.zeros(pages, dtype=torch.int32)
    for row in range(0, batch * width, 2):  # both beams of a sequence share their full pages
        full, held = lens[row] // page, -(-lens[row] // page)
        for r in (row, row + 1):
            table[r, :full] = torch.arange(at, at + full)
        at += full
        for r in (row, row + 1):
            table[r, full:held] = torch.arange(at, at + held - full)
            at += held - full
        refs += torch.bincount(table[row:row + 2][table[row:row + 2] >= 0].long(), minlength=pages).int()
    pool = seeded((2, pages, kv, page, 128), 1).to(dev)
    state = dict(pool=pool, table=table.to(dev), lens=ints(lens).to(dev), refs=refs.to(dev), page_size=page, eos=3,
                 width=width, layers=1, scores=torch.zeros(batch, width, device=dev),
                 done=torch.zeros(batch, width, dtype=torch.bool, device=dev))
    # Sequence 0 has one continuation left, sequence 1 none (for good); then two for sequence 0.
    want_lens = ([10, 0, 0, 0, 301, 301], [11, 11, 0, 0, 302, 302])
    for n, wanted in enumerate(want_lens):
        logits = seeded((batch, width, vocab), 10 + n).float()
        logits[0] = -float("inf")
        logits[0, 0, 5:6 + n] = 1.0
        if n == 0:
            logits[1] = -float("inf")
        state.update(logits=logits.to(dev), q=seeded((batch * width, 4, 128), 20 + n).to(dev),
                     k=seeded((batch * width, kv, 1, 128), 30 + n).to(dev),
                     v=seeded((batch * width, kv, 1, 128), 40 + n).to(dev))
        before = state["logits"].cpu(), state["scores"].cpu(), width, state["done"].cpu(), 3
        exec(step, state)
        assert _native.device_status() == 0
        want = oracle.beam_select(*before)
        assert state["parents"].tolist() == want[2].tolist() and state["tokens"].tolist() == want[1].tolist()
        assert state["lens"].tolist() == wanted and state["info"].tolist()[1] == 0
        rows = state["table"].cpu()
        assert [int((row >= 0).sum()) for row in rows] == [-(-x // page) for x in wanted]
        assert torch.equal(torch.bincount(rows[rows >= 0].long(), minlength=pages).int(), state["refs"].cpu())
        for r, x in enumerate(wanted):  # the new key stands where the row ends
            if x:
                held = pool[0, int(rows[r, (x - 1) // page]), :, (x - 1) % page]
                assert torch.equal(held, state["k"][r, :, 0])
        out, bound = oracle.attention_paged(state["q"].cpu()[:, :, None], pool[0].cpu(), pool[1].cpu(), rows, wanted,
                                            [min(1, x) for x in wanted], window=4096, sinks=4)
        check(state["out"].cpu(), out[:, :, 0], bound[:, :, 0])
