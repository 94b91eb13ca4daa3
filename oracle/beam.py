"""64-bit CPU restatement of beam search's selection (test infrastructure only)."""
from __future__ import annotations

import torch

__all__ = ["beam_worths", "beam_select"]


def beam_worths(logits, scores, done=None, eos=-1):
    """[B, W x V] FP64: what every continuation is worth; -inf where there is none."""
    batch, beams, vocab = logits.shape
    x = logits.double()
    most = torch.finfo(logits.dtype).max
    x = torch.where(torch.isnan(x), float("-inf"), x).clamp(max=most)
    s = scores.double()[..., None]
    # Relative to the largest: beside 3.4e38 even FP64 would lose the sum's logarithm.
    top = x.amax(-1, keepdim=True)
    part = x - torch.where(top == float("-inf"), 0.0, top)
    worth = part - torch.logsumexp(part, -1, keepdim=True) + s
    worth = torch.where((x == float("-inf")) | torch.isnan(s), float("-inf"), worth)
    if done is not None:
        only = torch.full((vocab,), float("-inf"), dtype=torch.float64)
        only[eos] = 0.0
        worth = torch.where(done[..., None], s + only, worth)
    return torch.where(torch.isnan(worth), float("-inf"), worth).reshape(batch, -1)


def beam_select(logits, scores, width, done=None, eos=-1):
    """(scores, tokens, parents, done) in plain Python order: best first, lowest index
    among equals; parents are rows b x W + beam."""
    batch, beams, vocab = logits.shape
    worth = beam_worths(logits, scores, done, eos)
    out = (torch.full((batch, width), float("-inf"), dtype=torch.float64),
           torch.full((batch, width), -1), torch.full((batch, width), -1),
           torch.zeros(batch, width, dtype=torch.bool))
    for b in range(batch):
        order = torch.argsort(worth[b], descending=True, stable=True)[:width].tolist()
        for k, at in enumerate(order):
            if worth[b, at] == float("-inf"):
                break
            out[0][b, k] = worth[b, at]
            out[1][b, k] = at % vocab
            out[2][b, k] = b * beams + at // vocab
            out[3][b, k] = at % vocab == eos or (done is not None and bool(done[b, at // vocab]))
    return out
