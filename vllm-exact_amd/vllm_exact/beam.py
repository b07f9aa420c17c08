"""Beam search's selection over beams and vocabulary on MI355X.

Kernels (libvllm_exact_amd.so, beam_select.hip): of all continuations of a request's beams, scored in more than 32 bits, the
best in order. A beam's continuations go by their logits, those of different beams by their scores in fp64, and equal ones by beam and
token, so the result does not depend on the batch. Its parents are rows of the logits: pages.fork_pages takes them, and
linear_attn.linear_step through the slots it reads.
"""
import torch

from . import _native as _nx

MAX_COUNT = 64  # the most continuations of a request


def beam_select(logits, scores, beams, out_scores, out_parents, out_tokens):
    """logits (requests * beams, vocabulary) fp32, bf16 or fp16, rows may be strided; scores (requests * beams,) fp32, the beams'
    sums of log probabilities. The score of a continuation is scores[b] + log_softmax(logits[b])[token]; out_scores fp32,
    out_parents int32 (the row of the logits) and out_tokens int64, (requests, count) and contiguous, take the `count` (at
    most 64) best of each request in order: a row's tokens by their logits (also where scores[b] is so large, -1e30 say, that
    their scores are equal), rows by scores in fp64, equal ones by row and token. A beam of score -inf (one that has ended, or
    all but the first after a prompt) has no continuations, nor has a token of logit -inf; places left over are -inf, -1, -1. A request
    with a NaN or +inf in the logits or scores of its other beams gets NaN, -1, -1. The outputs have no memory in common with each other or the
    inputs, but out_scores may be the scores themselves where count is beams. A row's log sum is taken from fp32 exponentials, eight at a
    time in fp32 and then in fp64: scores are off by less than 2^-20 besides their rounding to fp32. Returns the three."""
    status = (_nx._calls or _nx.calls()).beam_select(logits, scores, beams, out_scores, out_parents, out_tokens)
    if status:
        _nx.check(status, "beam_select")
    return out_scores, out_parents, out_tokens


def beam_select_torch(logits, scores, beams, count):
    """torch statement of the selection in fp64: (scores, parents, tokens)."""
    rows, V = logits.shape
    live = scores != -torch.inf
    x = logits.double()
    top = x.amax(dim=1, keepdim=True)
    total = scores.double()[:, None] + ((x - top) - (x - top).exp().sum(dim=1, keepdim=True).log())
    total = torch.where(live[:, None] & (x != -torch.inf), total, -torch.inf)
    bad = ((total != total) | (total == torch.inf)).any(dim=1) | ~(scores < torch.inf)
    token = x.sort(dim=1, descending=True, stable=True).indices  # the sorts leave equal ones in their order
    best, at = total.gather(1, token).view(-1, beams * V).sort(dim=1, descending=True, stable=True)
    best, at = best[:, :count], at[:, :count]
    token = token.view(-1, beams * V).gather(1, at)
    if best.shape[1] < count:
        pad = count - best.shape[1]
        best = torch.nn.functional.pad(best, (0, pad), value=-torch.inf)
        at, token = (torch.nn.functional.pad(i, (0, pad)) for i in (at, token))
    none = best == -torch.inf
    parents = torch.arange(rows // beams, device=logits.device)[:, None] * beams + at // V
    bad = bad.view(-1, beams).any(dim=1, keepdim=True)
    return (best.float().masked_fill(bad, torch.nan), parents.masked_fill(none | bad, -1).to(torch.int32), token.masked_fill(none | bad, -1))
