"""GPU checks of beam_select's outputs over its inputs: scores in place where there are as many continuations as beams, refused elsewhere."""
import pytest
import torch

from vllm_exact.beam import beam_select

pytestmark = pytest.mark.gpu
DEV = "cuda"


def outs(n, count):
    return torch.empty(n, count, device=DEV), torch.empty(n, count, device=DEV, dtype=torch.int32), torch.empty(n, count, device=DEV, dtype=torch.int64)


@pytest.mark.parametrize("count", [1, 3, 5, 8])
def test_other_requests_scores_are_not_written_over(count):
    """With fewer or more continuations than beams a request would write scores that another one has yet to read."""
    n, beams = 6, 4
    logits = torch.randn(n * beams, 500, device=DEV)
    buffer = torch.rand(n * max(beams, count) + 8, device=DEV)
    scores = buffer[:n * beams]
    _, parents, tokens = outs(n, count)
    before = buffer.clone()
    for at in (0, 1, n * beams - 1):
        best = buffer[at:at + n * count]
        if len(best) == n * count:
            with pytest.raises(ValueError, match="out_scores must not be"):
                beam_select(logits, scores, beams, best.view(n, count), parents, tokens)
    assert torch.equal(buffer, before)


def test_beside_the_scores_and_in_place():
    n, beams = 5, 4
    logits = torch.randn(n * beams, 700, device=DEV)
    buffer = torch.rand(2 * n * beams, device=DEV)
    scores, beside = buffer[:n * beams], buffer[n * beams:].view(n, beams)
    want = beam_select(logits, scores, beams, *outs(n, beams))
    got = beam_select(logits, scores, beams, beside, *outs(n, beams)[1:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = beam_select(logits, scores, beams, scores.view(n, beams), *outs(n, beams)[1:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_outputs_over_each_other_and_the_logits():
    n, beams = 3, 2
    logits, scores = torch.randn(n * beams, 64, device=DEV), torch.rand(n * beams, device=DEV)
    best, parents, tokens = outs(n, beams)
    both = torch.zeros(n, beams, device=DEV, dtype=torch.int64)
    over = logits.view(-1)[:n * beams].view(n, beams)
    for bad in ((best, both.view(-1).view(torch.int32)[:n * beams].view(n, beams), both), (best, best.view(torch.int32), tokens), (over, parents, tokens),
                (best, over.view(torch.int32), tokens), (best, scores.view(n, beams).view(torch.int32), tokens)):
        with pytest.raises(ValueError, match="must not be"):
            beam_select(logits, scores, beams, *bad)
