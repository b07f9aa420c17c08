"""GPU checks of the order of continuations whose scores are equal in fp64: tokens of one beam by their logits, beams by their rows."""
import pytest
import torch

from vllm_exact.beam import beam_select, beam_select_torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
LOWEST = -torch.finfo(torch.float32).max


def check(logits, scores, beams, count):
    n = len(logits) // beams
    got = beam_select(logits.to(DEV), scores.to(DEV), beams, torch.empty(n, count, device=DEV), torch.empty(n, count, device=DEV, dtype=torch.int32),
                      torch.empty(n, count, device=DEV, dtype=torch.int64))
    want = beam_select_torch(logits, scores, beams, count)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    return got


def rows(n, V, dtype, seed):
    return (torch.randn(n, V, generator=torch.Generator().manual_seed(seed)) * 2.5).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("score", [-1e30, LOWEST, -1e12])
@pytest.mark.parametrize("V,count", [(100000, 4), (33000, 64), (700, 9), (5, 4)])
def test_one_beam(V, count, score, dtype):
    logits = rows(1, V, dtype, V)
    best, _, tokens = check(logits, torch.tensor([score]), 1, count)
    assert tokens[0].tolist() == logits[0].float().sort(descending=True, stable=True).indices[:count].tolist()
    given = float(torch.tensor(score))  # a score is off by its own rounding; log probabilities here are above -200
    assert (best.cpu().double() / given - 1).abs().max() <= 2.0 ** -24 + 200 / abs(given)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("score", [-1e30, LOWEST])
def test_dead_beams_beside_one_of_few_tokens(score, dtype):
    """A request whose live beam has three tokens left, and one with none: the other places go to the first dead beam's best."""
    V, beams, count = 50001, 4, 16
    logits = rows(2 * beams, V, dtype, 1)
    live = torch.tensor([7, 20000, 50000])
    kept = logits[2, live].clone()
    logits[2] = -torch.inf
    logits[2, live] = kept
    logits[beams + 1] = -torch.inf
    scores = torch.full((2 * beams,), score)
    scores[2], scores[beams + 1] = -3.0, -1.0
    best, parents, tokens = check(logits, scores, beams, count)
    assert parents[0].tolist() == [2] * 3 + [0] * 13 and parents[1].tolist() == [beams] * 16
    assert tokens[0, 3:].tolist() == logits[0].float().sort(descending=True, stable=True).indices[:13].tolist()


def test_logits_nearer_than_a_score_resolves():
    """Beams at -1e9, whose scores have steps of 2^-23, and logits some 2^-30 apart, equal ones among them, over several slices."""
    V, beams = 30000, 3
    g = torch.Generator().manual_seed(2)
    logits = 0.5 ** 30 * torch.randint(0, 4000, (2 * beams, V), generator=g).float()
    for scores in ([-1e9] * 6, [-1e9, -1e9 + 64, -1e9, -1e9 - 64, -1e9, -1e9]):
        for count in (1, 5, 64):
            check(logits, torch.tensor(scores), beams, count)


def test_many_equal_logits_of_drowned_beams():
    logits = torch.randint(0, 2, (6, 20003), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    for scores in ([LOWEST] * 6, [-1e30, -1.0, -1e30, -1e30, -1e30, -1e30]):
        check(logits, torch.tensor(scores), 3, 64)
        check(logits, torch.tensor(scores), 6, 64)
