"""GPU checks of states that linear attention carries through many calls and many parts: the roundings of their decays do not add up."""
import pytest
import torch

from vllm_exact.linear_attn import linear_prompt

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def decayed(calls, rows, g, D):
    """The starting states, and what `calls` prompts of `rows` rows of zeros leave of them."""
    H = len(g)
    start = torch.randn(1, H, D, D, generator=torch.Generator().manual_seed(0)).to(DEV)
    state, slot = start.clone(), ints([0])
    zero, out = torch.zeros(rows, H, D, device=DEV, dtype=torch.bfloat16), torch.empty(rows, H, D, device=DEV)
    for _ in range(calls):
        linear_prompt(zero, zero, zero, ints([0, rows]), g, 1.0, out, state, slot, slot)
    return start, state


@pytest.mark.parametrize("calls,rows,D", [(4000, 1, 64), (400, 37, 128), (100, 65, 256), (60, 700, 64), (1, 1 << 17, 64)])
def test_decays_of_many_calls_and_parts(calls, rows, D):
    """A state meets a rounding of at most 2^-24 of itself for each chunk of 32 rows and each part: a walk of so many, with a deviation of
    2^-24 / sqrt(3) a step at most, and room for eight of its deviations (of some 130000 values). The rounding of a head's decay
    itself, up to 2^-25 of it, would add up to a straight line."""
    windows = torch.tensor([0.3, 0.7, 1.0, 1.9, 3.3, 4.1, 6.7, 9.9])
    g = (-windows / (calls * rows)).to(DEV)  # the states end at exp(-0.3) .. exp(-9.9) of what they were
    start, state = decayed(calls, rows, g, D)
    want = start.double() * torch.exp(g.double() * (calls * rows))[:, None, None]
    steps = calls * (-(-rows // 32) if rows <= 1000 else rows // 320 + 17)
    assert (state.double() / want - 1).abs().max() < 8 * steps ** 0.5 * 2.0 ** -24 / 3 ** 0.5 + 2.0 ** -24
