"""CPU checks of the order that the statement of beam search's selection gives to continuations whose scores are equal in fp64."""
import pytest
import torch

from vllm_exact.beam import beam_select_torch


@pytest.mark.parametrize("score", [-1e30, -torch.finfo(torch.float32).max, -20.0])
def test_a_beam_whose_score_drowns_its_logits_goes_by_them(score):
    logits = torch.randn(1, 1000, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).float()
    best, parents, tokens = beam_select_torch(logits, torch.tensor([score]), 1, 9)
    assert tokens[0].tolist() == logits[0].sort(descending=True, stable=True).indices[:9].tolist() and parents.eq(0).all()


def test_rows_before_logits_before_tokens():
    logits = torch.tensor([[1.0, 3.0, 2.0, 3.0], [9.0, 0.0, 1.0, 2.0], [0.0, 5.0, -torch.inf, -torch.inf]])
    best, parents, tokens = beam_select_torch(logits, torch.tensor([-1e30, -1e30, -2.0]), 3, 12)
    assert parents[0].tolist() == [2, 2, 0, 0, 0, 0, 1, 1, 1, 1, -1, -1]
    assert tokens[0].tolist() == [1, 0, 1, 3, 2, 0, 0, 3, 2, 1, -1, -1]
    assert best[0, :2].tolist() == sorted(best[0, :2].tolist(), reverse=True) and best[0, 2:10].eq(-1e30).all()
