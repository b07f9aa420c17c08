"""GPU checks of beam search with the operators together: the example on a hybrid model, the same with the selection's and pages'
statements in the kernels' place, and the beams' scores against whole passes over their texts."""
import importlib.util
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from vllm_exact.beam import beam_select_torch
from vllm_exact.linear_attn import linear_attention_torch
from vllm_exact.pages import fork_pages_torch, resize_pages_torch
from vllm_exact.prompt_attn import prompt_attention_torch

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "vllm-exact_amd" / "examples" / "beam_search.py"
    spec = importlib.util.spec_from_file_location("beam_search", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def beam_select(logits, scores, beams, best, parents, tokens):
    for out, want in zip((best, parents, tokens), beam_select_torch(logits.cpu(), scores.cpu(), beams, best.shape[1])):
        out.copy_(want)
    return best, parents, tokens


def fork_pages(caches, table, lens, parents, refs, page, out, out_lens):
    new, new_lens, counts, missing = fork_pages_torch(caches, table, lens, parents, refs, page)
    out.copy_(new), out_lens.copy_(new_lens), refs.copy_(counts)
    assert missing == 0


def resize_pages(table, lens, new_lens, refs, page):
    new, counts, missing = resize_pages_torch(table, lens, new_lens, refs, page)
    table.copy_(new), refs.copy_(counts)
    assert missing == 0


STATEMENTS = SimpleNamespace(beam_select=beam_select, fork_pages=fork_pages, resize_pages=resize_pages)


@pytest.mark.parametrize("lens,beams,count", [((3, 40, 16, 1), 3, 20), ((200,), 5, 9), ((15, 33), 1, 18)])
def test_the_same_beams_as_with_the_statements(lens, beams, count):
    ex = example()
    g = torch.Generator().manual_seed(len(lens))
    model = ex.Model()
    prompts = [torch.randint(0, model.vocab, (n,), generator=g).tolist() for n in lens]
    texts, scores, left = ex.generate(model, prompts, count, beams)
    want = ex.generate(model, prompts, count, beams, STATEMENTS)
    assert torch.equal(texts, want[0]) and left == want[2] == 0
    assert ((scores - want[1]).abs() <= 2.0 ** -22 * scores.abs()).all()
    assert (scores[:, 1:] <= scores[:, :-1]).all() and torch.isfinite(scores).all()
    for t in texts:
        assert len({tuple(x.tolist()) for x in t}) == beams


def test_scores_are_the_texts_log_probabilities():
    """A whole pass over prompt and text with the statements. The cache's 8 bits keep keys and values to 2^-8 of their largest, four
    layers of it and the log-sum over 19 tokens stay well within 0.5 a text, against some 60 of the whole score; a wrong parent,
    page or state moves it by several."""
    ex = example()
    model = ex.Model()
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, model.vocab, (n,), generator=g).tolist() for n in (30, 7)]
    texts, scores, _ = ex.generate(model, prompts, 19, 4)
    for r, prompt in enumerate(prompts):
        for b in range(4):
            row = prompt + texts[r, b].tolist()
            cu = torch.tensor([0, len(row)], dtype=torch.int32, device="cuda")

            def mix(i, q, k, v):
                if model.recurrent(i):
                    return linear_attention_torch(q, k, v, cu, model.log_decay, 0.125)
                return prompt_attention_torch(q, k, v, cu, 0.125)

            logits = model.forward(torch.tensor(row, device="cuda"), torch.arange(len(row), device="cuda"), mix)
            lp = torch.log_softmax(logits.double(), dim=-1)[len(prompt) - 1:-1]
            assert abs(float(lp.gather(1, texts[r, b][:, None]).sum()) - float(scores[r, b])) < 0.5


def test_example_runs():
    ex = example()
    model = ex.Model(layers=2)
    best = [float(ex.generate(model, [[1, 2, 3]], 12, beams)[1][0, 0]) for beams in (1, 8)]
    assert all(x < 0 for x in best)
