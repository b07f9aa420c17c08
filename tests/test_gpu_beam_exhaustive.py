"""GPU checks of the beam search example against all texts there are: a tiny vocabulary, as many beams as a search that misses nothing needs."""
import importlib.util
import itertools
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "vllm-exact_amd" / "examples" / "beam_search.py"
    spec = importlib.util.spec_from_file_location("beam_search", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("layers,prompts", [(2, ((0, 1, 2), (2, 2, 0, 1, 1, 0, 0, 2, 1, 0, 1, 1, 2, 0, 2, 1))), (4, ((1,), (0, 2)))])
def test_as_many_beams_as_texts_find_them_all(layers, prompts):
    """27 beams: every text of 3 tokens of 3 lives, and the last selection picks the 27 best of all 81 of 4. Their scores are added up here in
    fp64 from the logits that each text's row had. Theirs are rounded to fp32 four times, by 2^-24 of less than 16, and their
    log-sums are off by a few 2^-25."""
    ex = example()
    model, count, beams, n = ex.Model(layers=layers, vocab=3), 4, 27, len(prompts)
    texts_of = [()] * (n * beams)  # of the rows, as they are selected
    found = [{} for _ in prompts]  # request: text -> log probabilities of its next token

    def select(logits, scores, beams, best, parents, tokens):
        lp = torch.log_softmax(logits.double(), dim=-1).tolist()
        for row, score in enumerate(scores.tolist()):
            if score != -torch.inf:
                assert found[row // beams].setdefault(texts_of[row], lp[row]) is lp[row], "two beams have one text"
        out = ex.KERNELS.beam_select(logits, scores, beams, best, parents, tokens)
        texts_of[:] = [texts_of[p] + (t,) if p >= 0 else () for p, t in zip(parents.flatten().tolist(), tokens.flatten().tolist())]
        return out

    kernels = SimpleNamespace(beam_select=select, fork_pages=ex.KERNELS.fork_pages, resize_pages=ex.KERNELS.resize_pages)
    texts, scores, left = ex.generate(model, [list(p) for p in prompts], count, beams, kernels)
    assert left == 0
    for r in range(n):
        assert len(found[r]) == 1 + 3 + 9 + 27
        total = {t: sum(found[r][t[:i]][t[i]] for i in range(count)) for t in itertools.product(range(3), repeat=count)}
        got = [tuple(t) for t in texts[r].tolist()]
        assert len(set(got)) == beams
        room = count * (16 * 2.0 ** -24 + 2.0 ** -23)
        for text, score, want in zip(got, scores[r].tolist(), sorted(total.values(), reverse=True)):
            assert want > -16 and abs(score - total[text]) < room and abs(score - want) < room
