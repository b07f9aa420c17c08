"""GPU checks of fp16 weights far below the largest: many of them together count. A weight is held to half a step of 16 bits
(twice that many in the trees) and, below the type's normal range, to 2^-32 of the row's largest weight: weights are at most
2^15 and the row's largest is at least 2^7, in steps of 2^-24."""
import pytest
import torch

import test_gpu_prompt_attention as prompts
import test_gpu_tree_decode as trees
from attention64 import attend64, check

pytestmark = pytest.mark.gpu
DEV = "cuda"
LEAST = 2.0 ** -32


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("powers", [17.0, 23.5, 25.5])  # of two, that the other keys score below the first
def test_prompts(D, powers):
    n = 12000
    q = torch.ones(n, 1, D, dtype=torch.float16, device=DEV)
    k = torch.zeros(n, 1, D, dtype=torch.float16, device=DEV)
    k[0] = powers / 1.4426950408889634 * 8 / D
    v = torch.ones(n, 1, D, dtype=torch.float16, device=DEV)
    v[0] = 0
    out = prompts.run(q, k, v, torch.tensor([0, n], dtype=torch.int32, device=DEV), scale=0.125)
    last = slice(n - 40, n)
    want, bound = attend64(q[last, 0], k[:, 0], v[:, 0], torch.ones(40, n, dtype=torch.bool).tril(n - 40), 0.125, 2.0 ** -11, LEAST)
    check(out[last, 0], want, bound)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("powers", [17.0, 25.5, 31.0])
@pytest.mark.parametrize("nodes", [1, 40])
def test_trees(D, powers, nodes):
    n, page = 12000, 16
    s = trees.make((n - nodes,), (nodes,), 4, 1, D, page, torch.float16, False, seed=1)
    key, value = s["cache"][:2]
    s["q"].fill_(D ** -0.5)
    tok = torch.arange(n, device=DEV)
    where = s["bt"][0].long()[tok // page], tok % page
    key[where], value[where] = 0, 1
    first = int(s["bt"][0, 0]), 0
    key[first], value[first] = powers / 1.4426950408889634, 0
    out = trees.run(s)
    seen = torch.cat([torch.ones(nodes, n - nodes, dtype=torch.bool), (s["mask"].cpu()[:, None] >> torch.arange(nodes)) & 1 == 1], 1)
    want, bound = attend64(s["q"][:, 0], key[where][:, 0], value[where][:, 0], seen, D ** -0.5, 2.0 ** -22 + 3 * 2.0 ** -24, LEAST)
    for h in range(4):
        check(out[:, h], want, bound, f"head {h}")
