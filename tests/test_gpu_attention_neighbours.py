"""GPU checks that a row's bits are its own: other rows of its prompt or tree, in the same wave of the kernel or not, change
nothing, whatever they score."""
import pytest
import torch

import test_gpu_prompt_attention as prompts
import test_gpu_tree_decode as trees

pytestmark = pytest.mark.gpu


def steep(x, seed):
    """Other rows of the same shape whose scores differ by hundreds."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(x.shape, generator=g) * 30).to(x.dtype).to(x.device)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cut", [9, 211, 400])
def test_later_tokens_of_a_prompt(D, dtype, cut):
    q, k, v, cu = prompts.make((600,), 4, 2, D, dtype, seed=cut + D)
    q = q * 4
    want = prompts.run(q, k, v, cu)
    prompts.compare(want, q, k, v, cu, heads=(0, 3))
    q2, k2, v2 = q.clone(), k.clone(), v.clone()
    q2[cut:], k2[cut:], v2[cut:] = steep(q[cut:], 1), steep(k[cut:], 2), steep(v[cut:], 3)
    assert torch.equal(prompts.run(q2, k2, v2, cu)[:cut], want[:cut])
    k2 = k.clone()
    k2[cut] = float("inf")  # later rows score infinities of both signs
    assert torch.equal(prompts.run(q, k2, v, cu)[:cut], want[:cut])
    short = cu.clone()
    short[1] = cut
    assert torch.equal(prompts.run(q[:cut], k[:cut], v[:cut], short), want[:cut])


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [6, 10, 40])  # 24, 40 and 160 rows of a KV head
def test_other_nodes_of_a_tree(int8, D, nodes):
    s = trees.make((1500,), (nodes,), 8, 2, D, 16, torch.bfloat16, int8, seed=D + nodes)
    s["q"] *= 4
    want = trees.run(s)
    trees.compare(want, s, heads=(0, 7))
    keep = torch.arange(nodes) % 3 == 1
    q = s["q"].clone()
    q[~keep] = steep(q[~keep], 5)
    assert torch.equal(trees.run(dict(s, q=q))[keep], want[keep])
    q = s["q"].clone()
    q[:, 1::2] = steep(q[:, 1::2], 6)  # other heads of the same group
    assert torch.equal(trees.run(dict(s, q=q))[:, ::2], want[:, ::2])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [6, 40])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_infinite_keys_of_masked_drafts(D, nodes, bad):
    s = trees.make((500,), (nodes,), 8, 2, D, 16, torch.bfloat16, False, seed=D)
    s["q"] *= 4
    want = trees.run(s)
    for j in (0, nodes // 2, nodes - 1):
        sees = (s["mask"].cpu() >> j) & 1 == 1
        at = (int(s["bt"][0, (500 + j) // 16]), (500 + j) % 16)
        keep = s["cache"][0][at].clone()
        s["cache"][0][at] = bad
        assert torch.equal(trees.run(s)[~sees], want[~sees]), j
        s["cache"][0][at] = keep
