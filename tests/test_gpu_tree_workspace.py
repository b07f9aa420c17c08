"""GPU checks of tree decoding's workspace: what a call takes, and that its size leaves the bits."""
import pytest
import torch

import test_gpu_tree_decode as trees

pytestmark = pytest.mark.gpu


def peak(call):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    return torch.cuda.max_memory_allocated() - before


def test_a_large_call_takes_one_partial_sum_for_each_group():
    n, nodes, H, D, longest = 96, 3, 32, 128, 131072
    s = trees.make((40,) * n, (nodes,) * n, H, 8, D, 16, torch.bfloat16, True)
    out = trees.run(s)
    took = peak(lambda: trees.run(s, longest=longest))
    rows = n * nodes * H
    assert took <= rows * (longest // 2048) * (D + 2) * 4 + rows * D * 4 + (4 << 20)  # partial sums, the output, blocks' rounding
    assert torch.equal(trees.run(s, longest=longest), out)


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("D", [64, 256])
def test_every_layout_of_the_partial_sums(int8, D):
    """Strands, whole groups and chunks, of the same requests: alone, in a batch and beside requests of many rows."""
    s = trees.make((7000, 2500, 5000), (3, 1, 2), 8, 2, D, 16, torch.bfloat16, int8, seed=D)
    alone = trees.run(s)
    trees.compare(alone, s, heads=(0, 7))
    n = 20
    many = dict(s, q=s["q"].repeat(n, 1, 1), bt=s["bt"].repeat(n, 1), sl=s["sl"].repeat(n), mask=s["mask"].repeat(n),
                qsl=torch.tensor([0] + [3, 1, 2] * n).cumsum(0).to(torch.int32).cuda())
    for max_nodes in (3, 64):  # 64: room for requests of many rows
        for longest in (7003, 12000):
            assert torch.equal(trees.run(many, max_nodes=max_nodes, longest=longest), alone.repeat(n, 1, 1)), (max_nodes, longest)
            assert torch.equal(trees.run(s, max_nodes=max_nodes, longest=longest), alone), (max_nodes, longest)
