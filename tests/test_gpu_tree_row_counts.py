"""GPU checks of trees on both sides of the row counts at which requests go from one kernel to the other (32 rows of a KV head
at 256 dims, 96 below), and that at 256 dims too the batch leaves the bits."""
import pytest
import torch

import test_gpu_tree_decode as trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,G,nodes", [(256, 4, (8, 9)), (256, 1, (32, 33)), (256, 8, (4, 5)), (256, 33, (1, 1)), (256, 16, (2, 3)),
                                       (128, 4, (24, 25)), (128, 3, (32, 33)), (64, 2, (48, 49)), (64, 97, (1, 1)), (128, 96, (1, 2))])
def test_on_both_sides_of_a_switch(int8, dtype, D, G, nodes):
    s = trees.make((1300, 700), nodes, 2 * G, 2, D, 16, dtype, int8, seed=D + G)
    heads = (0, G - 1, G, 2 * G - 1)
    trees.compare(trees.run(s), s, heads=heads)
    trees.compare(trees.run(s, mask=False), s, mask=False, heads=heads)


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bits_of_many_rows_of_256_dims_do_not_depend_on_the_batch(int8, dtype):
    ctx, nodes = (4500, 3, 530, 2500, 1100), (30, 64, 9, 2, 8)
    s = trees.make(ctx, nodes, 8, 2, 256, 16, dtype, int8, seed=4)
    out = trees.run(s)
    assert torch.equal(trees.run(s, max_nodes=64, longest=9000), out)
    starts = s["qsl"].tolist()
    for b in range(len(ctx)):
        lo, hi = starts[b], starts[b + 1]
        one = dict(q=s["q"][lo:hi], cache=s["cache"], bt=s["bt"][b:b + 1], sl=s["sl"][b:b + 1],
                   qsl=torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda"), mask=s["mask"][lo:hi].contiguous())
        assert torch.equal(trees.run(one), out[lo:hi]), b
    n = 40
    many = dict(s, q=s["q"].repeat(n, 1, 1), bt=s["bt"].repeat(n, 1), sl=s["sl"].repeat(n), mask=s["mask"].repeat(n),
                qsl=torch.tensor([0] + list(nodes) * n).cumsum(0).to(torch.int32).cuda())
    assert torch.equal(trees.run(many), out.repeat(n, 1, 1))
