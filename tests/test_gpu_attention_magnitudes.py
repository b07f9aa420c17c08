"""GPU checks of finite values at the top of the range: a weighted mean of finite values is finite, however large its sum of
unnormalised terms. Tolerances as in the operators' own tests (attention64.attend64 adds up the terms, relative to the
largest values)."""
import pytest
import torch

import test_gpu_prompt_attention as prompts
import test_gpu_tree_decode as trees
from vllm_exact.int8_cache import make_cache, write_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"
HUGE = 3.0e38


def huge(v, seed, dims):
    """Values up to the largest of the type in `dims`, of both signs in the second of them."""
    g = torch.Generator().manual_seed(seed)
    v[..., dims[0]] = HUGE
    x = torch.rand(v.shape[:-1], generator=g) * 2 - 1
    v[..., dims[1]] = (x * HUGE).to(v.dtype).to(v.device)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompts(D, out_dtype):
    q, k, v, cu = prompts.make((1, 40, 700), 4, 2, D, torch.bfloat16, seed=D)
    q = q * 3
    clean = prompts.run(q, k, v, cu, out_dtype)
    huge(v, 1, (2, 7))
    out = prompts.run(q, k, v, cu, out_dtype)
    prompts.compare(out, q, k, v, cu)
    rest = [d for d in range(D) if d not in (2, 7)]
    assert torch.equal(out[:, :, rest], clean[:, :, rest])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [1, 7, 40])  # 4, 28 and 160 rows of a KV head
@pytest.mark.parametrize("ctx", [20, 1500, 9000])
def test_trees_over_a_16_bit_cache(D, nodes, ctx):
    s = trees.make((ctx,), (nodes,), 4, 1, D, 16, torch.bfloat16, False, seed=D + ctx)
    s["q"] *= 3
    clean = trees.run(s)
    v = s["cache"][1]
    keep = v.clone()
    for part in (slice(None), slice(0, 600), slice(800, 1000)):  # everywhere, in some segments only
        tok = torch.arange(ctx + nodes, device=DEV)[part]
        if tok.numel() == 0:
            continue
        where = s["bt"][0].long()[tok // 16], tok % 16
        rows = v[where]
        huge(rows, 3, (2, 7))
        v[where] = rows
        out = trees.run(s)
        trees.compare(out, s, heads=(0, 3))
        rest = [d for d in range(D) if d not in (2, 7)]
        assert torch.equal(out[:, :, rest], clean[:, :, rest]), part
        assert torch.equal(trees.run(s, max_nodes=64, longest=30000), out), part
        v.copy_(keep)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])  # of the queries
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [1, 7, 40])
@pytest.mark.parametrize("ctx", [20, 1500, 9000])
def test_trees_over_an_8_bit_cache(dtype, D, nodes, ctx):
    s = trees.make((ctx,), (nodes,), 4, 1, D, 16, dtype, True, seed=D + ctx)
    s["q"] *= 3
    page, blocks = 16, s["cache"][0].shape[0]
    g = torch.Generator().manual_seed(1)
    # (tokens with huge values, the part of the keys)
    for part in (slice(None), slice(0, 600), slice(800, 1000)):
        tok = torch.arange(ctx + nodes, device=DEV)[part]
        if tok.numel() == 0:
            continue
        rows = (torch.randn(tok.numel(), 1, D, generator=g) * 1e38).clamp(-HUGE, HUGE).to(torch.bfloat16).to(DEV)
        rows[:, :, 2] = HUGE
        t = dict(s, cache=tuple(x.clone() for x in s["cache"]))
        spare = make_cache(blocks, page, 1, D, DEV)
        slots = s["bt"][0].long()[tok // page] * page + tok % page
        write_cache(rows, rows, *spare, slots)
        at = slots // page, slots % page
        t["cache"][1][at], t["cache"][3][at] = spare[1][at], spare[3][at]
        out = trees.run(t)
        trees.compare(out, t, heads=(0, 3))
        assert torch.equal(trees.run(t, max_nodes=64, longest=30000), out), part


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [60, -60])
def test_values_times_a_power_of_two(D, power):
    """The outputs are the same bits times that power."""
    q, k, v, cu = prompts.make((1, 40, 700), 4, 2, D, torch.bfloat16, seed=D)
    out = prompts.run(q, k, v, cu)
    assert torch.equal(prompts.run(q, k, v * 2.0 ** power, cu), out * 2.0 ** power)
    for nodes in (3, 40):
        s = trees.make((9000,), (nodes,), 4, 1, D, 16, torch.bfloat16, False, seed=D)
        out = trees.run(s)
        s["cache"][1].mul_(2.0 ** power)
        assert torch.equal(trees.run(s), out * 2.0 ** power)
        s = trees.make((9000,), (nodes,), 4, 1, D, 16, torch.bfloat16, True, seed=D)
        out = trees.run(s)
        s["cache"][3].mul_(2.0 ** power)
        assert torch.equal(trees.run(s), out * 2.0 ** power)
