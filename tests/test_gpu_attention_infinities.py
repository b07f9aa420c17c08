"""GPU checks of values that are infinities or NaN where rows do attend to them: the formula's +inf, -inf or NaN in that
dimension, at any distance from the masked keys and for any weight above 0, and the usual bits in the others."""
import pytest
import torch

import test_gpu_prompt_attention as prompts
import test_gpu_tree_decode as trees

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")


def as_numbers(x):
    return x.nan_to_num(7.0, 8.0, 9.0)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nodes", [1, 7, 30])  # 4, 28 and 120 rows of a KV head
@pytest.mark.parametrize("ctx", [1530, 9000])
def test_context_of_a_tree(D, dtype, nodes, ctx):
    s = trees.make((ctx,), (nodes,), 8, 2, D, 16, dtype, False, seed=D + nodes)
    clean = trees.run(s)
    v = s["cache"][1]
    rest = [d for d in range(D) if d not in (3, 5)]
    for at in (0, 37, 700, 1029, ctx - 1):
        place = (int(s["bt"][0, at // 16]), at % 16)
        keep = v[place].clone()
        for bad in (INF, -INF, NAN):
            v[place][0, 3] = bad  # the first KV head
            out = trees.run(s)
            assert torch.equal(as_numbers(out[:, :4, 3]), as_numbers(torch.full_like(out[:, :4, 3], bad))), (at, bad)
            assert torch.equal(out[:, :4][:, :, rest], clean[:, :4][:, :, rest]), (at, bad)
            assert torch.equal(out[:, 4:], clean[:, 4:]), (at, bad)
        v[place][0, 3], v[place][0, 5] = INF, -INF
        other = (int(s["bt"][0, 64]), 9)  # key 1033
        keep2 = v[other].clone()
        v[other][0, 3] = -INF  # +inf and -inf together are NaN
        out = trees.run(s)
        assert torch.isnan(out[:, :4, 3]).all() and (out[:, :4, 5] == -INF).all(), at
        v[place], v[other] = keep, keep2
    assert torch.equal(trees.run(s), clean)


def line(n, D, dtype, low, high):
    """Keys that score 0, low or high (in nats) against queries of ones: k[i] = score * 8 / D at scale 1/8."""
    k = torch.zeros(n, 1, D, dtype=dtype, device=DEV)
    for i, x in {**low, **high}.items():
        k[i] = x * 8 / D
    return k


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype,low", [(torch.bfloat16, -128.0), (torch.float16, -32.0), (torch.float16, -128.0)])
def test_small_weights_of_infinite_values(D, dtype, low):
    """exp(-128) is above 0: an infinite value counts, also where it comes first and a far higher score later."""
    n = 700
    q, k = torch.ones(n, 2, D, dtype=dtype, device=DEV), line(n, D, dtype, {5: low, 300: low}, {600: 128.0})
    g = torch.Generator().manual_seed(0)
    v = torch.randn(n, 1, D, generator=g).to(dtype).to(DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    clean = prompts.run(q, k, v, cu, scale=0.125)
    v[5, 0, 1], v[300, 0, 2] = INF, -INF
    out = prompts.run(q, k, v, cu, scale=0.125)
    assert (out[5:, :, 1] == INF).all() and (out[300:, :, 2] == -INF).all()
    out[5:, :, 1], out[300:, :, 2] = clean[5:, :, 1], clean[300:, :, 2]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype,low", [(torch.bfloat16, -128.0), (torch.float16, -128.0)])
@pytest.mark.parametrize("nodes", [2, 70 // 2])
def test_small_weights_in_the_context_of_a_tree(D, dtype, low, nodes):
    n = 9000
    s = trees.make((n - nodes,), (nodes,), 4, 1, D, 16, dtype, False, seed=D)
    key, value = s["cache"][:2]
    s["q"].fill_(1 if D == 64 else 0.5)  # at scale D^-0.5
    score = D ** 0.5 * float(s["q"].flatten()[0])
    tok = torch.arange(n, device=DEV)
    where = s["bt"][0].long()[tok // 16], tok % 16
    key[where] = 0
    for i, x in ((5, low), (3000, low), (8200, 128.0)):
        key[int(s["bt"][0, i // 16]), i % 16] = x / score
    clean = trees.run(s)
    value[int(s["bt"][0, 0]), 5, 0, 1] = INF
    value[int(s["bt"][0, 3000 // 16]), 3000 % 16, 0, 2] = -INF
    out = trees.run(s)
    assert (out[:, :, 1] == INF).all() and (out[:, :, 2] == -INF).all()
    out[:, :, 1:3] = clean[:, :, 1:3]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("nodes", [2, 35])
@pytest.mark.parametrize("at", [3, 2900])
def test_an_infinite_scale(nodes, at):
    """8-bit cache: whole numbers times an infinite scale are infinities of their signs, and NaN for 0."""
    s = trees.make((3000,), (nodes,), 8, 2, 64, 16, torch.bfloat16, True, seed=at)
    clean = trees.run(s)
    place = (int(s["bt"][0, at // 16]), at % 16)
    s["cache"][3][place][0] = INF
    want = (s["cache"][1][place][0].float() * INF).expand(nodes, 4, 64)
    out = trees.run(s)
    assert torch.equal(as_numbers(out[:, :4]), as_numbers(want)) and torch.equal(out[:, 4:], clean[:, 4:])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_no_score_above_minus_infinity(D):
    """Where every score is -inf the formula gives no number, infinite values or not."""
    q, k, v, cu = prompts.make((90,), 2, 1, D, torch.bfloat16)
    q, k = q.abs() + 0.1, torch.full_like(k, -INF)
    v[0, 0, 3] = INF
    assert torch.isnan(prompts.run(q, k, v, cu)).all()
    for nodes in (2, 40):
        s = trees.make((600,), (nodes,), 4, 1, D, 16, torch.bfloat16, False)
        s["q"].abs_().add_(0.1)
        s["cache"][0][:] = -INF
        s["cache"][1][int(s["bt"][0, 0]), 3, 0, 5] = INF
        assert torch.isnan(trees.run(s)).all()
