"""CPU checks of whether two tensors have memory in common, against the sets of their bytes."""
import random

import pytest
import torch

from vllm_exact import _native as nx


def bytes_of(t):
    at, item = torch.zeros(1, dtype=torch.int64), t.element_size()
    for n, s in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n) * s).flatten()
    return set((t.data_ptr() + item * at[:, None] + torch.arange(item)).flatten().tolist())


def check(a, b):
    want = bool(bytes_of(a) & bytes_of(b))
    assert nx.calls().overlap(a, b) is want and nx.calls().overlap(b, a) is want
    return want


def test_rows_of_one_projection():
    """Queries, keys and values beside each other in rows, heads of groups between each other, halves of rows, and rows that follow."""
    x = torch.zeros(7, 12, 64, dtype=torch.bfloat16)
    q, k, v = x.split((8, 2, 2), dim=1)
    assert not any(check(a, b) for a, b in ((q, k), (q, v), (k, v))) and check(q, x[:, 7:9]) and check(x[3], x[3:])
    g = x.view(7, 2, 6, 64)
    assert not check(g[:, :, :4], g[:, :, 4]) and check(g[:, :, :4], g[:, :, 3]) and not check(g[:, :, 4], g[:, :, 5])
    assert not check(x[..., :32], x[..., 32:]) and check(x[..., :33], x[..., 32:]) and not check(x[:3], x[3:]) and check(x[:4], x[3:])
    assert not check(x[::2], x[1::2]) and check(x[::2], x[2:3]) and not check(x[:0], x)


def test_caches_keys_and_values_side_by_side():
    pool = torch.zeros(5, 2, 16, 24, dtype=torch.int8)
    k, v = pool.transpose(1, 2).split(12, dim=-1)
    assert not check(k, v) and check(k, pool[2]) and not check(k[1:3], v[1:3]) and not check(k[:2], k[2:]) and check(k, pool[..., 11:12])


@pytest.mark.parametrize("seed", range(4))
def test_random_strides(seed):
    rng = random.Random(seed)
    base = torch.zeros(4000, dtype=torch.uint8)
    met = 0
    for _ in range(400):
        views = []
        for _ in range(2):
            dims = rng.randint(0, 4)
            shape = [rng.randint(1, 4) for _ in range(dims)]
            strides = [rng.choice((0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 48, 100)) for _ in range(dims)]
            item = rng.choice((torch.uint8, torch.int16, torch.int32))
            views.append(base[rng.randint(0, 100) * 8:].view(item).as_strided(shape, strides))
        met += check(*views)
    assert 20 < met < 380  # both answers


def test_two_row_lengths():
    """Rows of two lengths in one buffer meet as their bytes do; so do those of many rows, looked through or not."""
    base = torch.zeros(1 << 16, dtype=torch.uint8)
    assert check(base[:700].view(7, 100)[:, :10], base[10:].as_strided((5, 10), (90, 1)))
    assert not check(base[:700].view(7, 100)[:, :10], base[10:].as_strided((5, 10), (100, 1)))
    assert not check(base[:700].view(7, 100)[:, :10], base[50:].as_strided((9, 10), (50, 1))[2:3])
    with pytest.raises(TypeError):
        nx.calls().overlap(base, 3)
