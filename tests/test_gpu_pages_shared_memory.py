"""GPU checks of the page operators on caches that share memory: tokens would be moved side by side twice."""
import pytest
import torch

from vllm_exact.pages import copy_pages, fork_pages, keep_drafted, keep_drafted_torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BLOCKS, PAGE, KV, D = 12, 16, 2, 96


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def pool():
    return torch.randint(-100, 100, (BLOCKS, PAGE, KV, D), device=DEV, dtype=torch.int16)


def keep(caches):
    table, lens = ints([[3, 1, 2, -1]]), ints([40])
    out = torch.empty_like(lens)
    return keep_drafted(caches, table, lens, ints([0, 10]), ints([0b1110110000], torch.int64), PAGE, out), table, lens


def test_keep_of_caches_with_memory_in_common():
    p = pool()
    before = p.clone()
    for caches in ([p, p], [p, p[..., :32]], [p[..., :64], pool(), p[..., 63:]], [p[:, :, :1], p[:, :, 0]], [p, p.view(torch.int8)], [p[..., :1].expand(BLOCKS, PAGE, KV, 4)],
                   [p[:, :, :1].expand(BLOCKS, PAGE, 3, D)]):
        with pytest.raises(ValueError, match="caches (must not|are views)"):
            keep(caches)
    assert torch.equal(p, before)


def test_keep_of_caches_side_by_side():
    a, b = pool(), pool().transpose(1, 2).contiguous().transpose(1, 2)
    views = lambda a, b: [a[..., :64], a[..., 64:], b[:, :, :1], b[:, :, 1], b[:0].new_empty(BLOCKS, PAGE, 0)]
    said = [a.clone(), b.clone()]
    got, table, lens = keep(views(a, b))
    want = keep_drafted_torch(views(*said)[:4], table, lens, ints([0, 10]), ints([0b1110110000], torch.int64), PAGE)
    assert torch.equal(got, want) and torch.equal(a, said[0]) and torch.equal(b, said[1])


def test_fork_and_copy_move_shared_memory_once():
    """Whole pages go to pages that nobody reads: twice the same."""
    p = pool()
    said = p.clone()
    copy_pages([p, p[..., 8:40], p], PAGE, ints([0, 1]), ints([5, 6]))
    said[5], said[6] = said[0], said[1]
    assert torch.equal(p, said)
    refs = torch.zeros(BLOCKS, dtype=torch.int32, device=DEV)
    refs[3] = 1
    out, out_lens = ints([[0], [0]]), ints([0, 0])
    fork_pages([p, p[..., :32]], ints([[3]]), ints([9]), ints([0, 0]), refs, PAGE, out, out_lens)
    said[0] = said[3]
    assert out.tolist() == [[3], [0]] and torch.equal(p, said)
