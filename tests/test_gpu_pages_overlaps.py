"""GPU checks of the page operators' outputs beside and over their inputs."""
import pytest
import torch

from vllm_exact.int8_cache import make_cache
from vllm_exact.pages import fork_pages, fork_pages_torch, keep_drafted, resize_pages, resize_pages_torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROWS, COLS, PAGE, BLOCKS = 4, 5, 16, 40


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def tables():
    """Two tables side by side in one buffer, the first one filled, and two vectors of lengths in another."""
    both = torch.full((ROWS, 2 * COLS), -1, dtype=torch.int32, device=DEV)
    table, other = both[:, :COLS], both[:, COLS:]
    table[:, :3] = torch.arange(3 * ROWS, device=DEV, dtype=torch.int32).view(ROWS, 3)
    lens = torch.zeros(2 * ROWS + 3, dtype=torch.int32, device=DEV)
    lens[:ROWS] = ints([40, 33, 48, 35])
    refs = torch.zeros(2 * BLOCKS, dtype=torch.int32, device=DEV)
    refs[:3 * ROWS] = 1
    return both, table, other, lens, refs


def test_fork():
    both, table, other, lens, refs = tables()
    parents = ints([1, 1, 2, 0])
    ok = dict(caches=[], table=table, lens=lens[:ROWS], parents=parents, refs=refs[:BLOCKS], page=PAGE, out=other, out_lens=lens[ROWS:2 * ROWS], out_refs=refs[BLOCKS:])
    before = [x.clone() for x in (both, lens, refs, parents)]
    for over in (dict(out=table), dict(out=both[:, 1:1 + COLS]), dict(out=both.view(-1)[2 * COLS:].as_strided((ROWS - 1, COLS), both.stride()), parents=parents[1:],
                                                                     out_lens=lens[ROWS:2 * ROWS - 1]),
                 dict(out_lens=lens[:ROWS]), dict(out_lens=lens[1:1 + ROWS]), dict(out_lens=parents), dict(out_lens=both.view(-1)[3:3 + ROWS]),
                 dict(out=torch.zeros(1, COLS, dtype=torch.int32, device=DEV).expand(ROWS, COLS)), dict(out_refs=refs[1:1 + BLOCKS]), dict(out_refs=refs[BLOCKS - 1:2 * BLOCKS - 1]),
                 dict(parents=refs[BLOCKS + 3:BLOCKS + 3 + ROWS])):
        with pytest.raises(ValueError, match="must not"):
            fork_pages(*dict(ok, **over).values())
    assert all(torch.equal(a, b) for a, b in zip(before, (both, lens, refs, parents)))
    want = fork_pages_torch([], table, lens[:ROWS], parents, refs[:BLOCKS], PAGE)
    fork_pages(*ok.values())
    assert torch.equal(other, want[0]) and torch.equal(ok["out_lens"], want[1]) and torch.equal(ok["out_refs"], want[2])


def test_resize():
    both, table, other, lens, refs = tables()
    new = ints([60, 0, 70, 35])
    ok = dict(table=table, lens=lens[:ROWS], new=new, refs=refs[:BLOCKS], page=PAGE, out=other, out_refs=refs[BLOCKS:])
    for over in (dict(out=both[:, 1:1 + COLS]), dict(out=both.view(-1)[2 * COLS:].as_strided((ROWS, COLS), (COLS, 1))), dict(out_refs=refs[1:1 + BLOCKS]),
                 dict(out=torch.zeros(1, COLS, dtype=torch.int32, device=DEV).expand(ROWS, COLS)), dict(new=both.view(-1)[COLS:COLS + ROWS]),
                 dict(lens=refs[BLOCKS:BLOCKS + ROWS])):
        with pytest.raises(ValueError, match="must not"):
            resize_pages(*dict(ok, **over).values())
    want = resize_pages_torch(table, lens[:ROWS], new, refs[:BLOCKS], PAGE)
    resize_pages(*ok.values())
    assert torch.equal(other, want[0]) and torch.equal(ok["out_refs"], want[1])
    resize_pages(*dict(ok, out=None, out_refs=None).values())
    assert torch.equal(table, want[0]) and torch.equal(refs[:BLOCKS], want[1])


def test_keep():
    both, table, other, lens, refs = tables()
    cs = list(make_cache(BLOCKS, PAGE, 2, 64, DEV))
    starts, keep = ints([0, 2, 4, 6, 8]), torch.full((ROWS,), 2, dtype=torch.int64, device=DEV)
    for out_lens in (lens[:ROWS], lens[2:2 + ROWS], starts[:ROWS], starts[1:], keep.view(torch.int32)[3:3 + ROWS], both.view(-1)[1:1 + ROWS]):
        with pytest.raises(ValueError, match="must not"):
            keep_drafted(cs, table, lens[:ROWS], starts, keep, PAGE, out_lens)
    assert keep_drafted(cs, table, lens[:ROWS], starts, keep, PAGE, lens[ROWS:2 * ROWS]).tolist() == [39, 32, 47, 34]
