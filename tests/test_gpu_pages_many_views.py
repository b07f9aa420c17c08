"""GPU checks of the page operators on more caches than a launch takes: every byte of every view."""
import pytest
import torch

from vllm_exact.int8_cache import make_cache
from vllm_exact.pages import fork_pages, fork_pages_torch, keep_drafted, keep_drafted_torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE, COLS, BLOCKS, ROWS = 8, 5, 400, 50


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def caches(count, g):
    """8-bit keys, values and scales, 16-bit ones, and rows of 5 bytes, in turn."""
    out = []
    while len(out) < count:
        out += list(make_cache(BLOCKS, PAGE, 2, 16, DEV))
        out += list(torch.empty(BLOCKS, PAGE, 2, 32, device=DEV, dtype=torch.bfloat16).split(16, dim=-1))
        out.append(torch.empty(BLOCKS, PAGE, 1, 7, device=DEV, dtype=torch.int8)[..., 1:6])
    for c in out[:count]:
        c.copy_(torch.randint(-127, 127, c.shape, generator=g))
    return out[:count]


def rows_of(lens, g):
    order, at = torch.randperm(BLOCKS, generator=g).tolist(), 0
    table = torch.full((len(lens), COLS), -1, dtype=torch.int32)
    for r, n in enumerate(lens):
        pages = -(-n // PAGE)
        table[r, :pages] = torch.tensor(order[at:at + pages], dtype=torch.int32)
        at += pages
    return table.to(DEV), torch.bincount(table[table >= 0].long(), minlength=BLOCKS).to(DEV, torch.int32)


@pytest.mark.parametrize("views", [32, 33, 72])
def test_fork(views):
    g = torch.Generator().manual_seed(views)
    lens, parents = torch.randint(0, PAGE * COLS, (ROWS,), generator=g).tolist(), torch.randint(0, ROWS, (ROWS + 20,), generator=g).tolist()
    table, refs = rows_of(lens, g)
    cs = caches(views, g)
    said, before = [c.clone() for c in cs], [c.clone() for c in cs]
    want = fork_pages_torch(said, table, ints(lens), ints(parents), refs, PAGE)
    out, out_lens = torch.empty(len(parents), COLS, dtype=torch.int32, device=DEV), torch.empty(len(parents), dtype=torch.int32, device=DEV)
    missing = fork_pages(cs, table, ints(lens), ints(parents), refs, PAGE, out, out_lens)
    assert torch.equal(out, want[0]) and torch.equal(out_lens, want[1]) and torch.equal(refs, want[2]) and int(missing) == want[3] == 0
    for i, (a, b, old) in enumerate(zip(cs, said, before)):
        assert torch.equal(a, b), i
        assert not torch.equal(a, old), i  # something was copied in every view


@pytest.mark.parametrize("views", [32, 33, 72])
def test_keep(views):
    g = torch.Generator().manual_seed(100 + views)
    counts = torch.randint(0, 20, (ROWS,), generator=g).tolist()
    lens = [c + int(torch.randint(0, PAGE * COLS - c, (1,), generator=g)) for c in counts]
    table, _ = rows_of(lens, g)
    cs = caches(views, g)
    said, before = [c.clone() for c in cs], [c.clone() for c in cs]
    starts = ints([0] + counts).cumsum(0).to(torch.int32)
    keep = torch.randint(0, 1 << 20, (ROWS,), generator=g).to(DEV)
    want = keep_drafted_torch(said, table, ints(lens), starts, keep, PAGE)
    assert torch.equal(keep_drafted(cs, table, ints(lens), starts, keep, PAGE, torch.empty_like(want)), want)
    for i, (a, b, old) in enumerate(zip(cs, said, before)):
        assert torch.equal(a, b), i
        assert not torch.equal(a, old), i
