"""GPU checks of copy_pages with many pairs: of those with one target the last counts, wherever they are, and the work grows as the pairs."""
import pytest
import torch

from vllm_exact.pages import copy_pages

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 5000])
@pytest.mark.parametrize("views", [1, 33])
def test_the_last_pair_of_a_target_counts(n, views):
    g = torch.Generator().manual_seed(n)
    blocks, page = 600, 2
    source = torch.randint(-3, 305, (n,), generator=g)  # pages from 0 on are read, those from 300 on written; some are none
    target = torch.randint(295, 605, (n,), generator=g)
    source[source >= 300] = 1 << 30
    target[target < 300] = -1
    caches = [torch.randint(-100, 100, (blocks, page, 2, 8), generator=g, dtype=torch.int16).to(DEV) for _ in range(views)]
    last = {}
    for a, b in zip(source.tolist(), target.tolist()):
        if 0 <= a < blocks and 0 <= b < blocks:
            last[b] = a
    want = [c.clone() for c in caches]
    for c in want:
        c[list(last)] = c[list(last.values())]
    copy_pages(caches, page, ints(source.tolist()), ints(target.tolist()))
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


def test_the_work_grows_as_the_pairs():
    """16 times as many pairs take at most 64 times as long (they would take 256 times, did every pair look through all others)."""
    few, many = 1 << 13, 1 << 17
    cache = torch.zeros(2 * many, 1, 1, 16, dtype=torch.int8, device=DEV)
    source = torch.arange(many, dtype=torch.int32, device=DEV)
    target = source + many

    def time(n):
        times = []
        for _ in range(7):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            copy_pages([cache], 1, source[:n], target[:n])
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[3]

    time(few)
    assert time(many) <= 64 * time(few)
