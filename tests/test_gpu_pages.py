"""GPU checks of the page operators against their statements: tables, counts and every byte of the caches are equal."""
import pytest
import torch

from vllm_exact.int8_cache import make_cache
from vllm_exact.pages import (copy_pages, fork_pages, fork_pages_torch, keep_drafted, keep_drafted_torch, resize_pages,
                              resize_pages_torch)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def fill(t, g):
    t.copy_(torch.randint(-127, 127, t.shape, generator=g))


def caches(blocks, page, g, KV=2, D=64, layers=1):
    """An 8-bit cache with scales, a 16-bit one of token-major pages, and rows whose bytes fit no wide unit."""
    out = []
    for _ in range(layers):
        out += list(make_cache(blocks, page, KV, D, DEV))
        out += list(torch.empty(blocks, page, KV, 2 * D, device=DEV, dtype=torch.bfloat16).split(D, dim=-1))
        out.append(torch.empty(blocks, page, KV, 7, device=DEV, dtype=torch.int8)[..., 1:6])
        out.append(torch.empty(blocks, page, KV, device=DEV, dtype=torch.float16))
    for c in out:
        fill(c, g)
    return out


def clone(cs):
    return [c.clone() for c in cs]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def rows_of(lens, page, cols, blocks, g, shared=0):
    """A table of permuted pages; the first `shared` pages of all rows are the first row's."""
    order, at = torch.randperm(blocks, generator=g).tolist(), 0
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    for r, n in enumerate(lens):
        for j in range(-(-n // page)):
            if r and j < shared and j < n // page and table[0, j] >= 0:
                table[r, j] = table[0, j]
            else:
                table[r, j] = order[at]
                at += 1
    refs = torch.bincount(table[table >= 0].long(), minlength=blocks).to(torch.int32)
    return table.to(DEV), refs.to(DEV)


def fork(cs, table, lens, parents, refs, page, new_rows=None, **kw):
    out = torch.full((len(parents), table.shape[1]), 77, dtype=torch.int32, device=DEV)
    out_lens = torch.full((len(parents),), 77, dtype=torch.int32, device=DEV)
    missing = fork_pages(cs, table, lens, parents, refs, page, out, out_lens, **kw)
    return out, out_lens, missing


@pytest.mark.parametrize("page,cols,lens,parents", [
    (16, 8, [100, 33, 16, 0, 128], [0, 0, 1, 2, 2, 2, 4, 3]),
    (16, 8, [100, 33, 16, 0, 128], [4, 3, 2, 1, 0]),
    (16, 8, [100, 33, 16, 0, 128], [1, 1, 1, 1, 1, -1, 0, 99, -5]),
    (7, 20, [1, 139, 140], [0, 0, 1, 1, 2, 2]),
    (528, 2, [700, 5], [1, 0, 1, 0]),
    (1, 5, [5, 3], [1, 1, 0]),
    (16, 8, [], [-1, 0]),
    (16, 8, [20, 30], []),
])
@pytest.mark.parametrize("shared", [0, 3])
def test_fork(page, cols, lens, parents, shared):
    g = torch.Generator().manual_seed(0)
    blocks = sum(-(-n // page) for n in lens) + len(parents) + 3
    table, refs = rows_of(lens, page, cols, blocks, g, shared)
    cs = caches(blocks, page, g)
    said = clone(cs)
    want = fork_pages_torch(said, table, ints(lens), ints(parents), refs, page)
    out_refs = torch.empty_like(refs)
    before = refs.clone()
    out, out_lens, missing = fork(cs, table, ints(lens), ints(parents), refs, page, out_ref_count=out_refs)
    assert torch.equal(out, want[0]) and torch.equal(out_lens, want[1]) and torch.equal(out_refs, want[2]) and int(missing) == want[3] == 0
    assert same(cs, said) and torch.equal(refs, before)
    fork(cs, table, ints(lens), ints(parents), refs, page)  # the same pages again, counts in place
    assert torch.equal(refs, want[2]) and same(cs, said)


def test_fork_of_pages_that_others_hold_and_too_few_free_ones():
    g = torch.Generator().manual_seed(1)
    lens, page = [40, 24, 9], 16
    table, refs = rows_of(lens, page, 4, 12, g)
    refs[table[0, 2]] += 1  # a page of the end that somebody else holds: every child copies
    refs[(refs == 0).nonzero()[3:, 0]] = 1
    parents = [0, 0, 1, 1, 2, 2]
    for spare in (False, True):
        if spare:  # one page less than they want
            refs[(refs == 0).nonzero()[0, 0]] = 5
        cs = caches(12, page, g)
        said = clone(cs)
        want = fork_pages_torch(said, table, ints(lens), ints(parents), refs, page)
        counts = refs.clone()
        out, out_lens, missing = fork(cs, table, ints(lens), ints(parents), counts, page)
        assert torch.equal(out, want[0]) and torch.equal(out_lens, want[1]) and torch.equal(counts, want[2])
        assert int(missing) == want[3] == (2 if spare else 1) and same(cs, said)


def test_fork_of_two_rows_that_share_their_end():
    """Both let go of the page while children copy it: it is not given out in the same call."""
    g = torch.Generator().manual_seed(2)
    table, refs = ints([[3, 5], [4, 5]]), torch.zeros(6, dtype=torch.int32, device=DEV)
    refs[[3, 4]], refs[5] = 1, 2
    cs = caches(6, 16, g)
    said = clone(cs)
    want = fork_pages_torch(said, table, ints([20, 20]), ints([0, 1]), refs, 16)
    out, _, missing = fork(cs, table, ints([20, 20]), ints([0, 1]), refs, 16)
    assert out.tolist() == want[0].tolist() == [[3, 0], [4, 1]] and torch.equal(refs, want[2]) and refs[5] == 0 and same(cs, said)


def test_fork_with_bad_pages_and_lengths():
    g = torch.Generator().manual_seed(3)
    table, lens = ints([[1, 99, -1], [2, -7, 1 << 30], [0, 3, 4]]), ints([40, 20, 1 << 30])
    refs = ints([1, 1, 1, 1, 1, 0, 0, 0])
    cs = caches(8, 16, g)
    said = clone(cs)
    parents = ints([0, 0, 1, 1, 2, 2])
    want = fork_pages_torch(said, table, lens, parents, refs, 16)
    out, out_lens, missing = fork(cs, table, lens, parents, refs, 16)
    assert torch.equal(out, want[0]) and torch.equal(out_lens, want[1]) and torch.equal(refs, want[2]) and int(missing) == want[3] and same(cs, said)


def test_fork_many_caches_and_rows():
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 40, (3000,), generator=g).tolist()
    parents = torch.randint(0, 3000, (4001,), generator=g).tolist()
    table, refs = rows_of(lens, 8, 5, 20000, g)
    cs = caches(20000, 8, g, KV=1, D=16, layers=9)  # more views than a launch takes
    said = clone(cs[:2] + cs[-1:])
    want = fork_pages_torch(said, table, ints(lens), ints(parents), refs, 8)
    before = clone(cs[2:-1])
    out, out_lens, missing = fork(cs, table, ints(lens), ints(parents), refs, 8)
    assert torch.equal(out, want[0]) and torch.equal(out_lens, want[1]) and torch.equal(refs, want[2]) and int(missing) == 0
    assert same(cs[:2] + cs[-1:], said)
    moved = (cs[0] != 0).flatten(1).any(1)  # wherever the first view is filled, the others are
    for c, old in zip(cs[2:-1], before):
        for r in range(0, 4001, 501):
            if lens[parents[r]] % 8:
                a, b = int(table[parents[r], lens[parents[r]] // 8]), int(out[r, lens[parents[r]] // 8])
                assert torch.equal(c[b], old[a])
    assert moved.all()


@pytest.mark.parametrize("page,cols,lens,new", [
    (16, 6, [0, 20, 96, 33, 40], [17, 0, 96, 34, 96]),
    (16, 6, [16, 32, 95], [17, 31, 200]),
    (3, 40, [0] * 50, list(range(50))),
    (16, 6, [], []),
    (16, 6, [10, -5, 50], [-3, 20, 50]),
])
@pytest.mark.parametrize("in_place", [True, False])
def test_resize(page, cols, lens, new, in_place):
    g = torch.Generator().manual_seed(5)
    blocks = 600
    table, refs = rows_of([max(0, n) for n in lens], page, cols, blocks, g)
    want = resize_pages_torch(table, ints(lens), ints(new), refs, page)
    if in_place:
        missing = resize_pages(table, ints(lens), ints(new), refs, page)
        got = table, refs
    else:
        got = torch.full_like(table, 77), torch.full_like(refs, 77)
        before = table.clone(), refs.clone()
        missing = resize_pages(table, ints(lens), ints(new), refs, page, *got)
        assert torch.equal(table, before[0]) and torch.equal(refs, before[1])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and int(missing) == want[2] == 0


@pytest.mark.parametrize("blocks", [1, 7, 1000, 8192, 8193, 70001])
def test_resize_takes_the_lowest_free_pages(blocks):
    g = torch.Generator().manual_seed(6)
    refs = (torch.rand(blocks, generator=g) < 0.7).to(torch.int32).to(DEV)
    for rows, each in ((1, 3), (300, 40)):
        table = torch.full((rows, 50), -1, dtype=torch.int32, device=DEV)
        lens, new = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.full((rows,), each * 4, dtype=torch.int32, device=DEV)
        counts = refs.clone()
        missing = resize_pages(table, lens, new, counts, 4)
        free = (refs == 0).nonzero()[:, 0].tolist()
        want = (free + [-1] * (rows * each))[:rows * each]
        assert table[:, :each].flatten().tolist() == want and (table[:, each:] == -1).all()
        assert int(missing) == max(0, rows * each - len(free)) and int(counts.sum() - refs.sum()) == min(rows * each, len(free))


def test_shared_pages_are_freed_with_their_last_holder():
    table, refs = ints([[0, 1], [0, 2]]), ints([2, 1, 1, 0])
    resize_pages(table, ints([32, 32]), ints([0, 32]), refs, 16)
    assert refs.tolist() == [1, 0, 1, 0] and table.tolist() == [[-1, -1], [0, 2]]
    resize_pages(table, ints([0, 32]), ints([0, 0]), refs, 16)
    assert refs.tolist() == [0, 0, 0, 0]


MASKS = [0b1, 0, 0b1010101, -1, (1 << 63) - 1 - 0b100, -(1 << 63), 0b1100, 0b110]


@pytest.mark.parametrize("page", [16, 5, 528])
@pytest.mark.parametrize("KV,D", [(1, 64), (3, 256)])
def test_keep(page, KV, D):
    g = torch.Generator().manual_seed(7)
    counts = [1, 3, 7, 64, 64, 64, 0, 2]
    context = [0, 15, 33, 600, 1, 100, 9, 31]
    lens = [c + n for c, n in zip(context, counts)]
    cols = -(-max(lens) // page)
    blocks = sum(-(-n // page) for n in lens) + 2
    table, _ = rows_of(lens, page, cols, blocks, g)
    cs = caches(blocks, page, g, KV, D)
    said = clone(cs)
    starts, keep = ints([0] + counts).cumsum(0).to(torch.int32), ints(MASKS, torch.int64)
    out = torch.empty(8, dtype=torch.int32, device=DEV)
    assert keep_drafted(cs, table, ints(lens), starts, keep, page, out) is out
    assert torch.equal(out, keep_drafted_torch(said, table, ints(lens), starts, keep, page)) and same(cs, said)
    assert out.tolist() == [1, 15, 37, 664, 63, 101, 9, 32]


def test_keep_of_bad_requests_and_pages():
    g = torch.Generator().manual_seed(8)
    lens, starts = ints([70, 3, 40, 40]), ints([0, 65, 70, 73, 76])  # 65 nodes; more nodes than tokens; a bad page; beyond the table
    table = ints([[0, 1, 2, 3], [4, -1, -1, -1], [5, 6, 99, -1], [7, 8, -1, -1]])
    cs = caches(9, 16, g)
    said = clone(cs)
    out = torch.empty(4, dtype=torch.int32, device=DEV)
    keep = ints([0b10] * 4, torch.int64)
    keep_drafted(cs, table, lens, starts, keep, 16, out)
    assert torch.equal(out, keep_drafted_torch(said, table, lens, starts, keep, 16)) and same(cs, said)
    assert out.tolist() == [70, 3, 38, 38]


def test_copy():
    g = torch.Generator().manual_seed(9)
    for page, KV, D in ((16, 2, 64), (528, 1, 256), (1, 3, 128)):
        cs = caches(12, page, g, KV, D)
        said = clone(cs)
        source, target = [0, 1, 2, -1, 3, 50, 0, 4], [7, 8, 7, 9, 12, 9, 10, -2]  # page 7 twice: the later pair counts
        for c in said:
            c[8], c[7], c[10] = c[1], c[2], c[0]
        copy_pages(cs, page, ints(source), ints(target))
        assert same(cs, said)
    copy_pages([], 16, ints([0]), ints([1]))
    copy_pages(cs, 1, ints([]), ints([]))


def test_captured_and_replayed():
    g = torch.Generator().manual_seed(10)
    lens, parents, page = [100, 33, 16, 50], [0, 0, 3, 3], 16
    table, refs = rows_of(lens, page, 8, 40, g)
    cs = caches(40, page, g)
    lens, parents, first = ints(lens), ints(parents), clone(cs)
    new, new_lens, counts = torch.empty_like(table), torch.empty_like(lens), torch.empty_like(refs)
    starts, keep, kept = ints([0, 2, 5, 5, 8]), ints([2, 4, 0, 5], torch.int64), torch.empty_like(lens)

    def step():
        a = fork_pages(cs, table, lens, parents, refs, page, new, new_lens, counts)
        keep_drafted(cs, new, new_lens, starts, keep, page, kept)
        return a, resize_pages(new, new_lens, kept + 40, counts, page)

    step()
    want = [x.clone() for x in (new, new_lens, counts, kept)] + clone(cs)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    for _ in range(3):
        for a, b in zip(cs, first):
            a.copy_(b)
        new.zero_(), counts.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same([new, new_lens, counts, kept] + cs, want)


def test_refusals():
    g = torch.Generator().manual_seed(11)
    table, refs = rows_of([20, 30], 16, 4, 10, g)
    cs, lens, parents = caches(10, 16, g), ints([20, 30]), ints([0, 1])
    out, out_lens = torch.empty_like(table), torch.empty_like(lens)
    ok = dict(caches=cs, table=table, lens=lens, parents=parents, refs=refs, page=16, out=out, out_lens=out_lens)
    for over, kind in ((dict(caches=cs[0]), ValueError), (dict(caches=["x"]), TypeError), (dict(caches=3), TypeError), (dict(caches=[cs[0].transpose(1, 3)]), ValueError),
                       (dict(caches=[cs[0], cs[1][:5]]), ValueError), (dict(caches=[cs[0].cpu()]), ValueError), (dict(table=table.long()), ValueError),
                       (dict(lens=lens.long()), ValueError), (dict(lens=lens[:1]), ValueError), (dict(parents=parents[:1]), ValueError),
                       (dict(refs=refs[:9]), ValueError), (dict(refs=refs.long()), ValueError), (dict(page=0), ValueError), (dict(page=8), ValueError),
                       (dict(out=table), ValueError), (dict(out=out[:, :3]), ValueError), (dict(out_lens=lens), ValueError)):
        with pytest.raises(kind):
            fork_pages(*dict(ok, **over).values())
    for over, kind in ((dict(out=out[:1]), ValueError), (dict(out=table[:, ::2]), ValueError), (dict(lens=lens[:1]), ValueError), (dict(new=lens.long()), ValueError),
                       (dict(page=-1), ValueError), (dict(out_refs=refs[:3]), ValueError)):
        with pytest.raises(kind):
            resize_pages(*dict(dict(table=table, lens=lens, new=lens, refs=refs, page=16, out=out, out_refs=None), **over).values())
    starts, keep = ints([0, 1, 2]), ints([1, 1], torch.int64)
    for over, kind in ((dict(keep=keep.int()), ValueError), (dict(starts=starts[:2]), ValueError), (dict(out_lens=lens), ValueError), (dict(page="x"), TypeError)):
        with pytest.raises(kind):
            keep_drafted(*dict(dict(caches=cs, table=table, lens=lens, starts=starts, keep=keep, page=16, out_lens=out_lens), **over).values())
    for over in (dict(source=parents.long()), dict(target=parents[:1])):
        with pytest.raises(ValueError):
            copy_pages(*dict(dict(caches=cs, page=16, source=parents, target=parents), **over).values())
    big = torch.empty(8193, 1, dtype=torch.int32, device=DEV)
    with pytest.raises(NotImplementedError):
        resize_pages(big, big[:, 0].contiguous(), big[:, 0].contiguous(), refs, 16)


def test_pages_far_apart():
    """Pages past 2^32 bytes from each other: copied, forked and compacted."""
    page, KV, D, stride = 4, 2, 64, (1 << 31) + 64
    far = torch.empty(3 * stride + page * KV * D, device=DEV, dtype=torch.int8).as_strided((4, page, KV, D), (stride, KV * D, D, 1))
    fill(far, torch.Generator().manual_seed(11))
    copy_pages([far], page, ints([0]), ints([3]))
    assert torch.equal(far[3], far[0])
    table, lens, refs = ints([[3, 0]]), ints([6]), ints([1, 0, 0, 1])
    out, out_lens, missing = fork([far], table, lens, ints([0, 0]), refs, page)  # the second row's end is copied to page 1
    assert out.tolist() == [[3, 0], [3, 1]] and out_lens.tolist() == [6, 6] and int(missing) == 0 and torch.equal(far[1], far[0])
    assert refs.tolist() == [1, 1, 0, 2]
    fill(far, torch.Generator().manual_seed(12))
    said = far.contiguous()
    kept = keep_drafted_torch([said], out[:1], lens[:1], ints([0, 5]), ints([0b11000], torch.int64), page)
    got = keep_drafted([far], out[:1], lens[:1], ints([0, 5]), ints([0b11000], torch.int64), page, torch.empty_like(lens))
    assert torch.equal(got, kept) and torch.equal(far, said)


@pytest.mark.parametrize("blocks", [1023, 1024, 1025, 4096, 4097, 8191, 16500])
@pytest.mark.parametrize("rows", [1, 20, 33])
@pytest.mark.parametrize("in_place", [True, False])
def test_resize_by_one_workgroup_or_several(blocks, rows, in_place):
    """Both sides of the sizes at which a resize is one launch, with free pages in between and fewer than are wanted."""
    page, cols = 4, 50
    g = torch.Generator().manual_seed(blocks + rows)
    lens = torch.randint(0, cols * page // 2, (rows,), generator=g).tolist()
    table, refs = rows_of(lens, page, cols, blocks, g)
    refs += (torch.rand(blocks, generator=g) < 0.7).to(torch.int32).to(DEV)  # others hold them
    new = torch.randint(0, cols * page + 1, (rows,), generator=g)
    lens, new = ints(lens), new.to(torch.int32).to(DEV)
    want = resize_pages_torch(table.cpu(), lens.cpu(), new.cpu(), refs.cpu(), page)
    if in_place:
        missing = resize_pages(table, lens, new, refs, page)
        out, counts = table, refs
    else:
        out, counts = torch.full_like(table, 5), torch.full_like(refs, 5)
        before = table.clone(), refs.clone()
        missing = resize_pages(table, lens, new, refs, page, out, counts)
        assert torch.equal(table, before[0]) and torch.equal(refs, before[1])
    assert torch.equal(out.cpu(), want[0]) and torch.equal(counts.cpu(), want[1]) and int(missing) == want[2]
