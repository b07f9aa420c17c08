"""GPU checks of beam selection, pages and linear attention at the largest sizes that they accept."""
import pytest
import torch

from linear64 import bounds, linear64
from vllm_exact.beam import beam_select, beam_select_torch
from vllm_exact.linear_attn import linear_prompt, linear_step
from vllm_exact.pages import fork_pages, fork_pages_torch, keep_drafted, keep_drafted_torch, resize_pages, resize_pages_torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


@pytest.mark.parametrize("n,beams,V,dtype", [
    (2, 1024, 50, torch.bfloat16),        # beams
    (1, 512, 8 * 8192, torch.float32),    # slices of a request, 8 of each beam
    (1, 1, 4096 * 8192, torch.float32),   # and of one beam
    (1, 2, 4096 * 4096 - 5, torch.bfloat16),
    (3, 256, 8193, torch.float16),
])
@pytest.mark.parametrize("kind", ["random", "few values"])
def test_beams(n, beams, V, dtype, kind):
    g = torch.Generator(device=DEV).manual_seed(beams)
    logits = torch.empty(n * beams, V, device=DEV, dtype=dtype).normal_(generator=g)
    if kind == "few values":
        logits.round_()
    scores = torch.rand(n * beams, device=DEV, generator=g) * -4
    scores[::3] = -1e30
    for count in (1, 64):
        got = beam_select(logits, scores, beams, torch.empty(n, count, device=DEV), torch.empty(n, count, device=DEV, dtype=torch.int32),
                          torch.empty(n, count, device=DEV, dtype=torch.int64))
        if beams * V <= 1 << 22:
            want = beam_select_torch(logits.cpu(), scores.cpu(), beams, count)
            parents, tokens = want[1].to(DEV), want[2].to(DEV)
        else:  # row by row: no beam has more than count of the best
            x, kept = logits.double(), []
            for b in range(beams):
                row = x[b] - torch.logsumexp(x[b], 0) if b % 3 else x[b]  # drowned: by the logits alone, behind all others
                top = row.sort(descending=True, stable=True)
                kept += [(1 if b % 3 == 0 else 0, -float(scores[b]) - v if b % 3 else 0.0, b, i, t) for i, (v, t) in enumerate(zip(top.values[:count].tolist(), top.indices[:count].tolist()))]
            kept.sort()
            parents, tokens = ints([k[2] for k in kept[:count]])[None], ints([k[4] for k in kept[:count]], torch.int64)[None]
        assert torch.equal(got[1], parents) and torch.equal(got[2], tokens)


def test_pages_of_8192_rows():
    g = torch.Generator().manual_seed(1)
    rows, page, cols, blocks = 8192, 4, 3, 40000
    lens = torch.randint(0, page * cols + 1, (rows,), generator=g)
    order, pages = torch.randperm(blocks, generator=g), -(-lens // page)
    starts = pages.cumsum(0) - pages
    at = torch.arange(cols)
    table = torch.where(at < pages[:, None], order[(starts[:, None] + at).clamp(max=blocks - 1)], -1).to(torch.int32)
    refs = torch.bincount(table[table >= 0].long(), minlength=blocks).to(torch.int32)
    parents = torch.randint(-1, rows + 1, (rows,), generator=g, dtype=torch.int32)
    cache = torch.randint(-99, 99, (blocks, page, 1, 3), generator=g, dtype=torch.int8)
    said = cache.clone()
    want = fork_pages_torch([said], table, lens.to(torch.int32), parents, refs, page)
    new, new_lens, counts, moved = torch.empty_like(table, device=DEV), torch.empty(rows, dtype=torch.int32, device=DEV), refs.to(DEV), cache.to(DEV)
    missing = fork_pages([moved], table.to(DEV), lens.to(DEV, torch.int32), parents.to(DEV), counts, page, new, new_lens)
    assert torch.equal(new.cpu(), want[0]) and torch.equal(new_lens.cpu(), want[1]) and torch.equal(counts.cpu(), want[2]) and int(missing) == want[3]
    assert torch.equal(moved.cpu(), said)
    longer = torch.randint(0, page * cols + 1, (rows,), generator=g, dtype=torch.int32)
    want = resize_pages_torch(want[0], want[1], longer, want[2], page)
    missing = resize_pages(new, new_lens, longer.to(DEV), counts, page)
    assert torch.equal(new.cpu(), want[0]) and torch.equal(counts.cpu(), want[1]) and int(missing) == want[2]


@pytest.mark.parametrize("heads,bytes_", [(64, 255), (40, 1000), (1, 16), (129, 576)])
def test_kept_rows_of_many_columns(heads, bytes_):
    """More columns than a launch's workgroups take at once: rows of odd bytes are moved one by one, up to 16320 of them."""
    page, blocks = 4, 9
    g = torch.Generator().manual_seed(heads)
    cache = torch.randint(-99, 99, (blocks, page, heads, bytes_), generator=g, dtype=torch.int8)
    table, lens, starts = torch.tensor([[3, 1, 7, 0], [2, 8, 4, 5]], dtype=torch.int32), torch.tensor([16, 13], dtype=torch.int32), torch.tensor([0, 14, 20], dtype=torch.int32)
    keep = torch.tensor([0b10110011001010, 0b101010])
    said, moved = cache.clone(), cache.to(DEV)
    want = keep_drafted_torch([said], table, lens, starts, keep, page)
    got = keep_drafted([moved], table.to(DEV), lens.to(DEV), starts.to(DEV), keep.to(DEV), page, torch.empty(2, dtype=torch.int32, device=DEV))
    assert torch.equal(got.cpu(), want) and torch.equal(moved.cpu(), said)


@pytest.mark.parametrize("step", [False, True])
def test_many_heads_and_sequences(step):
    """Heads that are no multiple of 8 and more than a wave's lanes; thousands of sequences, each with slots of its own."""
    n, H, D = 2500, 3, 64
    g = torch.Generator().manual_seed(3)
    lens = [1] * n if step else torch.randint(0, 4, (n,), generator=g).tolist()
    T = sum(lens)
    q, k, v = (torch.randn(T, h, D, generator=g).bfloat16().to(DEV) for h in (H, 1, 1))
    decay = torch.tensor([-0.1, -1.0, 0.0], device=DEV)
    state, slots = torch.zeros(n, H, D, D, device=DEV), torch.randperm(n, generator=g).to(DEV, torch.int32)
    out = torch.empty(T, H, D, device=DEV)
    if step:
        linear_step(q, k, v, decay, 0.125, out, state, slots, slots)
    else:
        linear_prompt(q, k, v, ints([0] + lens).cumsum(0).to(torch.int32), decay, 0.125, out, state, slots, slots)
    want, ends = linear64(q, k, v, lens, decay, 0.125)
    rows, states = bounds(q, k, v, lens, decay, 0.125)
    assert ((out - want).abs() <= rows + 2.0 ** -133).all() and ((state[slots.long()] - ends).abs() <= states + 2.0 ** -133).all()
    H = 130
    q, k, v = (torch.randn(70, h, D, generator=g).half().to(DEV) for h in (H, 13, 13))
    decay, out = (-torch.rand(H, generator=g)).to(DEV), torch.empty(70, H, D, device=DEV)
    linear_prompt(q, k, v, ints([0, 70]), decay, 0.125, out)
    want, _ = linear64(q, k, v, (70,), decay, 0.125)
    assert ((out - want).abs() <= bounds(q, k, v, (70,), decay, 0.125)[0]).all()
