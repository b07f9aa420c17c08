"""GPU checks of the 8-bit cache: the whole numbers and scales of a write equal the definition in float64, a read gives
q * scale (one fp32 rounding, then one to the output's type)."""
import pytest
import torch

from vllm_exact.int8_cache import dequantize_torch, make_cache, quantize_torch, read_cache, write_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows(T, KV, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, KV, D, generator=g) * 10 ** (torch.rand(T, KV, 1, generator=g) * 6 - 3)
    return x.to(dtype).to(DEV)


def definition(x):
    """(q, top / 127) in float64."""
    x = x.double().cpu()
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(127 * x / torch.where(top > 0, top, 1.0)), top[..., 0] / 127


def table(lens, page, seed=0, spare=3):
    """Block tables of permuted blocks, the pool's size, and the slots of all tokens."""
    g = torch.Generator().manual_seed(seed)
    cols = max(1, max(-(-n // page) for n in lens))
    blocks = cols * len(lens) + spare
    bt = torch.randperm(blocks, generator=g)[:cols * len(lens)].view(len(lens), cols)
    slots = torch.cat([bt[i][torch.arange(n) // page] * page + torch.arange(n) % page for i, n in enumerate(lens)])
    return bt.to(torch.int32).to(DEV), blocks, slots.to(DEV)


def starts(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,KV,D,page", [(1, 1, 64, 16), (37, 8, 128, 16), (130, 3, 256, 528), (61, 2, 64, 7)])
def test_write_gives_the_definition(dtype, T, KV, D, page):
    k, v = rows(T, KV, D, dtype, 1), rows(T, KV, D, dtype, 2)
    if T > 2:
        k[1], v[2] = 0, 0
    _, blocks, slots = table([T], page)
    cache = make_cache(blocks, page, KV, D, DEV)
    write_cache(k, v, *cache, slots)
    for x, q, s in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        want_q, want_s = definition(x)
        got_q, got_s = q[slots // page, slots % page].cpu(), s[slots // page, slots % page].cpu()
        if dtype == torch.float32:  # 127 x is rounded once: whole numbers next to a tie may be the tie's other side
            assert (got_q.double() - want_q).abs().max() <= 1
            exact = 127 * x.double().cpu() / torch.where(want_s > 0, want_s * 127, 1.0)[..., None]
            assert ((got_q.double() - exact).abs() <= 0.5 + 127 * 2.0 ** -22).all()
        else:
            assert torch.equal(got_q.double(), want_q)
        assert ((got_s.double() - want_s).abs() <= want_s * 2.0 ** -24).all()
        assert torch.equal(torch.stack([got_q.float(), got_s[..., None].expand_as(got_q)]),
                           torch.stack([t.float().cpu() if t.dim() == 3 else t[..., None].cpu().expand_as(got_q)
                                        for t in quantize_torch(x)]))
    rest = torch.ones(blocks * page, dtype=torch.bool, device=DEV)
    rest[slots] = False
    assert all(not t.flatten(0, 1)[rest].any() for t in cache)


def test_ties_go_to_even():
    """127 x / top halfway between whole numbers: top = 127 * 2^-7 makes every odd multiple of 2^-8 a tie."""
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=DEV)
    x[0, 0, 0] = 127 / 128
    x[0, 0, 1:33] = torch.arange(32, device=DEV) / 128 + 1 / 256
    cache = make_cache(1, 16, 1, 64, DEV)
    write_cache(x, -x, *cache, torch.zeros(1, dtype=torch.int64, device=DEV))
    want = torch.round(torch.arange(32) + 0.5)
    assert torch.equal(cache[0][0, 0, 0, 1:33].cpu().float(), want)
    assert torch.equal(cache[1][0, 0, 0, 1:33].cpu().float(), -want)


def test_padding_slots_special_rows_and_unaligned_rows():
    k, v = rows(9, 2, 64, torch.bfloat16, 3), rows(9, 2, 64, torch.bfloat16, 4)
    k[2, 0, 5], k[3, 1, 63], v[4, 0, 0] = float("nan"), float("inf"), -float("inf")
    slots = torch.tensor([3, -1, 5, 6, 7, 64, 1 << 40, -(1 << 50), 63], device=DEV)
    cache = make_cache(4, 16, 2, 64, DEV)
    write_cache(k, v, *cache, slots)
    bt = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    got = read_cache(*cache, bt, starts([64]), *(torch.empty(64, 2, 64, device=DEV) for _ in "kv"))
    for x, y in ((k, got[0]), (v, got[1])):
        want = torch.zeros_like(y)
        for t, s in ((0, 3), (2, 5), (3, 6), (4, 7), (8, 63)):
            want[s] = dequantize_torch(*quantize_torch(x[t]))
        assert torch.equal(y.nan_to_num(1e9), want.nan_to_num(1e9))
    assert torch.isnan(got[0][5, 0]).all() and torch.isnan(got[0][6, 1]).all() and torch.isnan(got[1][7, 0]).all()
    assert torch.isfinite(got[0][5, 1]).all() and torch.isfinite(got[0][6, 0]).all()
    again = make_cache(4, 16, 2, 64, DEV)
    odd = torch.empty(9, 2, 67, dtype=torch.bfloat16, device=DEV)  # rows at odd elements
    odd[..., 1:65] = k
    write_cache(odd[..., 1:65], v, *again, slots)
    assert all(torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)) for a, b in zip(cache, again))


@pytest.mark.parametrize("magnitude", [1e-40, 1e-30, 1.0, 1e30, 3e38])
def test_magnitudes(magnitude):
    x = (rows(4, 1, 64, torch.float32, 8).clamp(-1, 1) * magnitude).contiguous()
    cache = make_cache(1, 16, 1, 64, DEV)
    write_cache(x, x, *cache, torch.arange(4, device=DEV))
    q, s = quantize_torch(x.cpu())
    assert torch.equal(cache[0][0, :4, 0].cpu(), q[:, 0]) and torch.equal(cache[2][0, :4, 0].cpu(), s[:, 0])
    assert q.abs().amax() == 127


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lens,KV,D,page", [((1,), 1, 64, 16), ((0, 5, 0, 33, 16), 8, 128, 16), ((529, 3), 2, 256, 528),
                                            (tuple(range(130)), 1, 64, 5)])
def test_read(dtype, lens, KV, D, page):
    bt, blocks, slots = table(lens, page, seed=5)
    cache = make_cache(blocks, page, KV, D, DEV)
    k, v = rows(sum(lens), KV, D, torch.bfloat16, 6), rows(sum(lens), KV, D, torch.bfloat16, 7)
    write_cache(k, v, *cache, slots)
    outs = [torch.full((sum(lens) + 5, KV, D), 3.0, device=DEV, dtype=dtype) for _ in "kv"]
    read_cache(*cache, bt, starts(lens), *outs)
    for x, y in zip((k, v), outs):
        assert torch.equal(y[:-5], dequantize_torch(*quantize_torch(x)).to(dtype))
        assert (y[-5:] == 3).all()
    # ranges: the last tokens of each sequence, into strided rows
    first = torch.tensor([n // 3 for n in lens], dtype=torch.int32, device=DEV)
    part = [n - n // 3 for n in lens]
    wide = [torch.zeros(sum(part), KV, 2 * D, device=DEV, dtype=dtype)[..., D:] for _ in "kv"]
    read_cache(*cache, bt, starts(part), *wide, first=first)
    at = torch.cat([torch.arange(sum(lens[:i]) + n // 3, sum(lens[:i + 1])) for i, n in enumerate(lens)]).to(DEV)
    assert all(torch.equal(w, o[at]) for w, o in zip(wide, outs))


def test_bad_blocks_and_rows_past_the_table_read_as_nan():
    cache = make_cache(3, 16, 1, 64, DEV)
    write_cache(*(rows(48, 1, 64, torch.bfloat16, s) for s in (1, 2)), *cache, torch.arange(48, device=DEV))
    bt = torch.tensor([[0, 3, 2], [1, -1, 2]], dtype=torch.int32, device=DEV)
    k, v = read_cache(*cache, bt, starts([50, 48]), *(torch.zeros(98, 1, 64, device=DEV) for _ in "kv"))
    bad = torch.zeros(98, dtype=torch.bool)
    bad[16:32], bad[48:50], bad[66:82] = True, True, True
    for y in (k, v):
        assert torch.equal(torch.isnan(y).all(-1)[:, 0].cpu(), bad) and torch.equal(torch.isnan(y).any(-1)[:, 0].cpu(), bad)
    first = torch.tensor([-1, 40], dtype=torch.int32, device=DEV)
    k, _ = read_cache(*cache, bt, starts([2, 10]), *(torch.zeros(12, 1, 64, device=DEV) for _ in "kv"), first=first)
    assert torch.isnan(k[0]).all() and torch.isfinite(k[1:10]).all() and torch.isnan(k[10:]).all()


def test_a_cache_past_32_bit_offsets():
    page, KV, D = 16, 8, 128
    blocks = (5 << 30) // (page * KV * 2 * D)
    pool = torch.empty(blocks, KV, page, 2 * D, dtype=torch.int8, device=DEV)
    scales = torch.empty(blocks, KV, page, 2, device=DEV)
    cache = pool.transpose(1, 2).split(D, dim=-1) + scales.transpose(1, 2).unbind(-1)
    slots = torch.tensor([0, blocks * page - 1, blocks * page // 2], device=DEV)
    k, v = rows(3, KV, D, torch.float16, 1), rows(3, KV, D, torch.float16, 2)
    write_cache(k, v, *cache, slots)
    bt = (slots // page).to(torch.int32)[:, None]
    got = read_cache(*cache, bt, starts([1, 1, 1]), *(torch.empty(3, KV, D, device=DEV) for _ in "kv"),
                     first=(slots % page).to(torch.int32))
    for x, y in zip((k, v), got):
        assert torch.equal(y, dequantize_torch(*quantize_torch(x)))


def test_graph_replays():
    k, v = rows(20, 2, 128, torch.bfloat16, 1), rows(20, 2, 128, torch.bfloat16, 2)
    bt, blocks, slots = table([20], 16)
    cache = make_cache(blocks, 16, 2, 128, DEV)
    outs = [torch.empty(20, 2, 128, device=DEV) for _ in "kv"]
    cu = starts([20])
    write_cache(k, v, *cache, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write_cache(k, v, *cache, slots)
        read_cache(*cache, bt, cu, *outs)
    for i in range(4):
        k.copy_(rows(20, 2, 128, torch.bfloat16, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], dequantize_torch(*quantize_torch(k))), i
