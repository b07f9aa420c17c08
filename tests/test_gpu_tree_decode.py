"""GPU checks of the attention of drafted tokens against float64.

Tolerance: P is split into two parts of the 16-bit type (bf16: 2^-16 relative to each weight, fp16: 2^-22), scores and
sums are fp32 (attention64.attend64 adds up the terms), the 8-bit scales enter with three fp32 roundings, and the output is
rounded once."""
import pytest
import torch

from attention64 import attend64, check
from vllm_exact import paged_attn
from vllm_exact.int8_cache import make_cache, write_cache
from vllm_exact.tree_attn import tree_decode, tree_decode_torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
CHAIN = object()


def random_masks(counts, g):
    """Itself and its ancestors, for random trees; some nodes hang off the context."""
    out = []
    for n in counts:
        bits = []
        for i in range(n):
            parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
        out += bits
    return torch.tensor([b - (1 << 64) if b >> 63 else b for b in out], dtype=torch.int64)


def make(ctx, nodes, H, KV, D, page, dtype, int8, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens = [c + n for c, n in zip(ctx, nodes)]
    cols = max(1, max(-(-x // page) for x in lens))
    blocks = cols * len(lens) + 2
    bt = torch.randperm(blocks, generator=g)[:cols * len(lens)].view(len(lens), cols).to(torch.int32).to(DEV)
    if int8:
        cache = make_cache(blocks, page, KV, D, DEV)
        k, v = (torch.randn(blocks * page, KV, D, generator=g).to(dtype).to(DEV) for _ in "kv")
        write_cache(k, v, *cache, torch.arange(blocks * page, device=DEV))
    else:
        pool = torch.randn(blocks, KV, page, 2 * D, generator=g).to(dtype).to(DEV)
        cache = pool.transpose(1, 2).split(D, dim=-1) + (None, None)
    q = torch.randn(sum(nodes), H, D, generator=g).to(dtype).to(DEV)
    qsl = torch.tensor([0] + list(nodes)).cumsum(0).to(torch.int32).to(DEV)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return dict(q=q, cache=cache, bt=bt, sl=sl, qsl=qsl, mask=random_masks(nodes, g).to(DEV))


def run(s, out_dtype=torch.float32, max_nodes=None, longest=None, mask=True):
    out = torch.full(s["q"].shape, float("inf"), device=DEV, dtype=out_dtype)
    counts = (s["qsl"][1:] - s["qsl"][:-1])
    k, v, ks, vs = s["cache"]
    tree_decode(s["q"], k, v, s["bt"], s["sl"], s["qsl"], s["mask"] if mask else None, s["q"].shape[2] ** -0.5, out,
                int(counts.max()) if max_nodes is None else max_nodes, int(s["sl"].max()) if longest is None else longest,
                key_scale=ks, value_scale=vs)
    return out


def compare(out, s, mask=True, requests=None, heads=None):
    k, v, ks, vs = s["cache"]
    H, KV, D, page = s["q"].shape[1], k.shape[2], s["q"].shape[2], k.shape[1]
    step = 2.0 ** -16 if ks is not None or s["q"].dtype == torch.bfloat16 else 2.0 ** -22
    starts = s["qsl"].tolist()
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        n, length = hi - lo, int(s["sl"][b])
        if n == 0 or (requests is not None and b not in requests):
            continue
        tok = torch.arange(length, device=DEV)
        at = s["bt"][b].long()[tok // page], tok % page
        keys, vals = k[at].double(), v[at].double()
        if ks is not None:
            keys, vals = keys * ks[at][..., None].double(), vals * vs[at][..., None].double()
        node = torch.arange(n)
        draft = (s["mask"][lo:hi].cpu()[:, None] >> node) & 1 == 1 if mask else node[:, None] >= node
        seen = torch.cat([torch.ones(n, length - n, dtype=torch.bool), draft], dim=1)
        for h in range(H) if heads is None else heads:
            g = h // (H // KV)
            want, bound = attend64(s["q"][lo:hi, h], keys[:, g], vals[:, g], seen, D ** -0.5, step + 3 * 2.0 ** -24,
                                   0.0 if step == 2.0 ** -16 else 2.0 ** -25)
            check(out[lo:hi, h], want, bound, f"request {b} head {h}")


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ctx,nodes,H,KV,page", [
    ((0,), (1,), 8, 8, 16), ((40, 0, 511, 1), (1, 5, 1, 0), 8, 2, 16), ((500, 505, 512, 1030), (8, 7, 9, 3), 4, 1, 528),
    ((300, 31, 990), (64, 33, 50), 2, 2, 7), ((100, 700), (17, 61), 6, 2, 32)])
def test_against_float64(int8, dtype, D, ctx, nodes, H, KV, page):
    s = make(ctx, nodes, H, KV, D, page, dtype, int8, seed=D + len(ctx))
    compare(run(s), s)
    compare(run(s, mask=False), s, mask=False)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16])
def test_output_types_and_a_long_context(out_dtype):
    s = make((5000, 40), (4, 9), 16, 2, 128, 16, torch.bfloat16, True)
    compare(run(s, out_dtype), s)


def test_one_node_agrees_with_paged_decode():
    s = make((700, 2100, 15), (1, 1, 1), 8, 2, 128, 16, torch.bfloat16, False)
    out = torch.empty(3, 8, 128, device=DEV)
    paged_attn.paged_decode(s["q"], *s["cache"][:2], s["bt"], s["sl"], 128 ** -0.5, out, 3, 4096)
    assert (run(s) - out).abs().max() <= 4e-5 + 2.0 ** -16 * 5  # both are within their bounds of the 64-bit result


@pytest.mark.parametrize("int8", [True, False])
def test_bits_do_not_depend_on_the_batch(int8):
    """Other requests, bounds, physical blocks and batch sizes (and with them the kernel's variant) leave the bits."""
    ctx, nodes = (1200, 3, 530, 4000), (3, 64, 9, 1)
    s = make(ctx, nodes, 8, 2, 128, 16, torch.bfloat16, int8, seed=4)
    out = run(s)
    assert torch.equal(run(s, max_nodes=64, longest=9000), out)
    starts = s["qsl"].tolist()
    for b in range(4):
        lo, hi = starts[b], starts[b + 1]
        one = dict(q=s["q"][lo:hi], cache=s["cache"], bt=s["bt"][b:b + 1], sl=s["sl"][b:b + 1],
                   qsl=torch.tensor([0, hi - lo], dtype=torch.int32, device=DEV), mask=s["mask"][lo:hi].contiguous())
        assert torch.equal(run(one), out[lo:hi]), b
    many = dict(s, q=s["q"].repeat(40, 1, 1), bt=s["bt"].repeat(40, 1), sl=s["sl"].repeat(40), mask=s["mask"].repeat(40),
                qsl=torch.tensor([0] + list(nodes) * 40).cumsum(0).to(torch.int32).to(DEV))
    assert torch.equal(run(many), out.repeat(40, 1, 1))


@pytest.mark.parametrize("int8", [True, False])
def test_rows_that_attend_to_nothing_are_zero(int8):
    s = make((0, 0, 20), (3, 40, 2), 4, 2, 64, 16, torch.bfloat16, int8)
    s["mask"][1], s["mask"][3], s["mask"][44] = 0, -1 << 40, 0  # bits past the nodes name no key
    out = run(s)
    assert (out[1] == 0).all() and (out[3] == 0).all() and (out[44] != 0).any()
    compare(out, s)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_specials_of_masked_drafts_do_not_reach_a_row(D, dtype):
    """16-bit cache: a drafted key with an infinity or NaN changes only the rows that attend to it."""
    ctx, n = 500, 40
    s = make((ctx,), (n,), 2, 1, D, 16, dtype, False, seed=6)
    clean = run(s)
    k, v, _, _ = s["cache"]
    for j in (0, 5, 20, 39):
        sees = (s["mask"].cpu() >> j) & 1 == 1
        at = (int(s["bt"][0, (ctx + j) // 16]), (ctx + j) % 16)
        keep_k, keep_v = k[at].clone(), v[at].clone()
        k[at] = float("nan")
        out = run(s)
        assert torch.equal(out[~sees], clean[~sees]) and torch.isnan(out[sees]).all()
        k[at] = keep_k
        for bad in (float("nan"), float("inf"), -float("inf")):
            v[at][0, 3] = bad
            out = run(s)
            assert torch.equal(out[~sees], clean[~sees]), (j, bad)
            assert torch.equal(out[sees][:, :, 3].nan_to_num(7.0, 8.0, 9.0),
                               torch.full_like(out[sees][:, :, 3], bad).nan_to_num(7.0, 8.0, 9.0)), (j, bad)
            rest = [d for d in range(D) if d != 3]
            assert torch.equal(out[sees][:, :, rest], clean[sees][:, :, rest]), (j, bad)
            v[at] = keep_v


def test_special_scales_of_masked_drafts_do_not_reach_a_row():
    ctx, n = 500, 20
    s = make((ctx,), (n,), 4, 2, 128, 16, torch.bfloat16, True, seed=6)
    clean = run(s)
    for j in (0, 7, 19):
        sees = (s["mask"].cpu() >> j) & 1 == 1
        at = (int(s["bt"][0, (ctx + j) // 16]), (ctx + j) % 16)
        for scales in s["cache"][2:]:
            keep = scales[at].clone()
            scales[at] = float("nan")
            out = run(s)
            assert torch.equal(out[~sees], clean[~sees]) and torch.isnan(out[sees]).all()
            scales[at] = keep


def test_keys_past_the_length_are_not_read_into_a_row():
    """What lies behind a request's last key in its page, NaN as well, changes nothing."""
    s = make((37, 520), (3, 4), 4, 2, 128, 16, torch.bfloat16, False)
    clean = run(s)
    for b, length in ((0, 40), (1, 524)):
        for t in range(length, -(-length // 16) * 16):
            for c in s["cache"][:2]:
                c[int(s["bt"][b, t // 16]), t % 16] = float("nan")
    assert torch.equal(run(s), clean)


@pytest.mark.parametrize("int8", [True, False])
def test_requests_beyond_the_call_become_nan(int8):
    ctx, nodes = (600, 30, 700, 20), (2, 9, 2, 3)
    s = make(ctx, nodes, 4, 2, 64, 16, torch.float16, int8)
    good = run(s)
    out = run(s, max_nodes=8, longest=650)  # too many nodes in the second, too long the third
    assert torch.equal(out[:2], good[:2]) and torch.equal(out[13:], good[13:]) and torch.isnan(out[2:13]).all()
    t = dict(s, sl=s["sl"].clone())
    t["sl"][3] = 2  # shorter than its nodes
    out = run(t, longest=702)
    assert torch.equal(out[:13], good[:13]) and torch.isnan(out[13:]).all()
    t["sl"][3] = 100000  # past its block table
    out = run(t, longest=702)
    assert torch.equal(out[:13], good[:13]) and torch.isnan(out[13:]).all()
    for bad in (-1, s["cache"][0].shape[0]):
        t = dict(s, bt=s["bt"].clone())
        t["bt"][2, 40], t["bt"][1, 0] = bad, bad  # blocks that the cache does not have
        out = run(t)
        assert torch.equal(out[:2], good[:2]) and torch.equal(out[13:], good[13:]) and torch.isnan(out[2:13]).all()


def test_infinite_scores():
    s = make((70,), (1,), 1, 1, 64, 16, torch.bfloat16, False)
    s["q"].abs_().add_(0.1)
    k = s["cache"][0]
    at = (int(s["bt"][0, 1]), 4)
    drop = k[at].clone()
    k[at] = -float("inf")  # weighs nothing
    ref = dict(s, cache=(k.clone().index_put_(tuple(torch.tensor([i], device=DEV) for i in at), drop * 0 - 100), s["cache"][1], None, None))
    assert (run(s) - run(ref)).abs().max() <= 1e-5
    k[s["bt"][0].long()] = -float("inf")  # every score is -inf: the formula gives no number
    assert torch.isnan(run(s)).all()


def test_a_cache_past_32_bit_offsets():
    page, KV, D = 16, 2, 128
    blocks = (5 << 30) // (page * KV * 2 * D)
    pool = torch.empty(blocks, KV, page, 2 * D, dtype=torch.int8, device=DEV)
    scales = torch.empty(blocks, KV, page, 2, device=DEV)
    far = pool.transpose(1, 2).split(D, dim=-1) + scales.transpose(1, 2).unbind(-1)
    s = make((600, 40), (4, 2), 8, KV, D, page, torch.bfloat16, True)
    want = run(s)
    used = s["bt"].flatten().long()
    moved = blocks - 1 - torch.arange(used.numel(), device=DEV) * 977
    for a, b in zip(far, s["cache"]):
        a[moved] = b[used]
    assert torch.equal(run(dict(s, cache=far, bt=moved.view_as(s["bt"]).to(torch.int32))), want)


def test_graph_replays_and_the_statement():
    s = make((900, 70), (5, 12), 8, 2, 128, 16, torch.bfloat16, True)
    out = run(s)
    k, v, ks, vs = s["cache"]
    ref = tree_decode_torch(s["q"], k, v, s["bt"], s["sl"], s["qsl"], s["mask"], 128 ** -0.5, ks, vs)
    assert (out - ref).abs().max() <= 1e-4
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        tree_decode(s["q"], k, v, s["bt"], s["sl"], s["qsl"], s["mask"], 128 ** -0.5, out, 12, 905, key_scale=ks, value_scale=vs)
    for i in range(4):
        s["q"].copy_(torch.randn(s["q"].shape, generator=torch.Generator().manual_seed(i)))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(s)), i
