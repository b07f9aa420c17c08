"""GPU checks of the serving operators' variants: trees of many rows, which take the kernel that shares tiles through LDS, the
two ways to split long contexts, prompts in every grouping of heads and in large batches, quantisation next to ties, what the
calls refuse, and the example that runs the operators together. Tolerances as in the operators' own tests
(attention64.attend64 adds up the terms)."""
import importlib.util
from pathlib import Path

import pytest
import torch

import test_gpu_prompt_attention as prompts
import test_gpu_tree_decode as trees
from vllm_exact.int8_cache import make_cache, read_cache, write_cache
from vllm_exact.prompt_attn import prompt_attention
from vllm_exact.tree_attn import tree_decode

pytestmark = pytest.mark.gpu
DEV = "cuda"

# Rows (nodes times heads of a group) on both sides of 96; lengths on both sides of 512, 4096 and their multiples.
WIDE = [((480, 700), (61, 50), 16, 2), ((4090, 30), (25, 64), 8, 2), ((4072, 4072), (24, 25), 8, 2),
        ((100, 3000, 0, 2047), (3, 64, 30, 33), 4, 1), ((0, 448), (64, 64), 2, 1), ((6000,), (40,), 12, 4)]


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ctx,nodes,H,KV", WIDE)
def test_trees_of_many_rows(int8, dtype, D, ctx, nodes, H, KV):
    s = trees.make(ctx, nodes, H, KV, D, 16, dtype, int8, seed=D + sum(nodes))
    trees.compare(trees.run(s), s, heads=(0, H - 1))
    trees.compare(trees.run(s, mask=False), s, mask=False, heads=(H // 2,))


@pytest.mark.parametrize("int8", [True, False])
def test_bits_of_many_rows_do_not_depend_on_the_batch(int8):
    ctx, nodes = (4500, 3, 530, 2500), (30, 64, 25, 2)
    s = trees.make(ctx, nodes, 8, 2, 128, 16, torch.bfloat16, int8, seed=4)
    out = trees.run(s)
    assert torch.equal(trees.run(s, max_nodes=64, longest=9000), out)
    starts = s["qsl"].tolist()
    for b in range(4):
        lo, hi = starts[b], starts[b + 1]
        one = dict(q=s["q"][lo:hi], cache=s["cache"], bt=s["bt"][b:b + 1], sl=s["sl"][b:b + 1],
                   qsl=torch.tensor([0, hi - lo], dtype=torch.int32, device=DEV), mask=s["mask"][lo:hi].contiguous())
        assert torch.equal(trees.run(one), out[lo:hi]), b
    many = dict(s, q=s["q"].repeat(60, 1, 1), bt=s["bt"].repeat(60, 1), sl=s["sl"].repeat(60), mask=s["mask"].repeat(60),
                qsl=torch.tensor([0] + list(nodes) * 60).cumsum(0).to(torch.int32).to(DEV))
    assert torch.equal(trees.run(many), out.repeat(60, 1, 1))


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("length", [2048, 2049, 2560, 4095, 8200])
def test_one_strand_or_a_group_a_workgroup(int8, length):
    """A request alone is split over more workgroups than in a large batch: the same sums."""
    s = trees.make((length - 3,), (3,), 8, 2, 64, 16, torch.bfloat16, int8, seed=length)
    out = trees.run(s)
    trees.compare(out, s, heads=(0, 7))
    n = 400
    many = dict(s, q=s["q"].repeat(n, 1, 1), bt=s["bt"].repeat(n, 1), sl=s["sl"].repeat(n), mask=s["mask"].repeat(n),
                qsl=torch.arange(0, 3 * n + 1, 3, dtype=torch.int32, device=DEV))
    assert torch.equal(trees.run(many), out.repeat(n, 1, 1))


@pytest.mark.parametrize("n", [60, 130, 260, 300])
def test_large_batches_of_every_kind_of_request(n):
    """Requests of one to four segments past whole groups, empty ones, misfits and requests of many rows, in batches whose
    workgroups go by size (up to 256 requests) and beyond: each as it is alone."""
    kinds = [(2600, 1), (6000, 2), (0, 0), (5, 3), (2047, 1), (2048, 1), (4096, 64), (8191, 1), (3000, 30), (700, 4)]
    ctx, nodes = [k[0] for k in kinds], [k[1] for k in kinds]
    s = trees.make(ctx, nodes, 16, 4, 64, 16, torch.bfloat16, True, seed=11)
    longest = 8000  # the eighth is beyond it
    want = trees.run(s, longest=longest)
    starts = s["qsl"].tolist()
    assert torch.isnan(want[starts[7]:starts[8]]).all() and torch.isfinite(want[:starts[7]]).all()
    pick = torch.randint(0, len(kinds), (n,), generator=torch.Generator().manual_seed(n)).tolist()
    rows = torch.cat([torch.arange(starts[i], starts[i + 1]) for i in pick]).to(DEV)
    many = dict(s, q=s["q"][rows], bt=s["bt"][pick], sl=s["sl"][pick], mask=s["mask"][rows],
                qsl=torch.tensor([0] + [nodes[i] for i in pick]).cumsum(0).to(torch.int32).to(DEV))
    out = trees.run(many, longest=longest, max_nodes=64)
    assert torch.equal(out.nan_to_num(7.0), want[rows].nan_to_num(7.0)) and torch.equal(torch.isnan(out), torch.isnan(want[rows]))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_specials_of_masked_drafts_among_many_rows(D, dtype):
    ctx, n = 500, 64
    s = trees.make((ctx,), (n,), 2, 1, D, 16, dtype, False, seed=6)
    clean = trees.run(s)
    k, v, _, _ = s["cache"]
    for j in (0, 11, 12, 40, 63):
        sees = (s["mask"].cpu() >> j) & 1 == 1
        at = (int(s["bt"][0, (ctx + j) // 16]), (ctx + j) % 16)
        keep_k, keep_v = k[at].clone(), v[at].clone()
        k[at] = float("nan")
        out = trees.run(s)
        assert torch.equal(out[~sees], clean[~sees]) and torch.isnan(out[sees]).all()
        k[at] = keep_k
        for bad in (float("nan"), float("inf"), -float("inf")):
            v[at][0, 3] = bad
            out = trees.run(s)
            assert torch.equal(out[~sees], clean[~sees]), (j, bad)
            assert torch.equal(out[sees][:, :, 3].nan_to_num(7.0, 8.0, 9.0),
                               torch.full_like(out[sees][:, :, 3], bad).nan_to_num(7.0, 8.0, 9.0)), (j, bad)
            rest = [d for d in range(D) if d != 3]
            assert torch.equal(out[sees][:, :, rest], clean[sees][:, :, rest]), (j, bad)
            v[at] = keep_v


@pytest.mark.parametrize("int8", [True, False])
def test_empty_rows_and_bad_requests_among_many_rows(int8):
    s = trees.make((0, 700, 20, 600), (40, 64, 2, 50), 4, 1, 64, 16, torch.float16, int8)
    s["mask"][5], s["mask"][39] = 0, -1 << 50  # bits past the nodes name no key
    good = trees.run(s)
    assert (good[5] == 0).all() and (good[39] == 0).all() and torch.isfinite(good).all()
    trees.compare(good, s, heads=(0,))
    out = trees.run(s, max_nodes=60)  # too many nodes in the second
    assert torch.equal(out[:40], good[:40]) and torch.equal(out[104:], good[104:]) and torch.isnan(out[40:104]).all()
    for bad in (-1, s["cache"][0].shape[0]):
        t = dict(s, bt=s["bt"].clone())
        t["bt"][1, 33], t["bt"][3, 0] = bad, bad  # blocks that the cache does not have
        out = trees.run(t)
        assert torch.equal(out[:40], good[:40]) and torch.equal(out[104:106], good[104:106])
        assert torch.isnan(out[40:104]).all() and torch.isnan(out[106:]).all()


def test_trees_on_another_stream_beside_this_one():
    """The workspace belongs to the stream of the call."""
    s = trees.make((9000, 40), (4, 30), 8, 2, 128, 16, torch.bfloat16, True)
    want = trees.run(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = [trees.run(s) for _ in range(5)]
    b = [trees.run(s) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in a + b)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,KV", [(5, 5), (6, 3), (12, 3), (8, 1), (10, 5), (9, 3)])
def test_prompts_of_every_grouping(D, H, KV):
    q, k, v, cu = prompts.make((33, 260, 1, 95, 64), H, KV, D, torch.bfloat16, seed=H + D, fused=True)
    prompts.compare(prompts.run(q, k, v, cu), q, k, v, cu)


def test_hundreds_of_prompts():
    """More sequences than are looked through at a time, empty ones among them."""
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(0, 50, (700,), generator=g).tolist()
    lens[255:259] = [0, 200, 0, 130]
    q, k, v, cu = prompts.make(lens, 4, 1, 64, torch.float16, seed=3)
    out = prompts.run(q, k, v, cu)
    prompts.compare(out, q, k, v, cu, heads=(1,))
    starts = cu.tolist()
    for i in (256, 258, 512, 699):
        lo, hi = starts[i], starts[i + 1]
        if hi > lo:
            alone = prompts.run(q[lo:hi], k[lo:hi], v[lo:hi], torch.tensor([0, hi - lo], dtype=torch.int32, device=DEV))
            assert torch.equal(alone, out[lo:hi]), i


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_prompt_outputs_of_any_alignment(out_dtype):
    q, k, v, cu = prompts.make((100, 37), 4, 2, 64, torch.bfloat16)
    want = prompts.run(q, k, v, cu, out_dtype)
    for stride, shift in ((64, 1), (68, 4), (72, 0), (67, 3)):
        buf = torch.full((137 * 4 * stride + 80,), float("nan"), device=DEV, dtype=out_dtype)
        view = buf.as_strided((137, 4, 64), (4 * stride, stride, 1), shift)
        prompt_attention(q, k, v, cu, 64 ** -0.5, view)
        assert torch.equal(view, want), (stride, shift)
        assert torch.isnan(buf).sum() == buf.numel() - want.numel()


@pytest.mark.parametrize("H,KV", [(3, 3), (4, 1)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_specials_far_into_a_prompt(D, H, KV):
    q, k, v, cu = prompts.make((70, 500), H, KV, D, torch.bfloat16, seed=2)
    clean = prompts.run(q, k, v, cu)
    for at in (70 + 5, 70 + 255, 70 + 300, 70 + 499):
        vv = v.clone()
        vv[at, 0, 7], vv[at, 0, 9] = float("inf"), float("nan")
        out = prompts.run(q, k, vv, cu)
        heads = slice(0, H // KV)
        assert torch.equal(out[:at], clean[:at]) and torch.equal(out[:, H // KV:], clean[:, H // KV:]), at
        assert (out[at:, heads, 7] == float("inf")).all() and torch.isnan(out[at:, heads, 9]).all(), at
        rest = [d for d in range(D) if d not in (7, 9)]
        assert torch.equal(out[at:, heads][:, :, rest], clean[at:, heads][:, :, rest]), at


def whole_numbers(x):
    """round(127 x / max|x|), ties to even, in 64 bits."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(127 * x / torch.where(top > 0, top, 1.0))


def written(x):
    T, KV, D = x.shape
    k, v, ks, vs = make_cache(T, 1, KV, D, DEV)
    write_cache(x, -x, k, v, ks, vs, torch.arange(T, device=DEV))
    return k[:, 0], v[:, 0], ks[:, 0], vs[:, 0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_quantisation_at_and_beside_ties(dtype, D):
    g = torch.Generator().manual_seed(D)
    x = (torch.randn(20000, 2, D, generator=g) * torch.exp2(torch.randint(-12, 12, (20000, 2, 1), generator=g).float())).to(dtype)
    odd = torch.randint(-127, 127, (500, 2, D), generator=g) * 2 + 1  # halves of 254: every one a tie
    x[:500] = odd.to(dtype)
    x[:500, :, 0] = 254
    x[500:700] = x[500:700].clamp(-0.5, 0.5) / 64
    x[500:700, :, 1] = 508  # most round to zero, some lie at a half
    q, minus, scale, _ = written(x.to(DEV))
    want = whole_numbers(x)
    assert torch.equal(q.cpu().double(), want) and torch.equal(minus.cpu().double(), -want)
    top = x.double().abs().amax(-1)
    assert ((scale.cpu().double() - top / 127).abs() <= top / 127 * 2.0 ** -24).all()


@pytest.mark.parametrize("exponent", [-133, -126, -111, -110, -109, 99, 100, 101, 126])
def test_quantisation_of_tiny_and_huge_rows(exponent):
    g = torch.Generator().manual_seed(exponent + 200)
    x = (torch.randint(-255, 256, (300, 1, 64), generator=g).double() * 2.0 ** (exponent - 6)).to(torch.bfloat16)
    q, _, _, _ = written(x.to(DEV))
    assert torch.equal(q.cpu().double(), whole_numbers(x))


@pytest.mark.parametrize("KV,D", [(1, 64), (3, 64), (5, 128), (7, 256), (40, 64)])
@pytest.mark.parametrize("n", [1, 3, 2100])
def test_cache_sizes_of_every_split(KV, D, n):
    """Tokens that fill no workgroup or need several turns; fp32 rows read back are exactly q times the scale."""
    g = torch.Generator().manual_seed(KV * n)
    x = torch.randn(n, KV, D, generator=g).to(torch.bfloat16).to(DEV)
    page = 7
    cache = make_cache(n // page + 2, page, KV, D, DEV)
    bt = torch.randperm(n // page + 2, generator=g).to(torch.int32).to(DEV)[None]
    at = torch.arange(n, device=DEV)
    slots = bt[0, at // page].long() * page + at % page
    write_cache(x, -x, *cache, slots)
    k, v = torch.empty(n, KV, D, device=DEV), torch.empty(n, KV, D, device=DEV)
    read_cache(*cache, bt, torch.tensor([0, n], dtype=torch.int32, device=DEV), k, v)
    scale = cache[2][slots // page, slots % page]
    assert torch.equal(k, whole_numbers(x).float() * scale[..., None]) and torch.equal(v, -k)


def refused(kind, match, call, args, **change):
    with pytest.raises(kind, match=match):
        call(**{**args, **change})


def test_what_the_calls_refuse():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    args = dict(query=bf(6, 4, 64), key=bf(6, 2, 64), value=bf(6, 2, 64), cu_seqlens=ints(0, 6), scale=0.1, out=bf(6, 4, 64))
    no = lambda kind, match, **c: refused(kind, match, prompt_attention, args, **c)
    no(NotImplementedError, "all bf16 or all fp16", query=args["query"].float())
    no(NotImplementedError, "all bf16 or all fp16", key=args["key"].half())
    no(ValueError, "cu_seqlens", cu_seqlens=args["cu_seqlens"].long())
    no(ValueError, "cu_seqlens", cu_seqlens=ints())
    no(ValueError, "shapes", out=bf(6, 4, 32))
    no(ValueError, "shapes", key=bf(5, 2, 64))
    no(ValueError, "shapes", key=bf(6, 3, 64), value=bf(6, 3, 64))
    no(ValueError, "contiguous", out=bf(6, 64, 4).transpose(1, 2))
    no(ValueError, "floating dtype", out=args["out"].double())
    no(ValueError, "prompt_attention_torch", value=args["value"].cpu())
    no(TypeError, "tensor", out=None)
    no(TypeError, "number", scale="x")
    no(NotImplementedError, "prompt_attention", query=bf(6, 4, 48), key=bf(6, 2, 48), value=bf(6, 2, 48), out=bf(6, 4, 48))
    no(NotImplementedError, "prompt_attention", query=bf(6 * 4 * 64 + 1)[1:].view(6, 4, 64))

    cache = make_cache(4, 16, 2, 64, DEV)
    names = ("key_cache", "value_cache", "key_scale", "value_scale")
    args = dict(key=bf(6, 2, 64), value=bf(6, 2, 64), slot_mapping=torch.arange(6, device=DEV), **dict(zip(names, cache)))
    no = lambda kind, match, **c: refused(kind, match, write_cache, args, **c)
    no(NotImplementedError, "int8", key_cache=cache[0].float())
    no(NotImplementedError, "fp32", key_scale=cache[2].half())
    no(ValueError, "cache views", key_scale=cache[2][:, :8])
    no(ValueError, "tokens, KV, D", value=bf(6, 2, 64).half())
    no(ValueError, "tokens, KV, D", key=bf(6, 1, 64), value=bf(6, 1, 64))
    no(ValueError, "slot_mapping", slot_mapping=torch.arange(5, device=DEV))
    no(ValueError, "slot_mapping", slot_mapping=torch.arange(6, device=DEV).int())
    no(ValueError, "quantize_torch", slot_mapping=torch.arange(6))

    args = dict(block_table=ints(0, 1).view(1, 2), cu_seqlens=ints(0, 6), key=bf(6, 2, 64), value=bf(6, 2, 64), **dict(zip(names, cache)))
    no = lambda kind, match, **c: refused(kind, match, read_cache, args, **c)
    no(ValueError, "block_table", block_table=args["block_table"].long())
    no(ValueError, "block_table", block_table=ints(0, 1, 2, 3).view(2, 2).t()[:1])
    no(ValueError, "cu_seqlens", cu_seqlens=ints(0, 3, 6))
    no(ValueError, "first", first=ints(0, 0))
    no(ValueError, "tokens, KV, D", key=bf(6, 2, 128), value=bf(6, 2, 128))
    no(ValueError, "dequantize_torch", cu_seqlens=args["cu_seqlens"].cpu())

    args = dict(query=bf(3, 4, 64), block_table=ints(0, 1).view(1, 2), seq_lens=ints(9), query_start_loc=ints(0, 3),
                tree_mask=torch.ones(3, dtype=torch.int64, device=DEV), scale=0.1, out=bf(3, 4, 64), max_nodes=3, max_seq_len=20,
                **dict(zip(names, cache)))
    no = lambda kind, match, **c: refused(kind, match, tree_decode, args, **c)
    no(NotImplementedError, "bf16 or fp16", query=args["query"].float())
    no(ValueError, "come together", key_scale=None)
    no(NotImplementedError, "query's type", key_scale=None, value_scale=None)
    no(NotImplementedError, "fp32", value_scale=cache[3].double())
    no(ValueError, "shapes", out=bf(3, 2, 64))
    no(ValueError, "shapes", query=bf(3, 3, 64), out=bf(3, 3, 64))
    no(ValueError, "seq_lens", seq_lens=ints(9, 9))
    no(ValueError, "seq_lens", query_start_loc=ints(0))
    no(ValueError, "tree_mask", tree_mask=args["tree_mask"].int())
    no(ValueError, ">= 0", max_nodes=-1)
    no(NotImplementedError, "at most 64", max_nodes=65)
    no(TypeError, "integer", max_nodes="3")
    no(ValueError, "tree_decode_torch", tree_mask=args["tree_mask"].cpu())


def test_the_example():
    path = Path(__file__).resolve().parents[1] / "vllm-exact_amd" / "examples" / "draft_tree.py"
    spec = importlib.util.spec_from_file_location("draft_tree", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    g = torch.Generator().manual_seed(1)
    texts = [torch.randint(0, 64, (n,), generator=g).tolist() for n in (1, 40, 150, 17)]
    model = example.Model()
    plain, plain_steps = example.generate(model, texts, 40, 0)
    drafted, steps = example.generate(model, texts, 40, 15)
    assert plain == drafted and steps < plain_steps == 39
