"""GPU checks of causal attention over packed prompts against float64.

Tolerance: P is rounded to the element type (half a step relative to each weight), scores and sums are fp32
(attention64.attend64 adds up the terms), and the output is rounded once."""
import pytest
import torch

from attention64 import HALF_STEP, attend64, check
from vllm_exact.prompt_attn import prompt_attention, prompt_attention_torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
LEAST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def make(lens, H, KV, D, dtype, seed=0, fused=False, tail=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + tail
    if fused:
        q, k, v = torch.randn(T, H + 2 * KV, D, generator=g).to(dtype).to(DEV).split((H, KV, KV), dim=1)
    else:
        q, k, v = (torch.randn(T, n, D, generator=g).to(dtype).to(DEV) for n in (H, KV, KV))
    cu = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)
    return q, k, v, cu


def run(q, k, v, cu, out_dtype=torch.float32, scale=None):
    out = torch.full(q.shape, float("nan"), device=DEV, dtype=out_dtype)
    assert prompt_attention(q, k, v, cu, q.shape[2] ** -0.5 if scale is None else scale, out) is out
    return out


def compare(out, q, k, v, cu, scale=None, heads=None):
    H, KV, D = q.shape[1], k.shape[1], q.shape[2]
    starts = cu.tolist()
    for i, (lo, hi) in enumerate(zip(starts, starts[1:])):
        seen = torch.ones(hi - lo, hi - lo, dtype=torch.bool).tril()
        for h in range(H) if heads is None else heads:
            if hi > lo:
                want, bound = attend64(q[lo:hi, h], k[lo:hi, h // (H // KV)], v[lo:hi, h // (H // KV)], seen,
                                       D ** -0.5 if scale is None else scale, HALF_STEP[q.dtype], LEAST[q.dtype])
                check(out[lo:hi, h], want, bound, f"sequence {i} head {h}")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,H,KV", [((1,), 8, 8), ((0, 1, 0), 4, 1), ((17, 0, 63, 64, 65, 1), 6, 2),
                                       ((127, 128, 129), 4, 4), ((300, 2, 257), 8, 2), ((31, 32, 33, 96, 191, 193), 3, 1)])
def test_against_float64(D, dtype, lens, H, KV):
    q, k, v, cu = make(lens, H, KV, D, dtype, seed=D + len(lens))
    compare(run(q, k, v, cu), q, k, v, cu)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_views_of_a_fused_projection_and_output_types(out_dtype):
    q, k, v, cu = make((70, 200, 9), 8, 2, 128, torch.bfloat16, fused=True)
    out = run(q, k, v, cu, out_dtype)
    compare(out, q, k, v, cu)
    wide = torch.full((q.shape[0], 9, 160), float("nan"), device=DEV, dtype=out_dtype)
    prompt_attention(q, k, v, cu, 128 ** -0.5, wide[:, 1:, 16:144])
    assert torch.equal(wide[:, 1:, 16:144], out)
    assert torch.isnan(wide[:, 0]).all() and torch.isnan(wide[:, 1:, :16]).all() and torch.isnan(wide[:, 1:, 144:]).all()


def test_long_sequences_and_large_scores():
    q, k, v, cu = make((1500, 700), 4, 2, 128, torch.bfloat16, seed=5)
    compare(run(q * 8, k, v, cu), q * 8, k, v, cu)
    statement = prompt_attention_torch(q, k, v, cu, 128 ** -0.5)
    assert (run(q, k, v, cu) - statement).abs().max() < 0.02
    for scale in (0.0, -0.1, 0.3):
        assert (run(q, k, v, cu, scale=scale) - prompt_attention_torch(q, k, v, cu, scale)).abs().max() < 0.02


def test_rows_outside_the_sequences_are_left_alone():
    q, k, v, cu = make((40, 100), 4, 1, 64, torch.float16, tail=30)
    out = run(q, k, v, cu)
    assert torch.isnan(out[140:]).all() and torch.isfinite(out[:140]).all()
    compare(out, q, k, v, cu)
    later = cu + 20  # a first sequence that does not start at row 0
    out = run(q, k, v, later)
    assert torch.isnan(out[:20]).all() and torch.isnan(out[160:]).all()
    compare(out, q, k, v, later)


def test_many_sequences_and_the_same_bits_alone():
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 150, (150,), generator=g).tolist()
    q, k, v, cu = make(lens, 4, 2, 128, torch.bfloat16, seed=9)
    out = run(q, k, v, cu)
    compare(out, q, k, v, cu, heads=(0, 3))
    starts = cu.tolist()
    for i in (0, 1, 63, 64, 65, 149):
        lo, hi = starts[i], starts[i + 1]
        alone = run(q[lo:hi], k[lo:hi], v[lo:hi], torch.tensor([0, hi - lo], dtype=torch.int32, device=DEV))
        assert torch.equal(alone, out[lo:hi]), i


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinities_and_nan_of_later_keys_do_not_reach_a_row(D, dtype):
    """Rows before a special key keep their bits; rows from it on get what the formula gives."""
    q, k, v, cu = make((150,), 2, 1, D, dtype, seed=1)
    clean = run(q, k, v, cu)
    for at in (1, 40, 63, 64, 100, 149):
        kk = k.clone()
        kk[at] = float("nan")
        out = run(q, kk, v, cu)
        assert torch.equal(out[:at], clean[:at]) and torch.isnan(out[at:]).all(), at
        for bad in (float("nan"), float("inf"), -float("inf")):
            vv = v.clone()
            vv[at, 0, 3] = bad
            out = run(q, k, vv, cu)
            assert torch.equal(out[:at], clean[:at]), (at, bad)
            want = torch.full_like(out[at:, :, 3], bad)
            assert torch.equal(out[at:, :, 3].nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0)), (at, bad)
            rest = [d for d in range(D) if d != 3]
            assert torch.equal(out[at:, :, rest], clean[at:, :, rest]), (at, bad)


def test_keys_that_score_minus_infinity():
    q, k, v, cu = make((90,), 1, 1, 64, torch.bfloat16)
    q, k = q.abs() + 0.1, k.clone()
    k[20] = -float("inf")  # scores -inf for every row
    out = run(q, k, v, cu)
    keep = [j for j in range(90) if j != 20]
    want, bound = attend64(q[keep, 0], k[keep, 0], v[keep, 0], torch.ones(89, 89, dtype=torch.bool).tril(), 64 ** -0.5,
                           HALF_STEP[torch.bfloat16], 0.0)
    check(out[keep, 0], want, bound)
    k[0] = -float("inf")  # row 0 has no other key: the formula gives no number
    assert torch.isnan(run(q, k, v, cu)[0]).all()


def test_far_strides():
    """Rows further apart than 32-bit byte offsets reach."""
    T, stride = 300, 1 << 23
    big = torch.empty(T * stride, device=DEV, dtype=torch.bfloat16)
    view = lambda at, n: big.as_strided((T, n, 64), (stride, 64, 1), at)
    q, k, v, cu = make((T,), 2, 1, 64, torch.bfloat16, seed=2)
    far = [view(0, 2).copy_(q), view(1 << 20, 1).copy_(k), view(1 << 21, 1).copy_(v)]
    out = view(1 << 22, 2)
    prompt_attention(*far, cu, 0.125, out)
    assert torch.equal(out, run(q, k, v, cu, torch.bfloat16))


def test_graph_replays_and_another_stream():
    q, k, v, cu = make((200, 31), 4, 2, 128, torch.bfloat16)
    want = run(q, k, v, cu)
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prompt_attention(q, k, v, cu, 128 ** -0.5, out)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prompt_attention(q, k, v, cu, 128 ** -0.5, out)
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(q, k, v, cu)), i
