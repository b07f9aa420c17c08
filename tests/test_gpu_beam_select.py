"""GPU checks of beam search's selection against its torch statement in fp64 on the CPU: parents and tokens are equal."""
import pytest
import torch

from vllm_exact.beam import beam_select, beam_select_torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def select(logits, scores, beams, count):
    n = len(logits) // beams
    outs = torch.empty(n, count, device=DEV), torch.empty(n, count, device=DEV, dtype=torch.int32), torch.empty(n, count, device=DEV, dtype=torch.int64)
    got = beam_select(logits, scores, beams, *outs)
    assert all(a is b for a, b in zip(got, outs))
    return got


def check(logits, scores, beams, count):
    got = select(logits, scores, beams, count)
    want = beam_select_torch(logits.cpu(), scores.cpu(), beams, count)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    a, b = got[0].cpu().double(), want[0].double()
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a == -torch.inf, b == -torch.inf)
    fine = torch.isfinite(b)
    # both round to fp32 (2^-24 of the value each); the log-sums are off by a few 2^-25
    assert ((a - b).abs()[fine] <= 2 * 2.0 ** -24 * b.abs()[fine] + 2.0 ** -23).all()
    return got


def inputs(n, beams, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(n * beams, V, generator=g) * 2.5).to(dtype)
    return logits.to(DEV), (torch.rand(n * beams, generator=g) * -4 - 20).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,beams,V,count", [(1, 1, 1, 1), (3, 2, 5, 4), (2, 3, 255, 64), (1, 4, 8192, 4), (2, 8, 8193, 16), (5, 5, 50001, 11),
                                             (1, 64, 700, 64), (3, 1, 20000, 33), (1, 4, 151936, 4)])
def test_random_rows(n, beams, V, count, dtype):
    check(*inputs(n, beams, V, dtype), beams, count)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["equal", "two values", "steps", "rising", "falling", "zeros of both signs"])
def test_ties_and_orders(kind, dtype):
    V, beams = 20003, 3
    g = torch.Generator().manual_seed(1)
    rows = {"equal": torch.full((beams, V), 0.5), "two values": torch.randint(0, 2, (beams, V), generator=g).float(),
            "steps": torch.arange(V).div(3000, rounding_mode="floor").float().expand(beams, V), "rising": torch.arange(V).float().expand(beams, V) / 1000,
            "falling": -torch.arange(V).float().expand(beams, V) / 1000, "zeros of both signs": torch.where(torch.rand(beams, V, generator=g) < 0.5, 0.0, -0.0)}[kind]
    logits = rows.to(dtype).contiguous().to(DEV)
    for scores in ([-1.0, -1.0, -1.0], [-3.0, -1.0, -2.0]):
        check(logits, torch.tensor(scores, device=DEV), beams, 64)
        check(logits, torch.tensor(scores, device=DEV), beams, 5)


def test_equal_beams_tie_at_any_alignment():
    """The same row at even and odd elements: the same bits, so the first beam wins each tie."""
    V = 30011
    row = inputs(1, 1, V, torch.bfloat16, 2)[0][0]
    wide = torch.empty(4, V + 5, device=DEV, dtype=torch.bfloat16)
    logits = wide[:, 3:3 + V]
    logits.copy_(row.expand(4, V))
    best, parents, tokens = check(logits, torch.full((4,), -2.5, device=DEV), 4, 8)
    assert parents[0, :4].tolist() == [0, 1, 2, 3] and len(set(tokens[0, :4].tolist())) == 1  # further down, tokens of one row tie too


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_forbidden_tokens_and_ended_beams(dtype):
    n, beams, V = 6, 4, 9000
    logits, scores = inputs(n, beams, V, dtype, 3)
    logits[:, torch.rand(V, generator=torch.Generator().manual_seed(4)).to(DEV) < 0.9] = -torch.inf
    scores[1:4] = -torch.inf                 # the first request: one beam
    logits[4:8] = -torch.inf
    logits[5, 8191:8193] = 1.0               # the second: two tokens
    logits[8:12] = -torch.inf                # the third: none
    scores[12:16] = -torch.inf               # the fourth: no beam
    logits[16, 7], scores[16] = float("nan"), -torch.inf  # the fifth: an ended beam's logits count for nothing
    got = check(logits, scores, beams, 8)
    assert got[2][1, 2:].eq(-1).all() and got[1][2].eq(-1).all() and got[1][3].eq(-1).all() and torch.isfinite(got[0][4]).all()


@pytest.mark.parametrize("where", ["nan logit", "inf logit", "nan score", "inf score", "all nan"])
def test_nan_and_infinities_make_their_request_nan(where):
    logits, scores = inputs(3, 2, 9001, torch.float32, 5)
    if where == "nan logit":
        logits[2, 9000] = float("nan")
    elif where == "inf logit":
        logits[3, 0] = float("inf")
    elif where == "all nan":
        logits[3] = float("nan")
    else:
        scores[2] = float("nan") if where == "nan score" else float("inf")
    best, parents, tokens = check(logits, scores, 2, 4)
    assert torch.isnan(best[1]).all() and parents[1].eq(-1).all() and tokens[1].eq(-1).all()
    assert torch.isfinite(best[0]).all() and torch.isfinite(best[2]).all()


@pytest.mark.parametrize("score", [float("nan"), float("inf")])
def test_scores_count_where_a_beam_has_no_token(score):
    logits, scores = inputs(2, 2, 300, torch.float32, 7)
    logits[3], scores[3] = -torch.inf, score
    best, parents, tokens = check(logits, scores, 2, 4)
    assert torch.isnan(best[1]).all() and parents[1].eq(-1).all() and tokens[1].eq(-1).all() and torch.isfinite(best[0]).all()


@pytest.mark.parametrize("scale", [1e-3, 30.0, 1e4, 1e30])
def test_magnitudes(scale):
    logits, scores = inputs(2, 3, 10000, torch.float32, 6)
    got = select(logits * scale, scores, 3, 6)
    want = beam_select_torch((logits * scale).cpu(), scores.cpu(), 3, 6)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    fine = torch.isfinite(want[0])  # a score beyond fp32's range is -inf there
    assert torch.equal(torch.isfinite(got[0].cpu()), fine)
    assert ((got[0].cpu() - want[0]).abs()[fine] <= 2.0 ** -22 * (1 + want[0].abs()[fine])).all()


def test_bits_do_not_depend_on_the_batch_and_graphs_replay():
    logits, scores = inputs(5, 4, 30001, torch.bfloat16, 7)
    whole = select(logits, scores, 4, 8)
    for i in range(5):
        part = select(logits[4 * i:4 * i + 4], scores[4 * i:4 * i + 4], 4, 8)
        assert torch.equal(part[0], whole[0][i:i + 1]) and torch.equal(part[1] + 4 * i, whole[1][i:i + 1]) and torch.equal(part[2], whole[2][i:i + 1])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = [torch.empty_like(x) for x in whole]
    with torch.cuda.stream(side):
        beam_select(logits, scores, 4, *outs)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            beam_select(logits, scores, 4, *outs)
    for i in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, whole))
        select(logits[:4], scores[:4], 4, 8)


def test_refusals():
    logits, scores = inputs(2, 2, 100, torch.bfloat16)
    outs = lambda n=2, count=4: (torch.empty(n, count, device=DEV), torch.empty(n, count, device=DEV, dtype=torch.int32), torch.empty(n, count, device=DEV, dtype=torch.int64))
    for bad in (lambda: beam_select(logits, scores, 3, *outs()), lambda: beam_select(logits, scores, 0, *outs()),
                lambda: beam_select(logits, scores.double(), 2, *outs()), lambda: beam_select(logits, scores[:2], 2, *outs()),
                lambda: beam_select(logits, scores, 2, *outs(3)), lambda: beam_select(logits, scores, 2, *outs(2, 0)),
                lambda: beam_select(logits.double(), scores, 2, *outs()), lambda: beam_select(logits.t(), scores, 2, *outs()),
                lambda: beam_select(logits, scores, 2, *outs()[::-1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        beam_select(logits, scores, 2, *outs(2, 65))
    empty = logits[:0], scores[:0]
    assert beam_select(*empty, 2, *outs(0))[0].shape == (0, 4)


def test_rows_far_apart():
    """Rows past 2^31 elements from each other."""
    logits, scores = inputs(1, 4, 9001, torch.bfloat16, 8)
    stride = (1 << 30) + 1
    far = torch.empty(3 * stride + 9001, device=DEV, dtype=torch.bfloat16).as_strided(logits.shape, (stride, 1)).copy_(logits)
    a, b = select(far, scores, 4, 8), select(logits, scores, 4, 8)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_scores_updated_in_place():
    """As many continuations as beams: the next step's scores may be written over this one's."""
    logits, scores = inputs(5, 4, 1000, torch.float16, 9)
    want = select(logits, scores, 4, 4)
    parents, tokens = torch.empty(5, 4, device=DEV, dtype=torch.int32), torch.empty(5, 4, device=DEV, dtype=torch.int64)
    beam_select(logits, scores, 4, scores.view(5, 4), parents, tokens)
    assert torch.equal(scores.view(5, 4), want[0]) and torch.equal(parents, want[1]) and torch.equal(tokens, want[2])
