"""GPU checks of linear attention's infinities and NaN: infinite with the recurrence's sign, or NaN, where its torch statement is; the bits
of a call without them elsewhere."""
import pytest
import torch

from vllm_exact.linear_attn import linear_attention_torch, linear_prompt, linear_step

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def same_kind(got, want):
    """NaN where the statement has NaN, its infinities where it has infinities."""
    got, want = got.float().cpu(), want.float().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got == INF, want == INF) and torch.equal(got == -INF, want == -INF)
    return torch.isfinite(want)


def rows_of(T, H, KV, D, dtype, signs, seed):
    x = torch.randn(T, H + 2 * KV, D, generator=torch.Generator().manual_seed(seed))
    x = torch.where(x == 0, 1.0, x)
    if signs == "positive":  # of queries and keys: the terms of one value have one sign
        x[:, :H + KV] = x[:, :H + KV].abs() + 2.0 ** -10
    return [y.contiguous() for y in x.to(dtype).split((H, KV, KV), dim=1)]


DECAYS = torch.tensor([-0.01, 0.0, -100.0, -200.0, -INF])  # exp: ordinary, one, below the normal numbers, 0 in fp32, 0


@pytest.mark.parametrize("dtype,out_dtype,D", [(torch.bfloat16, torch.bfloat16, 64), (torch.bfloat16, torch.float32, 128), (torch.float16, torch.float16, 128),
                                               (torch.float16, torch.float32, 64), (torch.bfloat16, torch.bfloat16, 256), (torch.float16, torch.float16, 256)])
@pytest.mark.parametrize("what", ["q", "k", "v", "state"])
@pytest.mark.parametrize("signs", ["random", "positive"])
def test_prompts(what, signs, dtype, out_dtype, D):
    lens, H, KV = (700, 90, 33, 1), 5, 1
    rows = dict(zip("qkv", rows_of(sum(lens), H, KV, D, dtype, signs, 1)))
    cu, slots = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32), torch.arange(4, dtype=torch.int32)
    pool = torch.randn(4, H, D, D, generator=torch.Generator().manual_seed(2))
    pool = pool.abs() + 0.1 if signs == "positive" else pool

    def run():
        state, out = pool.to(DEV), torch.full((sum(lens), H, D), 7.0, device=DEV, dtype=out_dtype)
        linear_prompt(*(rows[x].to(DEV) for x in "qkv"), cu.to(DEV), DECAYS.to(DEV), 0.125, out, state, slots.to(DEV), slots.to(DEV))
        return out, state

    before = run()
    for i, value in enumerate((INF, -INF, NAN)):
        # in the first part of the first sequence and in its third one; in the others: one of each
        where = (40, 690) if i == 0 else (700 + 64,) if i == 1 else (790 + 32,)
        if what == "state":
            pool[(0, 1, 2)[i], :, 3, D // 2 + i] = value
        else:
            for row in where:
                rows[what][row, 0, 5 + i] = value
    after = run()
    state = pool.clone()
    want = linear_attention_torch(*(rows[x] for x in "qkv"), cu, DECAYS, 0.125, state, slots, slots)
    fine = same_kind(after[0], want).to(DEV)
    assert not fine.all() and fine[-1].all()
    assert torch.equal(after[0][fine], before[0][fine])
    fine = same_kind(after[1], state).to(DEV)
    assert torch.equal(after[1][fine], before[1][fine])


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 256)])
@pytest.mark.parametrize("signs", ["random", "positive"])
def test_steps(signs, dtype, D):
    n, H, KV = 6, 5, 1
    q, k, v = rows_of(n, H, KV, D, dtype, signs, 3)
    pool = torch.randn(n, H, D, D, generator=torch.Generator().manual_seed(4))
    pool = pool.abs() + 0.1 if signs == "positive" else pool
    pool[0, :, 1, 2], pool[1, :, 1, 2], pool[2, :, 1, 2] = INF, -INF, NAN
    q[3, 2, 7], k[4, 0, 7], v[5, 0, 7] = INF, -INF, INF
    cu, slots = torch.arange(n + 1), torch.arange(n, dtype=torch.int32)
    state, got = pool.clone(), pool.to(DEV)
    for _ in range(3):
        want = linear_attention_torch(q, k, v, cu, DECAYS, 0.125, state, slots, slots)
        out = torch.empty(n, H, D, device=DEV)
        linear_step(q.to(DEV), k.to(DEV), v.to(DEV), DECAYS.to(DEV), 0.125, out, got, slots.to(DEV), slots.to(DEV))
        same_kind(out, want)
        same_kind(got, state)


def test_infinities_through_many_parts():
    """An infinite value of the first row of a long sequence, of which 18 parts are made: a head's decay over a part is 0, over a row it is not."""
    T, H, D = 5700, 3, 64
    q, k, v = rows_of(T, H, 1, D, torch.bfloat16, "positive", 5)
    g = torch.tensor([-0.5, -90.0, 0.0])
    v[0, 0, 3], v[0, 0, 9] = INF, -INF
    state = torch.zeros(1, H, D, D, device=DEV)
    out = torch.empty(T, H, D, device=DEV)
    linear_prompt(q.to(DEV), k.to(DEV), v.to(DEV), ints([0, T]), g.to(DEV), 1.0, out, state, None, ints([0]))
    assert (out[..., 3] == INF).all() and (out[..., 9] == -INF).all() and (state[..., 3] == INF).all() and (state[..., 9] == -INF).all()
    rest = [i for i in range(D) if i not in (3, 9)]
    assert torch.isfinite(out[..., rest]).all() and torch.isfinite(state[..., rest]).all()


def test_captured():
    lens, H, D = (400, 20), 2, 128
    q, k, v = (x.to(DEV) for x in rows_of(sum(lens), H, 1, D, torch.float16, "random", 6))
    v[300, 0, 4] = INF
    cu, slots, g = ints([0, 400, 420]), ints([0, 1]), torch.tensor([-0.1, -0.01], device=DEV)
    state, out = torch.zeros(2, H, D, D, device=DEV), torch.empty(420, H, D, device=DEV)
    linear_prompt(q, k, v, cu, g, 0.1, out, state, None, slots)
    side, other, there = torch.cuda.Stream(), torch.empty_like(out), torch.empty_like(state)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        linear_prompt(q, k, v, cu, g, 0.1, other, there, None, slots)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            linear_prompt(q, k, v, cu, g, 0.1, other, there, None, slots)
    for _ in range(3):
        other.zero_(), there.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(other.view(torch.int32), out.view(torch.int32)) and torch.equal(there.view(torch.int32), state.view(torch.int32))
        linear_prompt(q, k, v, cu, g, 0.1, torch.empty_like(out), torch.empty_like(state), None, slots)
