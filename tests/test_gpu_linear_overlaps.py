"""GPU checks of linear attention's outputs and states beside and over other arguments in one buffer."""
import pytest
import torch

from vllm_exact.linear_attn import linear_prompt, linear_step

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, KV, D, T = 4, 2, 64, 21


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def run(step, q, k, v, out, state=None, read=None, write=None):
    g = torch.full((H,), -0.1, device=DEV)
    if step:
        state = torch.zeros(1, H, D, D, device=DEV) if state is None else state
        return linear_step(q, k, v, g, 0.125, out, state, read, write)
    return linear_prompt(q, k, v, ints([0, T]), g, 0.125, out, state, read, write)


@pytest.mark.parametrize("step", [False, True])
def test_out_over_rows_of_a_projection(step):
    """Rows of (q, k, v, room): the room beside them takes the outputs; a head further, or a row of another buffer over them, is refused."""
    x = torch.randn(T, 2 * H + 2 * KV, D, device=DEV).bfloat16()
    q, k, v, room = x.split((H, KV, KV, H), dim=1)
    want = run(step, q, k, v, torch.empty(T, H, D, device=DEV, dtype=torch.bfloat16))
    before = x.clone()
    flat = x.view(-1)
    bad = [x[:, 1:1 + H], x[:, H:2 * H], x[:, H + 1:2 * H + 1], x[:, H + 2 * KV - 1:2 * H + 2 * KV - 1],
           flat[D * 3:].as_strided((T, H, D), x.stride()), flat[:T * H * D].view(T, H, D), flat[-T * H * D:].view(T, H, D),
           x[:, :H, 1:].as_strided((T, H, D), x.stride())]
    for out in bad:
        with pytest.raises(ValueError, match="out must not be"):
            run(step, q, k, v, out)
    assert torch.equal(x, before)
    assert torch.equal(run(step, q, k, v, room), want) and torch.equal(x[:, :H + 2 * KV], before[:, :H + 2 * KV])


@pytest.mark.parametrize("step", [False, True])
def test_states_over_each_other_and_the_rows(step):
    q, k, v = (torch.randn(T, h, D, device=DEV).bfloat16() for h in (H, KV, KV))
    out, slots = torch.empty(T, H, D, device=DEV), ints(range(T) if step else [1])
    pool = torch.zeros(T + 1, H, D, D, device=DEV)
    over = [torch.zeros(1, H, D, D, device=DEV).expand(T + 1, H, D, D), torch.zeros(T + 1, 1, D, D, device=DEV).expand(T + 1, H, D, D),
            pool.view(-1).as_strided((T, H, D, D), (4 * D, D * D, D, 1)), pool.view(-1).as_strided((T, H, D, D), (D * D, D * D, D, 1))]
    for state in over:
        with pytest.raises(ValueError, match="states must not overlap"):
            run(step, q, k, v, out, state, None, slots)
    # heads outside of slots, and states that are only read, may lie as they like
    wide = torch.zeros(H, T + 1, D, D, device=DEV).transpose(0, 1)
    a, b = run(step, q, k, v, torch.empty_like(out), wide, None, slots), run(step, q, k, v, torch.empty_like(out), pool, None, slots)
    assert torch.equal(a, b) and torch.equal(wide, pool)
    run(step, q, k, v, out, over[0], slots, None)
    with pytest.raises(ValueError, match="out must not be"):
        run(step, q, k, v, pool.view(-1)[5:5 + T * H * D].view(T, H, D), pool, slots, None)
    rows = torch.zeros(1, H, D, D, device=DEV)
    with pytest.raises(ValueError, match="state must not be"):
        run(step, q, rows.view(torch.bfloat16).view(-1)[:T * KV * D].view(T, KV, D), v, out, rows, None, ints([0] * (T if step else 1)))
