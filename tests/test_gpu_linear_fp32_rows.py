"""GPU checks of linear attention's fp32 outputs: off by the roundings of fp32 sums alone, not by those of operands of fewer bits."""
import pytest
import torch

from linear64 import linear64
from vllm_exact.linear_attn import linear_prompt, linear_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,step", [((30,), False), ((1, 5), False), ((200, 64, 33), False), ((1,) * 7, True)])
@pytest.mark.parametrize("from_state", [False, True])
def test_rows_of_32_bits(lens, step, from_state, D, dtype):
    """The 2-norm of the error against that of the rows. An output is a sum of D terms with the state and of its chunk's rows; the state of
    a term for each row before. Were each addition rounded, by at most 2^-24 of a partial sum, with a deviation of 2^-24 / sqrt(3) of it,
    D + 2 rows of them in a walk leave sqrt((D + 2 rows) / 3) 2^-24 of sums that are no larger than the whole: 3 to 8 times 2^-24.
    Operands of 16 bits are off by up to 2^-17 of each term: 40 to 66 times 2^-24 of the rows."""
    H, n = 4, len(lens)
    g = torch.Generator().manual_seed(len(lens) + D)
    q, k, v = (torch.randn(sum(lens), h, D, generator=g).to(dtype).to(DEV) for h in (H, 2, 2))
    decay = (-(2.0 ** (-2.0 * (torch.arange(H) + 1)))).to(DEV)
    pool = 4 * torch.randn(n, H, D, D, generator=g).to(DEV)
    cu, slots = torch.tensor([0] + list(lens)).cumsum(0).to(DEV, torch.int32), torch.arange(n, dtype=torch.int32, device=DEV)
    want, ends = linear64(q, k, v, lens, decay, D ** -0.5, pool if from_state else None)
    read = slots if from_state else None
    out = torch.empty(sum(lens), H, D, device=DEV)
    if step:
        linear_step(q, k, v, decay, D ** -0.5, out, pool, read, slots)
    else:
        linear_prompt(q, k, v, cu, decay, D ** -0.5, out, pool, read, slots)
    room = ((D + 2 * max(lens)) / 3) ** 0.5 * 2.0 ** -24
    for got, exact in ((out, want), (pool, ends)):
        assert (got.double() - exact).norm() <= room * exact.norm(), float((got.double() - exact).norm() / exact.norm()) * 2 ** 24
    # 16-bit outputs are these, rounded once more: off by two halves of a step where the two forms round apart
    half = torch.empty_like(out, dtype=dtype)
    if step:
        return
    again = pool.clone()
    linear_prompt(q, k, v, cu, decay, D ** -0.5, half, again, None, None)
    plain = linear64(q, k, v, lens, decay, D ** -0.5)[0]
    assert (half.double() - plain).norm() <= torch.finfo(dtype).eps / 2 * plain.norm()
