"""Attention in float64, one sequence and head at a time, with what fp32 kernels may be off, for the tests."""
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attend64(q, k, v, seen, scale, p_step, p_least):
    """(out, bound) of queries (rows, D) over keys and values (keys, D), seen (rows, keys). The bound adds up, relative to
    sum_j w_j |v_j|: the rounding of P (p_step), twice what the fp32 score is off (its dot product of D terms, its scaling),
    the hardware exponential and the fp32 sums over the keys, and p_least for each P below the type's normal range."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    seen = seen.cpu()
    k0, v0 = torch.where(seen.any(0)[:, None], k, 0), torch.where(seen.any(0)[:, None], v, 0)
    s = torch.where(seen, (q @ k0.T) * scale, -torch.inf)
    none = ~seen.any(1)
    w = torch.where(seen, torch.exp(s - torch.where(none, 0, s.amax(1))[:, None]), 0.0)
    w = torch.where(none[:, None], 0.0, w / w.sum(1, keepdim=True))
    size = torch.where(seen, (q.abs() @ k0.abs().T) * scale, 0).amax(1, keepdim=True)
    n, d = k.shape
    off = p_step + 2 * (d + 4) * 2.0 ** -24 * size + (n + 16) * 2.0 ** -23
    return w @ v0, off * (w @ v0.abs()) + n * p_least * v0.abs().amax()


def check(got, want, bound, what=""):
    """got within the bound and one rounding to its own type of the 64-bit result."""
    step = HALF_STEP[got.dtype]
    err = (got.double().cpu() - want).abs()
    limit = bound + step * (want.abs() + bound) + 1e-30
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert (err <= limit).all(), f"{what}: {float((err / limit).max()):.3g} times the bound"
