"""Linear attention with a decay for each head in float64, a token at a time, with the sums of its terms' magnitudes, which the
tolerances of fp32 sums are stated in."""
import torch


def linear64(q, k, v, lens, log_decay, scale, starts=None):
    """Rows of all sequences in float64 (rows, H, D) and their end states (n, H, D, D); starts: (n, H, D, D) or None."""
    q, k, v, decay = q.double(), k.double(), v.double(), log_decay.double().exp()[:, None, None]
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, dim=1), v.repeat_interleave(group, dim=1)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    ends, row = [], 0
    for i, n in enumerate(lens):
        s = torch.zeros(q.shape[1], q.shape[2], q.shape[2], dtype=torch.float64, device=q.device) if starts is None else starts[i].double()
        for _ in range(n):
            s = decay * s + k[row, :, :, None] * v[row, :, None, :]
            out[row] = scale * torch.matmul(q[row][:, None, :], s)[:, 0]
            row += 1
        ends.append(s)
    return out, torch.stack(ends)


def bounds(q, k, v, lens, log_decay, scale, starts=None):
    """How far fp32 kernels may be off: (rows, states). Every sum is of fp32 terms, one rounding of 2^-24 of the magnitudes for
    each of the D dims and the rows before, and one for each decay (2^-24 of its exponent, which is at most the rows times |g| where
    the decay is not nothing).

    Operands of the matrix cores are two bf16 parts: the first is off by at most 2^-8 where the value is in [1, 2), so the second, below
    2^-8, by at most 2^-17. Every term of a row's sum meets one such operand, the state's or the score's: 2^-17. The other one of
    fp16 rows is two parts as well, exactly (11 bits), but the product of both second parts is left out: 2^-8 of 2^-8 more. A state's
    terms are exact parts; of fp16 keys the second part (2^-8) times the third of the value (below 2^-14) is left out, 2^-22."""
    out, ends = linear64(q.abs(), k.abs(), v.abs(), lens, log_decay, abs(scale), None if starts is None else starts.abs())
    n, d = max(lens) if lens else 0, q.shape[2]
    steps = (n + d + 64 + min(n * float(log_decay.abs().nan_to_num(posinf=0).max()), 90)) * 2.0 ** -24
    half = q.dtype == torch.float16
    return out * (2.0 ** -17 + half * 2.0 ** -16 + steps), ends * (half * 2.0 ** -22 + steps)
