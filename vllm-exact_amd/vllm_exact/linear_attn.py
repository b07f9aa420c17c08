"""Linear attention with a decay for each head on MI355X: the recurrent layers beside a model's attention layers.

    S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,   out_t = scale q_t S_t

Kernels (libvllm_exact_amd.so, linear_attention.hip): whole prompts, packed one after the other, and one new token of every
sequence. A state S is a D x D fp32 matrix of each head. States live in the slots of a pool: a sequence starts from one
slot (or zeros) and leaves its state in one, the same or another, so beams that continue one parent read its slot and no
state is copied. A row's bits depend on its own sequence, never on the rest of the batch. An infinity or NaN of a row or of the state that
a sequence starts from makes this row and the later ones that meet it, and the state, infinite or NaN as the recurrence
has it (infinities of both signs in one sum are NaN), never earlier ones. Prompts with such values take 3 to 20 times as long.
"""
import torch

from . import _native as _nx


def linear_prompt(query, key, value, cu_seqlens, log_decay, scale, out, state=None, read_slots=None, write_slots=None):
    """query (tokens, H, D), key/value (tokens, KV, D) bf16 or fp16, rows [cu_seqlens[i], cu_seqlens[i + 1]) of sequence i;
    cu_seqlens (n + 1,) int32 on the GPU, ascending; log_decay (H,) fp32, <= 0; out (tokens, H, D) fp32, bf16 or fp16; rows and heads
    may be strided (rows by less than 2^23 elements, all by multiples of 8 but for out), D is 64, 128 or 256 and contiguous. out has no memory in
    common with the others, a state that is written none with them or another state. state (slots, H, D, D) fp32, each matrix [key dim][value dim]
    contiguous. Sequence i starts from slot read_slots[i] (n,) int32 (None or negative: from zeros), and its state after its last
    row goes to slot write_slots[i] (None or negative: nowhere; an empty sequence's is the state that it starts from). No
    sequence writes a slot that another reads or writes: where that is not so, or a slot is not in the pool, the sequence's
    rows are NaN and its state is not written. Rows after cu_seqlens[n] are left alone.

    States and sums are fp32. An fp32 row is off by their roundings (fp16: and 2^-24 of the sum of its terms' magnitudes); rows of 16 bits
    by their own rounding and at most 2^-17 (fp16: 3 2^-17) of that sum besides. Returns out."""
    status = (_nx._calls or _nx.calls()).linear_prompt(query, key, value, cu_seqlens, log_decay, scale, out, state, read_slots, write_slots)
    if status:
        _nx.check(status, "linear_prompt")
    return out


def linear_step(query, key, value, log_decay, scale, out, state, read_slots, write_slots):
    """One new token of every sequence: row i of query (n, H, D), key/value (n, KV, D) and out, from slot read_slots[i] to slot
    write_slots[i], as in linear_prompt. Several sequences may read one slot that none writes. Returns out."""
    status = (_nx._calls or _nx.calls()).linear_step(query, key, value, log_decay, scale, out, state, read_slots, write_slots)
    if status:
        _nx.check(status, "linear_step")
    return out


def linear_attention_torch(query, key, value, cu_seqlens, log_decay, scale, state=None, read_slots=None, write_slots=None):
    """torch statement of both, a token at a time in fp32: fp32 (tokens, H, D), zeros outside the sequences. The states are written.
    For linear_step, cu_seqlens is arange(n + 1)."""
    T, H, D = query.shape
    group = H // key.shape[1]
    out = torch.zeros(T, H, D, device=query.device)
    decay = log_decay.exp()[:, None, None]
    starts, ends = cu_seqlens.tolist(), {}
    for i, (lo, hi) in enumerate(zip(starts, starts[1:])):
        read = -1 if read_slots is None else int(read_slots[i])
        s = torch.zeros(H, D, D, device=query.device) if read < 0 else state[read].clone()
        for t in range(lo, hi):
            k, v = (x[t].float().repeat_interleave(group, dim=0) for x in (key, value))
            s = decay * s + k[:, :, None] * v[:, None, :]
            out[t] = (query[t].float()[:, :, None] * s).sum(dim=1) * scale
        if write_slots is not None and int(write_slots[i]) >= 0:
            ends[int(write_slots[i])] = s
    for slot, s in ends.items():
        state[slot] = s
    return out
