"""Causal attention over whole prompts with a fixed reduction order on MI355X.

Kernel (libvllm_exact_amd.so, prompt_attention.hip): sequences of different lengths, their rows packed one after the
other as vLLM passes them, grouped heads, bf16 or fp16, heads of 64, 128 or 256 dims. Scores, the softmax and all sums are fp32 and every score is
computed once, on the matrix cores. A row's bits depend on its query and on the keys and values up to its own, never on later
rows or the rest of the batch. Finite values give finite rows; an infinity or NaN among the values that a row attends to is
what it gets in that dim.
"""
import torch

from . import _native as _nx


def prompt_attention(query, key, value, cu_seqlens, scale, out):
    """query (tokens, H, D), key/value (tokens, KV, D) bf16 or fp16, heads of row t belonging to the sequence whose
    [cu_seqlens[i], cu_seqlens[i + 1]) holds t; cu_seqlens (n + 1,) int32 on the GPU (vLLM's query_start_loc); out
    (tokens, H, D) fp32, bf16 or fp16. Row j of a sequence attends to its rows 0..j. Rows and heads may be strided (views of
    a fused projection), D is 64, 128 or 256 and contiguous. Rows after cu_seqlens[n] are left alone. Returns out."""
    status = (_nx._calls or _nx.calls()).prompt_attention(query, key, value, cu_seqlens, scale, out)
    if status:
        _nx.check(status, "prompt_attention")
    return out


def prompt_attention_torch(query, key, value, cu_seqlens, scale):
    """fp32 torch statement of the same attention: fp32 (tokens, H, D), zeros outside the sequences."""
    T, H, D = query.shape
    KV = key.shape[1]
    out = torch.zeros(T, H, D, device=query.device, dtype=torch.float32)
    starts = cu_seqlens.tolist()
    for lo, hi in zip(starts, starts[1:]):
        n = hi - lo
        if n == 0:
            continue
        q = query[lo:hi].float().view(n, KV, H // KV, D).permute(1, 2, 0, 3).reshape(KV, -1, D)
        k = key[lo:hi].float().permute(1, 2, 0).contiguous()
        v = value[lo:hi].float().transpose(0, 1).contiguous()
        later = torch.ones(n, n, dtype=torch.bool, device=query.device).triu(1)
        s = (torch.bmm(q, k) * scale).view(KV, H // KV, n, n).masked_fill(later, -torch.inf).view(KV, -1, n)
        o = torch.bmm(torch.softmax(s, dim=-1), v)
        out[lo:hi] = o.view(KV, H // KV, n, D).permute(2, 0, 1, 3).reshape(n, H, D)
    return out
