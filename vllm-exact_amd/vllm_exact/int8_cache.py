"""A paged KV cache in 8 bits: new tokens quantised as they are written, ranges read back (int8_cache.hip).

Each (token, KV head) row x of a key or value is held as whole numbers q = round(127 x / max|x|) in [-127, 127], ties to
even, and one fp32 scale max|x| / 127; it stands for q * scale. A row with an infinity or NaN reads back as NaN. At
D = 128 a cache takes 52 % of the 16-bit one's bytes.

The kernels take the cache as views (num_blocks, block_size, KV, D) and the scales as views (num_blocks, block_size,
KV), whatever the pool's layout; make_cache() lays a pool out with each head's page contiguous, K and V of a token
beside each other, as vLLM's FlashAttention cache has them. tree_attn.tree_decode attends to such a cache.
"""
import torch

from . import _native as _nx


def make_cache(num_blocks, block_size, num_kv_heads, head_dim, device):
    """(key_cache, value_cache, key_scale, value_scale), views of a zeroed pool [num_blocks, KV, block_size, 2 D] int8 and
    its scales [num_blocks, KV, block_size, 2] fp32."""
    pool = torch.zeros(num_blocks, num_kv_heads, block_size, 2 * head_dim, dtype=torch.int8, device=device)
    scales = torch.zeros(num_blocks, num_kv_heads, block_size, 2, dtype=torch.float32, device=device)
    return pool.transpose(1, 2).split(head_dim, dim=-1) + scales.transpose(1, 2).unbind(-1)


def write_cache(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping):
    """Quantise key and value (tokens, KV, D; fp32, bf16 or fp16) into the slots slot_mapping (tokens,) int64, a slot
    being block * block_size + place (vLLM's slot mapping). Slots outside the cache (-1: padding) are skipped; two tokens
    of one call never share a slot."""
    status = (_nx._calls or _nx.calls()).write_cache(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping)
    if status:
        _nx.check(status, "write_cache")


def read_cache(key_cache, value_cache, key_scale, value_scale, block_table, cu_seqlens, key, value, first=None):
    """Read ranges of sequences back into key and value (tokens, KV, D; fp32, bf16 or fp16), which are written and returned:
    packed rows [cu_seqlens[i], cu_seqlens[i + 1]) are the tokens first[i], first[i] + 1, ... of sequence i (first None:
    from its start), whose blocks are block_table[i]. A row past the block table or on a block outside the cache is NaN;
    rows of no sequence are left alone. cu_seqlens (n + 1,) and first (n,) are int32 on the GPU."""
    status = (_nx._calls or _nx.calls()).read_cache(key_cache, value_cache, key_scale, value_scale, block_table, cu_seqlens, key,
                                                    value, first)
    if status:
        _nx.check(status, "read_cache")
    return key, value


def quantize_torch(x):
    """torch statement of the quantisation of rows along the last axis: (int8 q, fp32 scale without that axis)."""
    x = x.float()
    top = x.abs().amax(dim=-1)
    special = ~torch.isfinite(top)
    down = torch.where(top > 2.0 ** 100, 2.0 ** -32, 1.0)
    div = torch.where((top > 0) & ~special, top * down, 1.0)
    q = torch.round(x * down[..., None] * 127 / div[..., None])
    scale = top / top.new_full((), 127.0)  # by a number, torch multiplies with its reciprocal on the GPU
    return torch.where(special[..., None], 0, q).to(torch.int8), torch.where(special, torch.nan, scale)


def dequantize_torch(q, scale):
    """torch statement of what such rows stand for, in fp32."""
    return q.float() * scale[..., None]
