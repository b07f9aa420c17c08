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


def check_views(what, key_cache, value_cache, key_scale, value_scale):
    """Raise unless the four tensors are the views of one 8-bit cache."""
    if key_cache.dtype != torch.int8 or value_cache.dtype != torch.int8:
        raise NotImplementedError(f"{what}: the cache must be int8")
    if key_scale.dtype != torch.float32 or value_scale.dtype != torch.float32:
        raise NotImplementedError(f"{what}: the scales must be fp32")
    if key_cache.dim() != 4 or value_cache.shape != key_cache.shape or key_scale.shape != key_cache.shape[:3] \
            or value_scale.shape != key_scale.shape:
        raise ValueError(f"{what}: cache views are (num_blocks, block_size, KV, D), scales (num_blocks, block_size, KV)")
    if key_cache.stride(3) != 1 or value_cache.stride(3) != 1:
        raise ValueError(f"{what}: the head dimension must be contiguous")


def _cache_args(key_cache, value_cache, key_scale, value_scale):
    st = _nx.strided
    return (*st(key_cache, 0, 1, 2), *st(value_cache, 0, 1, 2), *st(key_scale, 0, 1, 2), *st(value_scale, 0, 1, 2),
            key_cache.shape[0], key_cache.shape[1])


def _check_gpu(what, tensors, statement):
    if not all(t.is_cuda for t in tensors):
        raise ValueError(f"{what} runs the gfx950 HIP kernel and needs GPU tensors; use {statement} for the CPU statement")
    if any(t.device != tensors[0].device for t in tensors):
        raise ValueError(f"{what}: all tensors must be on one GPU")


def _check_rows(what, key, value, KV, D):
    if key.dim() != 3 or value.shape != key.shape or key.shape[1:] != (KV, D) or value.dtype != key.dtype:
        raise ValueError(f"{what}: key and value are (tokens, KV, D) of one type")
    if key.stride(2) != 1 or value.stride(2) != 1:
        raise ValueError(f"{what}: the head dimension must be contiguous")


def write_cache(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping):
    """Quantise key and value (tokens, KV, D; fp32, bf16 or fp16) into the slots slot_mapping (tokens,) int64, a slot
    being block * block_size + place (vLLM's slot mapping). Slots outside the cache (-1: padding) are skipped; two tokens
    of one call never share a slot."""
    _check_gpu("write_cache", (key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping), "quantize_torch")
    L = _nx.lib()
    check_views("write_cache", key_cache, value_cache, key_scale, value_scale)
    _check_rows("write_cache", key, value, *key_cache.shape[2:])
    if slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1 or not slot_mapping.is_contiguous() \
            or len(slot_mapping) != len(key):
        raise ValueError("write_cache: slot_mapping must be a contiguous int64 vector, one slot for each token")
    dtype = _nx.dtype_enum(key.dtype)
    if len(key) == 0:
        return
    st = _nx.strided
    status = _nx.launch(key.device, L.vxa_int8_cache_write, *st(key, 0, 1), *st(value, 0, 1), dtype, *key.shape,
                        *_cache_args(key_cache, value_cache, key_scale, value_scale), slot_mapping.data_ptr())
    if status:
        _nx.check(status, "write_cache")


def read_cache(key_cache, value_cache, key_scale, value_scale, block_table, cu_seqlens, key, value, first=None):
    """Read ranges of sequences back into key and value (tokens, KV, D; fp32, bf16 or fp16), which are written and returned:
    packed rows [cu_seqlens[i], cu_seqlens[i + 1]) are the tokens first[i], first[i] + 1, ... of sequence i (first None:
    from its start), whose blocks are block_table[i]. A row past the block table or on a block outside the cache is NaN;
    rows of no sequence are left alone. cu_seqlens (n + 1,) and first (n,) are int32 on the GPU."""
    tensors = (key_cache, value_cache, key_scale, value_scale, block_table, cu_seqlens, key, value)
    _check_gpu("read_cache", tensors if first is None else tensors + (first,), "dequantize_torch")
    L = _nx.lib()
    check_views("read_cache", key_cache, value_cache, key_scale, value_scale)
    _check_rows("read_cache", key, value, *key_cache.shape[2:])
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError("read_cache: block_table must be int32 with contiguous rows")
    n = len(block_table)
    if cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_contiguous() or cu_seqlens.shape != (n + 1,):
        raise ValueError("read_cache: cu_seqlens must be a contiguous int32 vector of the n + 1 starts")
    if first is not None and (first.dtype != torch.int32 or not first.is_contiguous() or first.shape != (n,)):
        raise ValueError("read_cache: first must be a contiguous int32 vector, one token for each sequence")
    dtype = _nx.dtype_enum(key.dtype)
    if len(key) == 0 or n == 0:
        return key, value
    st = _nx.strided
    status = _nx.launch(key.device, L.vxa_int8_cache_read, *_cache_args(key_cache, value_cache, key_scale, value_scale),
                        *st(block_table, 0), block_table.shape[1], cu_seqlens.data_ptr(), _nx.ptr(first), n, *key.shape,
                        *st(key, 0, 1), *st(value, 0, 1), dtype)
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
