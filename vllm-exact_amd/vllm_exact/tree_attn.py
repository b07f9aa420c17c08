"""Attention of drafted tokens over a paged cache with a fixed reduction order on MI355X.

Kernel (libvllm_exact_amd.so, tree_decode.hip): each request drafts a tree of up to 64 tokens, whose keys and values are
already in the cache behind its context; every node attends to the context and to those drafted tokens that its mask
names. One node is plain decoding. The cache holds the query's 16-bit type, or 8 bits with scales (int8_cache). Segments
of 512 keys and the order inside them are fixed, so a request's bits depend on its own length and nodes only.
"""
import torch

from . import _native as _nx
from . import int8_cache, paged_attn

MAX_NODES = 64  # bits of a mask


def tree_decode(query, key_cache, value_cache, block_table, seq_lens, query_start_loc, tree_mask, scale, out, max_nodes,
                max_seq_len, key_scale=None, value_scale=None):
    """query (tokens, H, D) bf16 or fp16, the nodes of all requests packed; key/value_cache (num_blocks, block_size, KV, D)
    views of the query's type, or int8 with key_scale and value_scale (num_blocks, block_size, KV) fp32; block_table (n,
    max_blocks) int32; seq_lens (n,) int32, the cached keys of a request with its nodes' own; query_start_loc (n + 1,) int32;
    tree_mask (tokens,) int64, bit j set where the node attends to the request's drafted token j (its own bit included), or
    None: to the drafted tokens up to its own; out (tokens, H, D) fp32, bf16 or fp16. A node that attends to nothing
    gives zeros. max_nodes (at most 64) and max_seq_len (0 or None: paged_attn.MAX_LEN) bound the nodes and seq_lens of every
    request: one beyond them, or shorter than its nodes, or with a block outside the cache, gets NaN rows. Returns out."""
    tensors = [query, key_cache, value_cache, block_table, seq_lens, query_start_loc, out]
    tensors += [t for t in (tree_mask, key_scale, value_scale) if t is not None]
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("tree_decode runs the gfx950 HIP kernel and needs GPU tensors; "
                             "use tree_decode_torch for the CPU statement")
    L = _nx.lib()
    if any(t.device != query.device for t in tensors):
        raise ValueError("tree_decode: all tensors must be on the query's GPU")
    if query.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError("tree_decode: query must be bf16 or fp16")
    if (key_scale is None) != (value_scale is None):
        raise ValueError("tree_decode: key_scale and value_scale come together")
    if key_scale is not None:
        int8_cache.check_views("tree_decode", key_cache, value_cache, key_scale, value_scale)
    elif key_cache.dtype != query.dtype or value_cache.dtype != query.dtype:
        raise NotImplementedError("tree_decode: the cache must have the query's type, or be int8 with scales")
    if query.dim() != 3 or key_cache.dim() != 4 or value_cache.shape != key_cache.shape or out.shape != query.shape:
        raise ValueError("tree_decode: inconsistent shapes")
    T, H, D = query.shape
    blocks, page, KV, _ = key_cache.shape
    if key_cache.shape[3] != D or KV == 0 or H % KV:
        raise ValueError("tree_decode: inconsistent shapes")
    if query.stride(2) != 1 or key_cache.stride(3) != 1 or value_cache.stride(3) != 1 or out.stride(2) != 1:
        raise ValueError("tree_decode: the head dimension must be contiguous")
    if block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32 or query_start_loc.dtype != torch.int32:
        raise ValueError("tree_decode: block_table, seq_lens and query_start_loc must be int32")
    n = len(seq_lens)
    if block_table.dim() != 2 or len(block_table) != n or query_start_loc.shape != (n + 1,) or seq_lens.dim() != 1:
        raise ValueError("tree_decode: one block-table row and length for each request, and n + 1 starts")
    if (block_table.shape[1] > 1 and block_table.stride(1) != 1) or not seq_lens.is_contiguous() \
            or not query_start_loc.is_contiguous():
        raise ValueError("tree_decode: block_table rows, seq_lens and query_start_loc must be contiguous")
    if tree_mask is not None and (tree_mask.dtype != torch.int64 or tree_mask.shape != (T,) or not tree_mask.is_contiguous()):
        raise ValueError("tree_decode: tree_mask must be a contiguous int64 vector, one mask for each node")
    max_nodes, max_seq_len = int(max_nodes), int(max_seq_len or paged_attn.MAX_LEN)
    if max_nodes < 0 or max_seq_len < 0:
        raise ValueError("tree_decode: max_nodes and max_seq_len must be >= 0")
    if max_nodes > MAX_NODES:
        raise NotImplementedError(f"tree_decode: at most {MAX_NODES} nodes a request, got {max_nodes}")
    if T == 0 or n == 0 or max_nodes == 0:
        return out
    ws_bytes = _nx.tree_workspace(T, H, D, max_seq_len)
    ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=query.device) if ws_bytes else None
    st = _nx.strided
    status = _nx.launch(query.device, L.vxa_tree_decode, *st(query, 0, 1), _nx.dtype_enum(query.dtype),
                        *st(key_cache, 0, 1, 2), *st(value_cache, 0, 1, 2), *st(key_scale, 0, 1, 2), *st(value_scale, 0, 1, 2),
                        blocks, page, *st(block_table, 0), block_table.shape[1], seq_lens.data_ptr(),
                        query_start_loc.data_ptr(), _nx.ptr(tree_mask), float(scale), out.data_ptr(),
                        _nx.dtype_enum(out.dtype), out.stride(0), out.stride(1), n, T, H, KV, D, max_nodes, max_seq_len,
                        _nx.ptr(ws), ws_bytes)
    if status:
        _nx.check(status, "tree_decode")
    return out


def tree_decode_torch(query, key_cache, value_cache, block_table, seq_lens, query_start_loc, tree_mask, scale, key_scale=None,
                      value_scale=None):
    """fp32 torch statement of the same attention: fp32 (tokens, H, D)."""
    T, H, D = query.shape
    page, KV = key_cache.shape[1:3]
    out = torch.zeros(T, H, D, device=query.device, dtype=torch.float32)
    starts = query_start_loc.tolist()
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        n, length = hi - lo, int(seq_lens[b])
        if n == 0:
            continue
        tok = torch.arange(length, device=query.device)
        at = block_table[b].long()[tok // page], tok % page
        keys, vals = key_cache[at].float(), value_cache[at].float()
        if key_scale is not None:
            keys, vals = keys * key_scale[at][..., None], vals * value_scale[at][..., None]
        node = torch.arange(n, device=query.device)
        seen = node[:, None] >= node if tree_mask is None else (tree_mask[lo:hi, None] >> node) & 1 == 1
        seen = torch.cat([torch.ones(n, length - n, dtype=torch.bool, device=query.device), seen], dim=1)
        q = query[lo:hi].float().view(n, KV, H // KV, D).permute(1, 0, 2, 3).reshape(KV, -1, D)
        s = torch.bmm(q, keys.permute(1, 2, 0).contiguous()) * scale
        s = s.masked_fill(~seen.repeat_interleave(H // KV, dim=0), -torch.inf)
        p = torch.where(seen.any(dim=1).repeat_interleave(H // KV)[:, None], torch.softmax(s, dim=-1), 0.0)
        o = torch.bmm(p, vals.transpose(0, 1).contiguous())
        out[lo:hi] = o.view(KV, n, H // KV, D).permute(1, 0, 2, 3).reshape(n, H, D)
    return out
