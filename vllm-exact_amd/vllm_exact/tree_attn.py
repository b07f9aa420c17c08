"""Attention of drafted tokens over a paged cache with a fixed reduction order on MI355X.

Kernel (libvllm_exact_amd.so, tree_decode.hip): each request drafts a tree of up to 64 tokens, whose keys and values are
already in the cache behind its context; every node attends to the context and to those drafted tokens that its mask
names. One node is plain decoding. The cache holds the query's 16-bit type, or 8 bits with scales (int8_cache). How a
request's keys are cut and in which order they are summed is fixed by its own length and number of nodes, and a node's bits do
not depend on the other nodes' queries. Finite values give finite rows; an infinity or NaN among the values that a node attends
to is what it gets in that dim.
"""
import torch

from . import _native as _nx
from . import paged_attn

MAX_NODES = 64  # bits of a mask: the most nodes of a request


def tree_decode(query, key_cache, value_cache, block_table, seq_lens, query_start_loc, tree_mask, scale, out, max_nodes,
                max_seq_len, key_scale=None, value_scale=None):
    """query (tokens, H, D) bf16 or fp16, the nodes of all requests packed; key/value_cache (num_blocks, block_size, KV, D)
    views of the query's type, or int8 with key_scale and value_scale (num_blocks, block_size, KV) fp32; block_table (n,
    max_blocks) int32; seq_lens (n,) int32, the cached keys of a request with its nodes' own; query_start_loc (n + 1,) int32;
    tree_mask (tokens,) int64, bit j set where the node attends to the request's drafted token j (its own bit included), or
    None: to the drafted tokens up to its own; out (tokens, H, D) fp32, bf16 or fp16. A node that attends to nothing
    gives zeros. max_nodes (at most 64) and max_seq_len (0 or None: paged_attn.MAX_LEN) bound the nodes and seq_lens of every
    request: one beyond them, or shorter than its nodes, or with a block outside the cache, gets NaN rows; max_nodes 0 does
    nothing. Returns out."""
    status = (_nx._calls or _nx.calls()).tree_decode(
        query, key_cache, value_cache, block_table, seq_lens, query_start_loc, tree_mask, scale, out, max_nodes,
        max_seq_len or paged_attn.MAX_LEN, key_scale, value_scale)
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
