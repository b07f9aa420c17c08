"""Pages of paged caches on MI355X: copied, shared by forked rows, given out and taken back, and drafted tokens kept.

Kernels (libvllm_exact_amd.so, pages.hip). A page (block) belongs to as many holders as ref_count (num_blocks,) int32 on the GPU
says; a page of count 0 is free. The rows of a block table hold the pages of their tokens; whoever else holds a page (a
prefix that is kept, say) adds to its count. Nothing waits for the host, and new pages are the lowest free ones in the
order of rows and places, so a program gives the same tables each time.

`caches` are all tensors whose pages the table names, of every layer: views (num_blocks, block_size, KV, D) or (num_blocks,
block_size, KV) of any type, as int8_cache.make_cache gives them.
"""
import torch

from . import _native as _nx


def copy_pages(caches, block_size, source, target):
    """Copy page source[i] to target[i] in every cache; source and target (n,) int32 on the GPU. Pairs with a page that the cache
    does not have (-1, say) are skipped; of pairs with one target the last counts; no page is a source and a target."""
    status = (_nx._calls or _nx.calls()).copy_pages(caches, block_size, source, target)
    if status:
        _nx.check(status, "copy_pages")


def fork_pages(caches, block_table, seq_lens, parents, ref_count, block_size, out_table, out_lens, out_ref_count=None):
    """The rows of out_table continue those of block_table: row r takes row parents[r]'s pages and length (a negative parent, or
    one that is no row: an empty row). Whole pages are shared. A page that the length ends in is copied, in every cache, to the
    lowest free page, but for the first row of a parent where nobody else holds that page. Pages of rows that none
    continues lose a holder. block_table (rows, max_blocks) and out_table (new rows, max_blocks) int32; entries
    behind a row's pages are -1. seq_lens (rows,), parents and out_lens (new rows,) int32. out_ref_count None: ref_count is
    updated. Outputs have no memory in common with each other or the inputs. Returns a (1,) int32 tensor: how many rows found no free page; theirs is -1, which the attention answers with
    NaN."""
    missing = ref_count.new_empty(1)
    status = (_nx._calls or _nx.calls()).fork_pages(caches, block_table, seq_lens, parents, ref_count, block_size, out_table, out_lens,
                                                    ref_count if out_ref_count is None else out_ref_count, missing)
    if status:
        _nx.check(status, "fork_pages")
    return missing


def resize_pages(block_table, seq_lens, new_lens, ref_count, block_size, out_table=None, out_ref_count=None):
    """Rows get the pages of new_lens tokens in place of seq_lens: the lowest free ones (free before the call) where they grow, in the order of
    rows and places; where they shrink, 0 for a row that has ended, the pages behind lose a holder and their entries
    are -1. A row has at most max_blocks pages. A grown row's last page is written to next: it should have no other holder, as
    fork_pages leaves it. out_table and out_ref_count None: block_table and ref_count are updated; others have no memory in common with
    each other or the inputs. Returns a (1,) int32 tensor: how
    many pages were missing; their entries are -1."""
    missing = ref_count.new_empty(1)
    status = (_nx._calls or _nx.calls()).resize_pages(block_table, seq_lens, new_lens, ref_count, block_size,
                                                      block_table if out_table is None else out_table,
                                                      ref_count if out_ref_count is None else out_ref_count, missing)
    if status:
        _nx.check(status, "resize_pages")
    return missing


def keep_drafted(caches, block_table, seq_lens, query_start_loc, keep, block_size, out_lens):
    """After tree_attn.tree_decode: of each request's drafted tokens, the last query_start_loc[i + 1] - query_start_loc[i] (at most
    64) of its seq_lens[i] cached ones, those with bit j of keep[i] set (an accepted node's tree_mask) move side by side behind the
    context, in every cache, bit for bit. keep (n,) int64; out_lens (n,) int32, apart from the inputs, takes the lengths with the kept
    tokens alone, for resize_pages and the next step. No other row holds the drafted tokens' pages, and no two caches the same memory (values that are a slice of
    the keys are moved with them). A request with more drafted
    tokens than 64 or than cached ones stays as it is. Returns out_lens."""
    status = (_nx._calls or _nx.calls()).keep_drafted(caches, block_table, seq_lens, query_start_loc, keep, block_size, out_lens)
    if status:
        _nx.check(status, "keep_drafted")
    return out_lens


def _pages(length, block_size, cols):
    return min(-(-max(length, 0) // block_size), cols)


def fork_pages_torch(caches, block_table, seq_lens, parents, ref_count, block_size):
    """Statement of fork_pages row by row; the caches are written: (out_table, out_lens, out_ref_count, missing)."""
    rows, cols = block_table.shape
    blocks, table, counts = len(ref_count), block_table.tolist(), ref_count.tolist()
    lens = [min(max(n, 0), cols * block_size) for n in seq_lens.tolist()]
    free = [b for b in range(blocks) if counts[b] == 0]
    new, new_lens, seen, missing, before = [], [], set(), 0, list(counts)
    for r in range(rows):
        for b in table[r][:_pages(lens[r], block_size, cols)]:
            if 0 <= b < blocks:
                counts[b] -= 1
    for parent in parents.tolist():
        n = lens[parent] if 0 <= parent < rows else 0
        row = table[parent][:_pages(n, block_size, cols)] if n else []
        if n % block_size and 0 <= row[-1] < blocks and (parent in seen or before[row[-1]] != 1):
            page = free.pop(0) if free else -1
            missing += page < 0
            for c in caches:
                if page >= 0:
                    c[page] = c[row[-1]]
            row[-1] = page
        seen.add(parent)
        for b in row:
            if 0 <= b < blocks:
                counts[b] += 1
        new.append(row + [-1] * (cols - len(row)))
        new_lens.append(n)
    like = lambda x, shape: torch.tensor(x, dtype=torch.int32, device=block_table.device).reshape(shape)
    return like(new, (len(new), cols)), like(new_lens, -1), like(counts, -1), missing


def resize_pages_torch(block_table, seq_lens, new_lens, ref_count, block_size):
    """Statement of resize_pages row by row: (out_table, out_ref_count, missing)."""
    rows, cols = block_table.shape
    blocks, table, counts = len(ref_count), block_table.tolist(), ref_count.tolist()
    free = [b for b in range(blocks) if counts[b] == 0]
    missing = 0
    for row, n, m in zip(table, seq_lens.tolist(), new_lens.tolist()):
        had, has = _pages(n, block_size, cols), _pages(m, block_size, cols)
        for j in range(cols):
            if has <= j < had and 0 <= row[j] < blocks:
                counts[row[j]] -= 1
            if j >= has:
                row[j] = -1
            elif j >= had:
                row[j] = free.pop(0) if free else -1
                missing += row[j] < 0
                if row[j] >= 0:
                    counts[row[j]] += 1
    like = lambda x, shape: torch.tensor(x, dtype=torch.int32, device=block_table.device).reshape(shape)
    return like(table, (rows, cols)), like(counts, -1), missing


def keep_drafted_torch(caches, block_table, seq_lens, query_start_loc, keep, block_size):
    """Statement of keep_drafted token by token; the caches are written: out_lens."""
    starts, out = query_start_loc.tolist(), []
    for i, (n, mask) in enumerate(zip(seq_lens.tolist(), keep.tolist())):
        count = starts[i + 1] - starts[i]
        if not 0 <= count <= 64 or count > n:
            out.append(n)
            continue
        at = n - count
        for j in range(count):
            if mask >> j & 1:
                place = [int(block_table[i, t // block_size]) if t // block_size < block_table.shape[1] else -1 for t in (n - count + j, at)]
                if all(0 <= b < c.shape[0] for b in place for c in caches):
                    for c in caches:
                        c[place[1], at % block_size] = c[place[0], (n - count + j) % block_size]
                at += 1
        out.append(at)
    return torch.tensor(out, dtype=torch.int32, device=block_table.device)
