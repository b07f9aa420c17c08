"""A step of beam search over a model of attention and recurrent layers, as cases that can be timed and checked.

A serving program that decodes with beams, or drafts trees, over paged caches and recurrent states meets these operators:

* ``prompt``: linear attention with a decay for each head over whole prompts, sequences of different lengths packed one after the
  other, from a carried state or none, and the states that they end with.
* ``step``: the same for one new token of every sequence; each reads a state's slot and writes another, which is how beams
  that continue one parent get its state.
* ``beam``: the best continuations over beams and vocabulary from a step's logits.
* ``fork``: the cache's pages follow the beams: rows take their parents' pages, partly filled ones are copied, the pages of beams
  that ended are given back, and every row gets room for its next token.
* ``keep``: the drafted tokens that a model agreed with are moved side by side in the cache, and the pages behind them are
  given back.

``run`` computes a case from elementary torch operations in 32 bits (whole numbers, and 64 bits for the beams' scores, whose order
counts) or, where ``own`` is set, by the framework's kernels.
"""
import functools
import random
import sys
from pathlib import Path

import torch

own = False

# (query heads, key/value heads) that the models of this repository's benchmarks and cases have.
HEADS = ((32, 8), (16, 2), (32, 4), (16, 8), (8, 8))
# Vocabularies of this repository's lm_heads.
VOCABULARIES = (151936, 248320)
MOST_TOKENS = 16384 * 32 * 128  # values of q in the largest prompt pass
MOST_STATES = 64 * 32 * 128 * 128  # values of all states of the largest step
MOST_LOGITS = 32 * 8 * 248320
MOST_POOL = 4 * 10000 * 16 * 8 * 256  # bytes of the layers' caches of the largest fork
PAGE = 16


def listed():
    return [
        # The smallest call: one short prompt, where latency counts.
        {"name": "prompt-1x17", "kind": "prompt", "batch": 1, "longest": 17, "ragged": 1.0, "heads": 8, "kv_heads": 8, "dim": 64, "dtype": "bf16", "fused": False, "carried": False},
        # An ordinary prefill batch from carried states (prompts in pieces), rows inside a fused qkv projection's output.
        {"name": "prompt-16x1k-ragged", "kind": "prompt", "batch": 16, "longest": 1024, "ragged": 0.0, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "fused": True, "carried": True},
        # Wide heads in fp16, odd lengths.
        {"name": "prompt-3x2111-d256", "kind": "prompt", "batch": 3, "longest": 2111, "ragged": 0.5, "heads": 16, "kv_heads": 2, "dim": 256, "dtype": "fp16", "fused": True, "carried": False},
        # One long prompt.
        {"name": "prompt-1x8192", "kind": "prompt", "batch": 1, "longest": 8192, "ragged": 1.0, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "fused": True, "carried": False},
        # Plain decoding of one sequence, then a loaded server's step.
        {"name": "step-1", "kind": "step", "batch": 1, "heads": 8, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        {"name": "step-64", "kind": "step", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # One request of four beams; a loaded server with eight beams a request, twice as many candidates as beams.
        {"name": "beam-1x4", "kind": "beam", "batch": 1, "beams": 4, "count": 4, "vocab": 151936, "dtype": "bf16", "first": False},
        {"name": "beam-32x8", "kind": "beam", "batch": 32, "beams": 8, "count": 16, "vocab": 248320, "dtype": "bf16", "first": False},
        # Four beams' pages in one layer's 8-bit cache; a loaded server's in four layers.
        {"name": "fork-1x4", "kind": "fork", "batch": 1, "beams": 4, "context": 700, "new": 90, "layers": 1, "kv_heads": 8, "dim": 128, "cache": "int8"},
        {"name": "fork-32x8", "kind": "fork", "batch": 32, "beams": 8, "context": 2048, "new": 200, "layers": 4, "kv_heads": 8, "dim": 128, "cache": "int8"},
        # One request's drafted tree of 16 bits; a loaded server's trees in four layers.
        {"name": "keep-1x7", "kind": "keep", "batch": 1, "nodes": 7, "context": 777, "layers": 1, "kv_heads": 2, "dim": 256, "cache": "16"},
        {"name": "keep-64x40", "kind": "keep", "batch": 64, "nodes": 40, "context": 1500, "layers": 4, "kv_heads": 8, "dim": 128, "cache": "int8"},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random())) if hi > lo else lo


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "step", "beam", "beam", "fork", "keep"))
    heads, kv_heads = rng.choice(HEADS)
    dim = rng.choice((64, 128, 128, 256))
    dtype = "fp16" if rng.random() < 0.3 else "bf16"
    if kind == "prompt":
        longest = _log_int(rng, 1, 8192)
        batch = _log_int(rng, 1, max(1, min(64, MOST_TOKENS // (longest * heads * max(dim, 128)), 16384 // longest)))
        return {"kind": kind, "batch": batch, "longest": longest, "ragged": rng.choice((0.0, 0.5, 1.0)), "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "dtype": dtype, "fused": rng.random() < 0.5, "carried": rng.random() < 0.5}
    if kind == "step":
        return {"kind": kind, "batch": _log_int(rng, 1, min(256, MOST_STATES // (heads * dim * dim))), "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    if kind == "beam":
        beams = rng.randint(1, 12)
        vocab = rng.choice(VOCABULARIES + (_log_int(rng, 500, 200000),))
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        batch = _log_int(rng, 1, max(1, min(64, MOST_LOGITS // (beams * vocab * (2 if dtype == "fp32" else 1)))))
        return {"kind": kind, "batch": batch, "beams": beams, "count": rng.choice((beams, 2 * beams, 2 * beams + 1)), "vocab": vocab, "dtype": dtype, "first": rng.random() < 0.2}
    layers, cache = rng.randint(1, 4), rng.choice(("int8", "16"))
    row = layers * kv_heads * dim * (2 if cache == "int8" else 4)
    case = {"kind": kind, "layers": layers, "kv_heads": kv_heads, "dim": dim, "cache": cache}
    if kind == "fork":
        beams, context, new = rng.randint(2, 10), _log_int(rng, 1, 4096), _log_int(rng, 1, 300)
        most = MOST_POOL // (row * (context + beams * (new + 3 * PAGE)))
        return {**case, "batch": _log_int(rng, 1, max(1, min(64, most))), "beams": beams, "context": context, "new": new}
    nodes, context = _log_int(rng, 1, 64), _log_int(rng, 1, 4096)
    return {**case, "batch": _log_int(rng, 1, max(1, min(64, MOST_POOL // (row * (context + nodes + PAGE))))), "nodes": nodes, "context": context}


# ---------------------------------------------------------------------------------- inputs
def _dtype(case):
    return {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}[case["dtype"]]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case, what, lo, hi):
    """One sequence has the longest length; the others lie between `lo` and `hi`. They are the case's own: the shapes of a pass do
    not go by the seed."""
    rng = random.Random(repr(sorted(case.items())) + what)
    n = [rng.randint(lo, hi) for _ in range(case["batch"])]
    n[rng.randrange(case["batch"])] = hi
    return n


def _prompt_lengths(case):
    return _lengths(case, "longest", max(1, int(case["ragged"] * case["longest"])), case["longest"])


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _starts(lengths):
    return torch.tensor([0] + lengths).cumsum(0).to("cuda", torch.int32)


def _hidden(g, *shape):
    """Rows as projections give them: N(0, 1) with a few channels of larger magnitude."""
    x = torch.empty(*shape, device="cuda", dtype=torch.float32).normal_(generator=g)
    x[..., torch.randint(0, shape[-1], (3,), device="cuda", generator=g)] *= 4
    return x


def _decays(heads):
    """Logarithms of the heads' decays, from windows of a token to windows of some hundreds."""
    return -(2.0 ** (-8.0 * (torch.arange(heads, device="cuda") + 1) / heads))


def _states(g, slots, h, d):
    return torch.empty(slots, h, d, d, device="cuda").normal_(generator=g).mul_(4)


def _pools(g, case, blocks):
    """Every layer's filled cache: [blocks, KV, page, 2 D], in 8 bits with scales [blocks, KV, page, 2] or in 16."""
    kv, d, pools = case["kv_heads"], case["dim"], []
    for _ in range(case["layers"]):
        if case["cache"] == "int8":
            pool = torch.randint(-(1 << 62), 1 << 62, (blocks, kv, PAGE, d // 4), device="cuda", generator=g).view(torch.int8)
            pools += [pool, torch.rand(blocks, kv, PAGE, 2, device="cuda", generator=g) * 0.02 + 0.015]
        else:
            pools.append(torch.empty(blocks, kv, PAGE, 2 * d, device="cuda", dtype=torch.bfloat16).normal_(generator=g))
    return pools


def _prepare_fork(case, g, s):
    """Beams that share their prompt's pages and have pages of their own behind, then a step's parents."""
    b, beams, rows = case["batch"], case["beams"], case["batch"] * case["beams"]
    prompt = torch.tensor(_lengths(case, "context", (case["context"] + 1) // 2, case["context"]), device="cuda")
    lengths = prompt.repeat_interleave(beams) + case["new"]
    shared, pages = (prompt // PAGE).repeat_interleave(beams)[:, None], -(-lengths // PAGE)
    cols = int(-(-(case["context"] + case["new"] + 1) // PAGE))
    at = torch.arange(cols, device="cuda").expand(rows, cols)
    row = torch.arange(rows, device="cuda")[:, None]
    owner = torch.where(at < shared, row // beams * beams, row)  # the request's first beam names the prompt's pages
    cells = owner * cols + at
    used = torch.unique(cells[at < pages[:, None]])
    blocks = used.numel() + 2 * rows + 5  # what a step may take, and a few more
    names = torch.randperm(blocks, device="cuda", generator=g)[:used.numel()]
    table = torch.full((rows * cols,), -1, device="cuda", dtype=torch.int64)
    table[used] = names
    s["table"] = torch.where(at < pages[:, None], table[cells], -1).to(torch.int32)
    s["lengths"] = lengths.to(torch.int32)
    s["refs"] = torch.bincount(s["table"][s["table"] >= 0].long(), minlength=blocks).to(torch.int32)
    s["parents"] = (torch.randint(0, beams, (b, beams), device="cuda", generator=g) + torch.arange(b, device="cuda")[:, None] * beams).flatten().to(torch.int32)
    s["pools"] = _pools(g, case, blocks)
    s.update(new_table=torch.empty_like(s["table"]), new_lengths=torch.empty_like(s["lengths"]), new_refs=torch.empty_like(s["refs"]))


def _prepare_keep(case, g, s):
    """Trees of drafted tokens behind contexts, and the path of each that is kept."""
    b, nodes = case["batch"], case["nodes"]
    counts = _lengths(case, "nodes", (nodes + 1) // 2, nodes)
    lengths = torch.tensor(_lengths(case, "context", (case["context"] + 1) // 2, case["context"])) + torch.tensor(counts)
    cols = -(-(case["context"] + nodes) // PAGE)
    blocks = b * cols + 3
    table = torch.randperm(blocks, device="cuda", generator=g)[:b * cols].view(b, cols)
    pages = (-(-lengths // PAGE)).cuda()[:, None]
    s["table"] = torch.where(torch.arange(cols, device="cuda") < pages, table, -1).to(torch.int32)
    s["lengths"], s["starts"] = lengths.to("cuda", torch.int32), _starts(counts)
    s["refs"] = torch.bincount(s["table"][s["table"] >= 0].long(), minlength=blocks).to(torch.int32)
    # A path of a tree: each node is kept or not, the root is.
    kept = torch.rand(b, nodes, device="cuda", generator=g) < 0.4
    kept[:, 0] = True
    kept &= torch.arange(nodes, device="cuda") < torch.tensor(counts, device="cuda")[:, None]
    bit = torch.tensor([1 << i if i < 63 else -(1 << 63) for i in range(nodes)], device="cuda")
    s["kept"] = (kept.long() * bit).sum(1)
    s["pools"] = _pools(g, case, blocks)
    s.update(new_lengths=torch.empty_like(s["lengths"]), new_table=torch.empty_like(s["table"]), new_refs=torch.empty_like(s["refs"]))


def prepare(case, seed):
    g, s = _generator(seed), {"case": case}
    if case["kind"] == "fork":
        _prepare_fork(case, g, s)
        return s
    if case["kind"] == "keep":
        _prepare_keep(case, g, s)
        return s
    b, dt = case["batch"], _dtype(case)
    if case["kind"] == "beam":
        rows, k = b * case["beams"], case["count"]
        logits = torch.empty(rows, case["vocab"], device="cuda").normal_(generator=g).mul_(2.5)
        logits[torch.rand(rows, case["vocab"], device="cuda", generator=g) < 0.01] = -torch.inf  # tokens that a grammar forbids
        s["logits"] = logits.to(dt)
        s["scores"] = torch.rand(rows, device="cuda", generator=g) * -4 - 20
        if case["first"]:  # after the prompt only the first beam of a request lives
            s["scores"].view(b, -1)[:, 1:] = -torch.inf
        s.update(best=torch.empty(b, k, device="cuda"), parents=torch.empty(b, k, device="cuda", dtype=torch.int32),
                 tokens=torch.empty(b, k, device="cuda", dtype=torch.int64))
        return s
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    s["decay"] = _decays(h)
    if case["kind"] == "step":
        s["q"], s["k"], s["v"] = _hidden(g, b, h + 2 * kv, d).to(dt).split((h, kv, kv), dim=1)
        s["state"] = _states(g, 2 * b, h, d)
        s["read"] = torch.randint(0, b, (b,), device="cuda", generator=g).to(torch.int32)  # beams continue some parents twice
        s["write"] = (torch.randperm(b, device="cuda", generator=g) + b).to(torch.int32)
        s["out"] = torch.empty(b, h, d, device="cuda", dtype=dt)
        return s
    n = _prompt_lengths(case)
    total = sum(n)
    if case["fused"]:  # one projection's output, q, k and v beside each other in its rows
        s["q"], s["k"], s["v"] = _hidden(g, total, h + 2 * kv, d).to(dt).split((h, kv, kv), dim=1)
    else:
        s["q"], s["k"], s["v"] = (_hidden(g, total, x, d).to(dt) for x in (h, kv, kv))
    s["state"] = _states(g, 2 * b, h, d)
    s["read"] = torch.randperm(b, device="cuda", generator=g).to(torch.int32) if case["carried"] else None
    s["write"] = (torch.randperm(b, device="cuda", generator=g) + b).to(torch.int32)
    s.update(cu=_starts(n), out=torch.empty(total, h, d, device="cuda", dtype=dt))
    return s


# ---------------------------------------------------------------------------------- passes
@functools.lru_cache(maxsize=None)
def _framework():
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "vllm-exact_amd"))
    from vllm_exact import beam, linear_attn, pages
    return linear_attn, beam, pages


def _views(s):
    """The layers' caches as (blocks, page, KV, D) keys and values, and (blocks, page, KV) scales."""
    return [v for p in s["pools"] for v in (p.transpose(1, 2).unbind(-1) if p.dtype == torch.float32 else p.transpose(1, 2).split(s["case"]["dim"], dim=-1))]


def _run_own(s):
    linear_attn, beam, pages = _framework()
    case = s["case"]
    if case["kind"] == "prompt":
        linear_attn.linear_prompt(s["q"], s["k"], s["v"], s["cu"], s["decay"], case["dim"] ** -0.5, s["out"], s["state"], s["read"], s["write"])
        return [s["out"], s["state"]]
    if case["kind"] == "step":
        linear_attn.linear_step(s["q"], s["k"], s["v"], s["decay"], case["dim"] ** -0.5, s["out"], s["state"], s["read"], s["write"])
        return [s["out"], s["state"]]
    if case["kind"] == "beam":
        return list(beam.beam_select(s["logits"], s["scores"], case["beams"], s["best"], s["parents"], s["tokens"]))
    if case["kind"] == "fork":
        short = pages.fork_pages(_views(s), s["table"], s["lengths"], s["parents"], s["refs"], PAGE, s["new_table"], s["new_lengths"], s["new_refs"])
        short2 = pages.resize_pages(s["new_table"], s["new_lengths"], s["new_lengths"] + 1, s["new_refs"], PAGE)
        return [s["new_table"], s["new_lengths"], s["new_refs"], short, short2] + s["pools"]
    pages.keep_drafted(_views(s), s["table"], s["lengths"], s["starts"], s["kept"], PAGE, s["new_lengths"])
    short = pages.resize_pages(s["table"], s["lengths"], s["new_lengths"], s["refs"], PAGE, s["new_table"], s["new_refs"])
    return [s["new_table"], s["new_lengths"], s["new_refs"], short] + s["pools"]


def _by_head(x, rows, heads):
    """Rows (batch, n) of (tokens, KV, D) as (batch * heads, n, D) in 32 bits."""
    x = x[rows].float().repeat_interleave(heads // x.shape[1], dim=2)
    return x.transpose(1, 2).reshape(-1, rows.shape[1], x.shape[-1])


def _plain_prompt(s):
    case, cu = s["case"], s["cu"]
    b, n, h, d, g = case["batch"], case["longest"], case["heads"], case["dim"], s["decay"].view(1, -1, 1)
    at = torch.arange(n, device="cuda")
    total, length = s["q"].shape[0], (cu[1:] - cu[:-1]).view(b, 1, 1)
    rows = (cu[:-1, None] + at).clamp_(max=total - 1)
    q, k, v = (_by_head(s[x], rows, h) for x in "qkv")
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).view(b, h, n, n)
    back = at[:, None] - at
    scores.mul_((g.view(h, 1, 1) * back.clamp(min=0)).exp_()).masked_fill_(back < 0, 0)
    out = torch.bmm(scores.view(b * h, n, n), v)
    del scores
    left = length - 1 - at  # tokens of the sequence after this one
    weight = (g * left.clamp(min=0)).exp().masked_fill(left < 0, 0).view(b * h, n, 1)
    state = torch.bmm((k * weight).transpose(1, 2).contiguous(), v).view(b, h, d, d)
    if s["read"] is not None:
        start = s["state"][s["read"].long()]
        out += torch.bmm(q, start.view(b * h, d, d)) * (g * (at + 1)).exp().expand(b, h, n).reshape(b * h, n, 1)
        state += start * (g * length).exp().unsqueeze(-1)
    s["state"][s["write"].long()] = state
    rows = torch.arange(total, device="cuda")
    seq = torch.searchsorted(cu[1:], rows.to(torch.int32), right=True)
    out = out.view(b, h, n, d)[seq, :, rows - cu[seq]] * d ** -0.5
    return [out.to(s["q"].dtype), s["state"]]


def _plain_step(s):
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    q, k, v = s["q"].float(), s["k"].float().repeat_interleave(group, dim=1), s["v"].float().repeat_interleave(group, dim=1)
    state = s["state"][s["read"].long()] * s["decay"].exp().view(1, -1, 1, 1) + k[..., None] * v[..., None, :]
    s["state"][s["write"].long()] = state
    out = (q[..., None] * state).sum(dim=2) * case["dim"] ** -0.5
    return [out.to(s["q"].dtype), s["state"]]


def _plain_beam(s):
    case, k = s["case"], s["case"]["count"]
    x = s["logits"].double()
    top = x.amax(dim=1, keepdim=True)
    x = x - top
    x = (s["scores"].double()[:, None] + (x - x.exp().sum(dim=1, keepdim=True).log())).nan_to_num(-torch.inf, torch.inf, -torch.inf).view(case["batch"], -1)
    kth = x.topk(k, dim=1).values[:, -1:]
    above, ties = x > kth, x == kth
    taken = above | (ties & (ties.cumsum(dim=1) <= k - above.sum(dim=1, keepdim=True)))  # the first of those that tie for the last places
    at = taken.nonzero()[:, 1].view(-1, k)
    best, order = x.gather(1, at).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    first = torch.arange(case["batch"], device="cuda")[:, None] * case["beams"]
    none = best == -torch.inf
    return [best.float(), (first + at // case["vocab"]).masked_fill(none, -1).to(torch.int32), (at % case["vocab"]).masked_fill(none, -1)]


def _references(table, lengths, blocks):
    """How often the rows name each page."""
    at = torch.arange(table.shape[1], device="cuda")
    named = (at < (-(-lengths // PAGE))[:, None]) & (table >= 0)
    return torch.zeros(blocks + 1, device="cuda", dtype=torch.int32).index_add_(
        0, torch.where(named, table, blocks).flatten().long(), torch.ones(table.numel(), device="cuda", dtype=torch.int32))[:blocks]


def _take(refs, wanted):
    """The lowest free pages, one for each place that wants one in order: those pages (-1: none left), and how many were missing."""
    free = (refs == 0).nonzero()[:, 0]
    rank = wanted.flatten().cumsum(0).view_as(wanted) - 1
    got = torch.cat([free, free.new_full((wanted.numel(),), -1)])[rank.clamp(min=0)]
    return got, (wanted.sum() - free.numel()).clamp(min=0).to(torch.int32).view(1)


def _plain_resize(table, lengths, new_lengths, refs):
    at = torch.arange(table.shape[1], device="cuda")
    had, has = -(-lengths // PAGE)[:, None], -(-new_lengths // PAGE)[:, None]
    wanted = (at >= had) & (at < has)
    got, short = _take(refs, wanted)
    new = torch.where(wanted, got, table).masked_fill(at >= has, -1).to(torch.int32)
    return new, refs - _references(table, lengths, refs.numel()) + _references(new, new_lengths, refs.numel()), short


def _plain_fork(s):
    table, lengths, parents, refs = s["table"], s["lengths"], s["parents"].long(), s["refs"]
    rows = torch.arange(len(parents), device="cuda")
    new_lengths = lengths[parents]
    last = (new_lengths - 1).clamp(min=0) // PAGE
    page = table[parents].gather(1, last[:, None].long())[:, 0]
    first = torch.full_like(rows, len(rows)).scatter_reduce_(0, parents, rows, "amin")[parents] == rows
    copied = (new_lengths % PAGE != 0) & ~(first & (refs[page.clamp(min=0).long()] == 1))
    got, short = _take(refs, copied)
    new = table[parents].scatter(1, last[:, None].long(), torch.where(copied, got, page)[:, None].to(torch.int32))
    at = copied & (got >= 0)
    new_refs = refs - _references(table, lengths, refs.numel()) + _references(new, new_lengths, refs.numel())
    [p.index_copy_(0, got[at], p[page[at].long()]) for p in s["pools"]]
    new, new_refs, short2 = _plain_resize(new, new_lengths, new_lengths + 1, new_refs)
    return [new, new_lengths, new_refs, short, short2] + s["pools"]


def _plain_keep(s):
    case, table, lengths = s["case"], s["table"], s["lengths"]
    counts = s["starts"][1:] - s["starts"][:-1]
    node = torch.arange(case["nodes"], device="cuda")
    kept = ((s["kept"][:, None] >> node) & 1 == 1) & (node < counts[:, None])
    context = (lengths - counts)[:, None]
    rank = kept.cumsum(dim=1) - 1
    request, at = kept.nonzero(as_tuple=True)
    old, new = (context + node)[request, at], (context + rank)[request, at]
    source, target = table[request, old // PAGE].long(), table[request, new // PAGE].long()
    [p.index_put_((target, slice_, new % PAGE), p[source, slice_, old % PAGE]) for p, slice_ in _token_rows(s["pools"])]
    new_lengths = (context[:, 0] + kept.sum(dim=1)).to(torch.int32)
    new_table, new_refs, short = _plain_resize(table, lengths, new_lengths, s["refs"])
    return [new_table, new_lengths, new_refs, short] + s["pools"]


def _token_rows(pools):
    """The pools with their heads first, and the index of all heads beside one of tokens."""
    return [(p, torch.arange(p.shape[1], device="cuda")[:, None]) for p in pools]


def run(state):
    if own:
        return _run_own(state)
    return {"prompt": _plain_prompt, "step": _plain_step, "beam": _plain_beam, "fork": _plain_fork, "keep": _plain_keep}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------- accounting
def work(case):
    b = case["batch"]
    if case["kind"] == "beam":
        size = 4 if case["dtype"] == "fp32" else 2
        rows = b * case["beams"]
        return {"bytes": rows * (case["vocab"] * size + 4) + b * case["count"] * 16, "flops": 3 * rows * case["vocab"]}
    if case["kind"] in ("prompt", "step"):
        h, kv, d = case["heads"], case["kv_heads"], case["dim"]
        total = b if case["kind"] == "step" else sum(_prompt_lengths(case))
        # a token: its row of scores with the state, and the state's update
        states = 2 if case["kind"] == "step" or case["carried"] else 1
        return {"bytes": total * d * 2 * (2 * h + 2 * kv) + states * b * h * d * d * 4 + 4 * h, "flops": 4 * total * h * d * d}
    token = case["layers"] * case["kv_heads"] * (2 * case["dim"] + 8 if case["cache"] == "int8" else 4 * case["dim"])
    if case["kind"] == "fork":  # a third of the rows copy half a page; tables and counts in and out
        rows, cols = b * case["beams"], -(-(case["context"] + case["new"] + 1) // PAGE)
        return {"bytes": rows // 3 * token * PAGE + 8 * rows * (cols + 2) + 8 * rows * (case["new"] // PAGE), "flops": 0}
    return {"bytes": 2 * b * (case["nodes"] // 4) * token + 16 * b * -(-(case["context"] + case["nodes"]) // PAGE), "flops": 0}


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    if case["kind"] in ("fork", "keep"):  # whole numbers and moved values: nothing is computed
        return None

    def recurrence(case, s):
        """The recurrence, a token of all sequences at a time."""
        cu, group = s["cu"].long(), case["heads"] // case["kv_heads"]
        length = cu[1:] - cu[:-1]
        decay = s["decay"].double().exp().view(1, -1, 1, 1)
        state = torch.zeros(s["state"][:case["batch"]].shape, device="cuda", dtype=torch.float64)
        if s["read"] is not None:
            state = s["state"][s["read"].long()].double()
        out = torch.empty(s["out"].shape, device="cuda", dtype=torch.float64)
        for t in range(case["longest"]):
            live = (length > t).nonzero()[:, 0]
            rows = cu[live] + t
            k, v = (s[x][rows].double().repeat_interleave(group, dim=1) for x in "kv")
            now = decay * state[live] + k.unsqueeze(3) * v.unsqueeze(2)
            state[live] = now
            out[rows] = torch.matmul(s["q"][rows].double().unsqueeze(2), now).squeeze(2) * case["dim"] ** -0.5
        states = s["state"].double()
        states[s["write"].long()] = state
        return [out, states]

    s = prepare(case, seed)
    if case["kind"] == "prompt":
        return recurrence(case, s)
    if case["kind"] == "step":
        one = {**case, "longest": 1}
        s["cu"] = torch.arange(case["batch"] + 1, device="cuda")
        return recurrence(one, s)
    best = []
    for logits, scores in zip(s["logits"].view(case["batch"], case["beams"], -1), s["scores"].view(case["batch"], -1)):
        x = scores.double()[:, None] + torch.log_softmax(logits.double(), dim=1)
        best.append(x.flatten().sort(descending=True).values[:case["count"]])
    return [torch.stack(best), None, None]
