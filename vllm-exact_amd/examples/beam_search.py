"""Beam search on a small hybrid model with random weights: attention layers over an 8-bit paged cache, recurrent layers of linear
attention between them.

    python vllm-exact_amd/examples/beam_search.py

A step of all beams of all requests, without a copy to the host:

* the beams' tokens go through the layers: ``write_cache`` and ``tree_decode`` (a tree of one token) in the attention layers,
  ``linear_step`` in the recurrent ones, each beam reading its parent's state and writing a slot of its own;
* ``beam_select`` scores all continuations and picks the best of each request;
* ``fork_pages`` gives the chosen beams their parents' pages, ``resize_pages`` room for the next token; states need no copy:
  the next step reads the parents' slots and writes the other half of the pool.

Prompts go through ``prompt_attention``, ``write_cache`` and ``linear_prompt`` once, then every beam but a request's first scores -inf.
"""
import argparse
import sys
from pathlib import Path
from types import SimpleNamespace

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from vllm_exact.beam import beam_select  # noqa: E402
from vllm_exact.int8_cache import make_cache, write_cache  # noqa: E402
from vllm_exact.linear_attn import linear_prompt, linear_step  # noqa: E402
from vllm_exact.pages import fork_pages, resize_pages  # noqa: E402
from vllm_exact.prompt_attn import prompt_attention  # noqa: E402
from vllm_exact.tree_attn import tree_decode  # noqa: E402

PAGE = 16
KERNELS = SimpleNamespace(beam_select=beam_select, fork_pages=fork_pages, resize_pages=resize_pages)


class Model:
    """Pre-norm layers in fp32, queries, keys and values in bf16: attention, whose positions enter as a rotation, and linear
    attention in turn, with a gated MLP each."""

    def __init__(self, layers=4, heads=4, kv_heads=2, dim=64, vocab=97, device="cuda", seed=0):
        g = torch.Generator().manual_seed(seed)
        hidden = heads * dim
        w = lambda *s: (torch.randn(*s, generator=g) / s[0] ** 0.5).to(device)
        self.heads, self.kv_heads, self.dim, self.vocab, self.device = heads, kv_heads, dim, vocab, device
        self.embed = w(vocab, hidden) * vocab ** 0.5
        self.layers = [(w(hidden, (heads + 2 * kv_heads) * dim), w(hidden, hidden), w(hidden, 4 * hidden), w(2 * hidden, hidden)) for _ in range(layers)]
        self.head = 2 * w(hidden, vocab)
        self.freq = 10000.0 ** -(torch.arange(dim // 2, device=device) / (dim // 2))
        self.log_decay = -(2.0 ** -(8.0 * (torch.arange(heads, device=device) + 1) / heads))

    def recurrent(self, layer):
        return layer % 2 == 1

    def rotate(self, x, pos):
        angle = pos[:, None, None].float() * self.freq
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], dim=-1)

    def forward(self, tokens, pos, mix):
        """Logits of all rows; mix(layer, q, k, v) is a layer's attention, of one kind or the other."""
        norm = lambda x: torch.nn.functional.rms_norm(x, x.shape[-1:])
        x = self.embed[tokens]
        for i, (qkv, proj, up, down) in enumerate(self.layers):
            q, k, v = (norm(x) @ qkv).view(len(x), -1, self.dim).split((self.heads, self.kv_heads, self.kv_heads), dim=1)
            if not self.recurrent(i):
                q, k = self.rotate(q, pos), self.rotate(k, pos)
            x = x + norm(mix(i, q.bfloat16(), k.bfloat16(), v.bfloat16()).flatten(1)) @ proj
            gate, value = (norm(x) @ up).chunk(2, dim=-1)
            x = x + (torch.nn.functional.silu(gate) * value) @ down
        return norm(x) @ self.head


def generate(model, prompts, count, beams=4, kernels=KERNELS):
    """The `beams` best texts of `count` tokens after each prompt that beam search finds, with their scores: (tokens (requests, beams,
    count), scores (requests, beams), the pages that are left in use once every row has been given back)."""
    dev, dim, n, rows = model.device, model.dim, len(prompts), len(prompts) * beams
    scale, most = dim ** -0.5, max(map(len, prompts)) + count + 1
    cols = -(-most // PAGE)
    attention = [i for i in range(len(model.layers)) if not model.recurrent(i)]
    caches = {i: make_cache(rows * (cols + 1), PAGE, model.kv_heads, dim, dev) for i in attention}
    views = [view for cache in caches.values() for view in cache]
    states = [torch.zeros(2 * rows, model.heads, dim, dim, device=dev) for _ in model.layers]
    ints = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device=dev)
    place = lambda table, row, at: table[row, at // PAGE].long() * PAGE + at % PAGE

    # The prompts, one row of the table and one state each.
    lengths = ints([len(p) for p in prompts])
    refs = torch.zeros(rows * (cols + 1), dtype=torch.int32, device=dev)
    table = torch.full((n, cols), -1, dtype=torch.int32, device=dev)
    kernels.resize_pages(table, torch.zeros_like(lengths), lengths, refs, PAGE)
    cu = ints([0] + [len(p) for p in prompts]).cumsum(0).to(torch.int32)
    row = torch.repeat_interleave(torch.arange(n, device=dev), lengths)
    pos = torch.arange(len(row), device=dev) - cu[:-1].long()[row]
    slots = place(table, row, pos)
    ends = rows + beams * torch.arange(n, dtype=torch.int32, device=dev)  # states: the steps' beams read the pool's upper half first

    def mix_prompt(i, q, k, v):
        out = torch.empty(q.shape, device=dev)
        if model.recurrent(i):
            return linear_prompt(q, k, v, cu, model.log_decay, scale, out, states[i], None, ends)
        write_cache(k, v, *caches[i], slots)
        return prompt_attention(q, k, v, cu, scale, out)

    logits = model.forward(ints(sum(prompts, []), torch.int64), pos, mix_prompt)[cu[1:].long() - 1]
    # Every request's beams are its prompt's row; after the first selection they are its best first tokens.
    logits = logits.repeat_interleave(beams, dim=0)
    scores = torch.full((n, beams), -torch.inf, device=dev)
    scores[:, 0] = 0
    scores = scores.flatten()
    of_beams = torch.arange(rows, dtype=torch.int32, device=dev) // beams
    texts = torch.zeros(rows, 0, dtype=torch.int64, device=dev)
    table, lengths = _fork(kernels, views, table, lengths, of_beams, refs)
    read = ends.repeat_interleave(beams)  # the slots that hold the beams' states
    half = 0
    for step in range(count):
        best, parents, tokens = kernels.beam_select(logits, scores, beams, torch.empty(n, beams, device=dev), torch.empty(n, beams, dtype=torch.int32, device=dev),
                                                    torch.empty(n, beams, dtype=torch.int64, device=dev))
        scores, parents, tokens = best.flatten(), parents.flatten(), tokens.flatten()
        texts = torch.cat([texts[parents.long()], tokens[:, None]], dim=1)
        if step + 1 == count:
            break
        table, lengths = _fork(kernels, views, table, lengths, parents, refs)
        kernels.resize_pages(table, lengths, lengths + 1, refs, PAGE)
        pos, lengths = lengths.long(), lengths + 1
        slots = place(table, torch.arange(rows, device=dev), pos)
        read = read[parents.long()]
        write = torch.arange(rows, dtype=torch.int32, device=dev) + half * rows
        qsl = torch.arange(rows + 1, dtype=torch.int32, device=dev)

        def mix_step(i, q, k, v):
            out = torch.empty(q.shape, device=dev)
            if model.recurrent(i):
                return linear_step(q, k, v, model.log_decay, scale, out, states[i], read, write)
            key, value, key_scale, value_scale = caches[i]
            write_cache(k, v, key, value, key_scale, value_scale, slots)
            return tree_decode(q, key, value, table, lengths, qsl, None, scale, out, 1, most, key_scale=key_scale, value_scale=value_scale)

        logits = model.forward(tokens, pos, mix_step)
        read, half = write, 1 - half
    kernels.resize_pages(table, lengths, torch.zeros_like(lengths), refs, PAGE)
    return texts.view(n, beams, count), scores.view(n, beams), int((refs != 0).sum())


def _fork(kernels, views, table, lengths, parents, refs):
    new, new_lengths = table.new_empty(len(parents), table.shape[1]), torch.empty_like(parents)
    kernels.fork_pages(views, table, lengths, parents, refs, PAGE, new, new_lengths)
    return new, new_lengths


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=32)
    a = ap.parse_args()
    g = torch.Generator().manual_seed(1)
    model = Model()
    prompts = [torch.randint(0, model.vocab, (int(n),), generator=g).tolist() for n in torch.randint(1, 200, (a.requests,), generator=g)]
    greedy = generate(model, prompts, a.tokens, 1)[1]
    texts, scores, left = generate(model, prompts, a.tokens, a.beams)
    print(f"{a.requests} requests, {a.beams} beams, {a.tokens} tokens: best log probability {scores[:, 0].mean():.2f} a text, greedy {greedy[:, 0].mean():.2f}; "
          f"{left} pages left in use")


if __name__ == "__main__":
    main()
