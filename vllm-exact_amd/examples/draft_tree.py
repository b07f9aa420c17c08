"""Greedy serving with an 8-bit KV cache and drafted trees, on a small transformer with random weights.

    python vllm-exact_amd/examples/draft_tree.py

The serving operators as a decoding loop uses them:

* prompts of different lengths, packed, go through ``prompt_attention``; their keys and values through ``write_cache``;
* each step drafts a tree for every request: its root is the token that the last step decided, below it hang guesses from
  the request's own text. The nodes' keys and values are written behind the context and ``tree_decode`` scores all nodes of
  all requests in one call;
* the longest path that the model agrees with is kept. Its keys and values lie apart in the cache where a sibling was drafted
  between them: ``keep_drafted`` moves them side by side, in the caches of all layers at once.

``generate(..., guesses=0)`` drafts nothing but the root: plain decoding, the same tokens.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from vllm_exact.int8_cache import make_cache, write_cache  # noqa: E402
from vllm_exact.pages import keep_drafted  # noqa: E402
from vllm_exact.prompt_attn import prompt_attention  # noqa: E402
from vllm_exact.tree_attn import tree_decode  # noqa: E402

PAGE = 16


class Model:
    """Pre-norm layers of attention and a gated MLP in fp32, queries, keys and values in bf16; positions enter as a rotation of
    queries and keys. The layers add little to the embedding, so that texts repeat themselves and drafts come true."""

    def __init__(self, layers=2, heads=8, kv_heads=2, dim=64, vocab=64, device="cuda", seed=0):
        g = torch.Generator().manual_seed(seed)
        hidden = heads * dim
        w = lambda *s: (torch.randn(*s, generator=g) / s[0] ** 0.5).to(device)
        self.heads, self.kv_heads, self.dim, self.device = heads, kv_heads, dim, device
        self.embed = w(vocab, hidden) * vocab ** 0.5
        self.layers = [(w(hidden, (heads + 2 * kv_heads) * dim), 0.3 * w(hidden, hidden), w(hidden, 4 * hidden), 0.3 * w(2 * hidden, hidden))
                       for _ in range(layers)]
        self.head = w(hidden, vocab)
        self.freq = 10000.0 ** -(torch.arange(dim // 2, device=device) / (dim // 2))

    def rotate(self, x, pos):
        angle = pos[:, None, None].float() * self.freq
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], dim=-1).to(torch.bfloat16)

    def forward(self, tokens, pos, attend):
        """Logits of all rows; attend(layer, q, k, v) gives a layer's attention."""
        norm = lambda x: torch.nn.functional.rms_norm(x, x.shape[-1:])
        x = self.embed[tokens]
        for i, (qkv, proj, up, down) in enumerate(self.layers):
            q, k, v = (norm(x) @ qkv).view(len(x), -1, self.dim).split((self.heads, self.kv_heads, self.kv_heads), dim=1)
            x = x + attend(i, self.rotate(q, pos), self.rotate(k, pos), v.bfloat16()).flatten(1) @ proj
            gate, value = (norm(x) @ up).chunk(2, dim=-1)
            x = x + (torch.nn.functional.silu(gate) * value) @ down
        return norm(x) @ self.head


def draft(text, guesses):
    """A tree below the last token of `text`: [(token, parent)], the root first. What followed earlier occurrences of the
    last token is drafted as chains of up to three tokens, the latest occurrence first, prefixes shared."""
    nodes = [(text[-1], -1)]
    for at in range(len(text) - 2, -1, -1):
        if text[at] != text[-1]:
            continue
        parent = 0
        for token in text[at + 1:at + 4]:
            child = next((i for i, n in enumerate(nodes) if n == (token, parent)), None)
            if child is None:
                if len(nodes) > guesses:
                    return nodes
                nodes.append((token, parent))
                child = len(nodes) - 1
            parent = child
    return nodes


def generate(model, prompts, count, guesses=7):
    """`count` greedy tokens after each prompt, and how many steps they took."""
    dev, dim, n = model.device, model.dim, len(prompts)
    scale = dim ** -0.5
    most = max(map(len, prompts)) + count + guesses + 4
    pages = -(-most // PAGE)
    table = torch.randperm(n * pages, device=dev).view(n, pages).to(torch.int32)
    caches = [make_cache(n * pages, PAGE, model.kv_heads, dim, dev) for _ in model.layers]
    ints = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device=dev)
    starts = lambda lengths: ints([0] + lengths).cumsum(0).to(torch.int32)

    def slots(places):  # [(request, place)] as places of the cache
        r, at = ints([p[0] for p in places], torch.int64), ints([p[1] for p in places], torch.int64)
        return table[r, at // PAGE].long() * PAGE + at % PAGE

    # The prompts, packed.
    lengths = [len(p) for p in prompts]
    cu = starts(lengths)
    pos = torch.cat([torch.arange(x, device=dev) for x in lengths])
    where = slots([(i, j) for i, x in enumerate(lengths) for j in range(x)])

    def attend_prompt(layer, q, k, v):
        write_cache(k, v, *caches[layer], where)
        return prompt_attention(q, k, v, cu, scale, torch.empty(q.shape, device=dev))

    logits = model.forward(ints(sum(prompts, []), torch.int64), pos, attend_prompt)
    texts = [p + [t] for p, t in zip(prompts, logits[cu[1:].long() - 1].argmax(-1).tolist())]
    steps = 0
    while min(len(t) - len(p) for t, p in zip(texts, prompts)) < count:
        steps += 1
        trees = [draft(t, guesses) for t in texts]
        ctx = [len(t) - 1 for t in texts]  # cached tokens of each request
        masks, depth = [], []
        for tree in trees:
            m, d = [], []
            for i, (_, parent) in enumerate(tree):
                m.append((m[parent] if parent >= 0 else 0) | 1 << i)
                d.append(d[parent] + 1 if parent >= 0 else 0)
            masks += m
            depth.append(d)
        sizes = [len(t) for t in trees]
        qsl, first = starts(sizes), ints(ctx)
        lens = first + ints(sizes)
        bits = ints(masks, torch.int64)
        where = slots([(i, ctx[i] + j) for i, s in enumerate(sizes) for j in range(s)])
        pos = ints([c + x for c, d in zip(ctx, depth) for x in d])

        def attend_tree(layer, q, k, v):
            key, value, key_scale, value_scale = caches[layer]
            write_cache(k, v, key, value, key_scale, value_scale, where)
            return tree_decode(q, key, value, table, lens, qsl, bits, scale, torch.empty(q.shape, device=dev), guesses + 1, most,
                               key_scale=key_scale, value_scale=value_scale)

        best = model.forward(ints([t for tree in trees for t, _ in tree], torch.int64), pos, attend_tree).argmax(-1).tolist()
        keep, row = [], 0  # of each request, the kept nodes as bits
        for i, tree in enumerate(trees):
            kept = [0]
            while True:
                token = best[row + kept[-1]]
                texts[i].append(token)
                child = next((j for j, node in enumerate(tree) if node == (token, kept[-1])), None)
                if child is None:
                    break
                kept.append(child)
            keep.append(masks[row + kept[-1]])
            row += len(tree)
        views = [view for cache in caches for view in cache]
        keep_drafted(views, table, lens, qsl, ints(keep, torch.int64), PAGE, torch.empty_like(lens))
    return [t[len(p):len(p) + count] for t, p in zip(texts, prompts)], steps


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--guesses", type=int, default=7)
    a = ap.parse_args()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 64, (int(n),), generator=g).tolist() for n in torch.randint(1, 200, (a.requests,), generator=g)]
    model = Model()
    plain, plain_steps = generate(model, prompts, a.tokens, 0)
    drafted, steps = generate(model, prompts, a.tokens, a.guesses)
    same = sum(x == y for x, y in zip(plain, drafted))
    print(f"{a.requests} requests, {a.tokens} tokens each: {plain_steps} steps without drafts, {steps} with; "
          f"{same} of {a.requests} texts are the same")


if __name__ == "__main__":
    main()
