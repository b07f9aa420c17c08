"""CPU checks of linear attention, beam selection and the page operators: what the entry points refuse before anything is launched,
and the torch statements."""
import math

import pytest
import torch

from linear64 import bounds, linear64
from vllm_exact import _native as nx
from vllm_exact.beam import beam_select, beam_select_torch
from vllm_exact.int8_cache import make_cache
from vllm_exact.linear_attn import linear_attention_torch, linear_prompt, linear_step
from vllm_exact.pages import (copy_pages, fork_pages, fork_pages_torch, keep_drafted, keep_drafted_torch, resize_pages,
                              resize_pages_torch)

FAKE = 1 << 20  # never dereferenced: validation fails first
BF, F32 = nx.VXA_BF16, nx.VXA_F32


def calls(fn, defaults):
    return lambda **over: getattr(nx.lib(), fn)(*dict(defaults, **over).values())


def view(**over):
    return (nx.CacheView * 1)(nx.CacheView(**dict(dict(data=FAKE, stride_block=4096, stride_token=128, stride_head=2048, heads=2, row_bytes=64), **over)))


def test_linear_attention_refusals():
    rows = dict(q=FAKE, sqt=1024, sqh=128, k=FAKE, skt=256, skh=128, v=FAKE, svt=256, svh=128, dtype=BF)
    rest = dict(g=FAKE, scale=0.1, out=FAKE, od=BF, sot=1024, soh=128, state=FAKE, slots=4, sss=8 * 128 * 128, ssh=128 * 128, read=FAKE, write=FAKE,
                H=8, KV=2, D=128)
    prompt = calls("vxa_linear_prompt", dict(rows, cu=FAKE, n=2, tokens=100, **rest, ws=FAKE, wsb=1 << 40, st=None))
    step = calls("vxa_linear_step", dict(rows, n=2, **rest, st=None))
    for call in (prompt, step):
        assert call(n=0) == nx.VXA_OK
        for bad in (dict(n=-1), dict(H=0), dict(KV=0), dict(D=0), dict(H=7), dict(dtype=F32), dict(dtype=9), dict(od=9), dict(q=None), dict(k=None),
                    dict(v=None), dict(out=None), dict(g=None), dict(state=None), dict(slots=-1)):
            assert call(**bad) == nx.VXA_ERR_ARG, bad
        for bad in (dict(D=96), dict(D=32), dict(q=FAKE + 2), dict(k=FAKE + 8), dict(v=FAKE + 8), dict(sqt=1020), dict(skh=4), dict(svt=2), dict(state=FAKE + 4),
                    dict(sss=2), dict(ssh=6), dict(n=1 << 40), dict(slots=1 << 40), dict(n=1 << 24, H=1 << 16, KV=1)):
            assert call(**bad) == nx.VXA_ERR_UNSUPPORTED, bad
    assert prompt(tokens=-1) == nx.VXA_ERR_ARG and prompt(cu=None) == nx.VXA_ERR_ARG and prompt(tokens=1 << 40) == nx.VXA_ERR_UNSUPPORTED


def test_linear_attention_rows_too_far_apart():
    rows = dict(q=FAKE, sqt=1024, sqh=128, k=FAKE, skt=256, skh=128, v=FAKE, svt=256, svh=128, dtype=BF)
    rest = dict(g=FAKE, scale=0.1, out=FAKE, od=BF, sot=1024, soh=128, state=FAKE, slots=4, sss=8 * 128 * 128, ssh=128 * 128, read=FAKE, write=FAKE,
                H=8, KV=2, D=128)
    for call in (calls("vxa_linear_prompt", dict(rows, cu=FAKE, n=2, tokens=100, **rest, ws=FAKE, wsb=1 << 40, st=None)),
                 calls("vxa_linear_step", dict(rows, n=2, **rest, st=None))):
        for name in ("sqt", "skt", "svt", "sot"):
            assert call(**{name: 1 << 23}) == nx.VXA_ERR_UNSUPPORTED and call(**{name: -8}) == nx.VXA_ERR_UNSUPPORTED, name


def test_beam_select_refusals():
    call = calls("vxa_beam_select", dict(x=FAKE, stride=1000, dtype=BF, scores=FAKE, n=2, beams=4, vocab=1000, count=8, a=FAKE, b=FAKE, c=FAKE, ws=FAKE,
                                         wsb=1 << 30, st=None))
    assert call(n=0) == nx.VXA_OK
    for bad in (dict(n=-1), dict(beams=0), dict(vocab=0), dict(count=0), dict(dtype=7), dict(x=None), dict(scores=None), dict(a=None), dict(b=None), dict(c=None)):
        assert call(**bad) == nx.VXA_ERR_ARG, bad
    for bad in (dict(count=65), dict(beams=1025), dict(vocab=1 << 40), dict(vocab=1 << 30, beams=4), dict(beams=1000, vocab=200000), dict(n=1 << 40),
                dict(n=1 << 28, beams=16)):
        assert call(**bad) == nx.VXA_ERR_UNSUPPORTED, bad
    assert call(ws=None) == nx.VXA_ERR_WORKSPACE and call(ws=FAKE + 4) == nx.VXA_ERR_WORKSPACE and call(wsb=100) == nx.VXA_ERR_WORKSPACE


def test_page_refusals():
    copy = calls("vxa_pages_copy", dict(caches=view(), count=1, blocks=9, page=16, source=FAKE, target=FAKE, n=3, st=None))
    fork = calls("vxa_pages_fork", dict(caches=view(), count=1, bt=FAKE, sbt=4, cols=4, sl=FAKE, rows=2, parents=FAKE, many=3, refs=FAKE, blocks=9, page=16,
                                        out=2 * FAKE, sot=4, lens=2 * FAKE, out_refs=FAKE, missing=FAKE, ws=FAKE, wsb=1 << 20, st=None))
    resize = calls("vxa_pages_resize", dict(bt=FAKE, sbt=4, cols=4, sl=FAKE, new=FAKE, rows=2, refs=FAKE, blocks=9, page=16, out=FAKE, sot=4, out_refs=FAKE,
                                            missing=FAKE, ws=FAKE, wsb=1 << 20, st=None))
    keep = calls("vxa_pages_keep", dict(caches=view(), count=1, bt=FAKE, sbt=4, cols=4, sl=FAKE, cu=FAKE, keep=FAKE, n=2, blocks=9, page=16, lens=2 * FAKE, st=None))
    assert copy(n=0) == nx.VXA_OK and copy(count=0) == nx.VXA_OK and copy(blocks=0) == nx.VXA_OK and keep(n=0) == nx.VXA_OK
    for call in (copy, fork, keep):
        for bad in (dict(page=0), dict(blocks=-1), dict(count=-1), dict(caches=None), dict(caches=view(data=None)), dict(caches=view(heads=0)), dict(caches=view(row_bytes=0))):
            assert call(**bad) == nx.VXA_ERR_ARG, bad
        for bad in (dict(blocks=1 << 40), dict(caches=view(row_bytes=1 << 30))):
            assert call(**bad) == nx.VXA_ERR_UNSUPPORTED, bad
    for call, names in ((copy, ("source", "target")), (fork, ("bt", "sl", "parents", "refs", "out", "lens", "out_refs", "missing")),
                        (resize, ("bt", "sl", "new", "refs", "out", "out_refs", "missing")), (keep, ("bt", "sl", "cu", "keep", "lens"))):
        for name in names:
            assert call(**{name: None}) == nx.VXA_ERR_ARG, name
    for call in (fork, resize):
        for bad in (dict(rows=-1), dict(cols=-1), dict(page=0)):
            assert call(**bad) == nx.VXA_ERR_ARG, bad
        for bad in (dict(rows=8193), dict(cols=1 << 30), dict(blocks=1 << 29), dict(page=1 << 31)):
            assert call(**bad) == nx.VXA_ERR_UNSUPPORTED, bad
        assert call(ws=None) == nx.VXA_ERR_WORKSPACE and call(wsb=3) == nx.VXA_ERR_WORKSPACE
    assert fork(many=8193) == nx.VXA_ERR_UNSUPPORTED and fork(out=FAKE) == nx.VXA_ERR_ARG and fork(lens=FAKE) == nx.VXA_ERR_ARG
    assert resize(sot=8) == nx.VXA_ERR_ARG and keep(lens=FAKE) == nx.VXA_ERR_ARG and copy(n=1 << 30) == nx.VXA_ERR_UNSUPPORTED


def test_cpu_tensors_and_wrong_arguments_are_refused():
    q, g, cu, state = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(2), torch.tensor([0, 3]).int(), torch.zeros(3, 2, 64, 64)
    slots, table, lens = torch.zeros(3).int(), torch.zeros(1, 2).int(), torch.ones(1).int()
    cache = make_cache(2, 16, 1, 64, "cpu")
    refs = torch.zeros(2).int()
    for call in (lambda: linear_prompt(q, q, q, cu, g, 1.0, q), lambda: linear_step(q, q, q, g, 1.0, q, state, slots, slots),
                 lambda: beam_select(torch.zeros(2, 5), torch.zeros(2), 2, torch.zeros(1, 2), torch.zeros(1, 2).int(), torch.zeros(1, 2).long()),
                 lambda: copy_pages(cache, 16, lens, lens), lambda: fork_pages(cache, table, lens, lens, refs, 16, table.clone(), lens.clone()),
                 lambda: resize_pages(table, lens, lens, refs, 16), lambda: keep_drafted(cache, table, lens, cu, lens.long(), 16, lens.clone())):
        with pytest.raises(ValueError, match="GPU tensors"):
            call()
    for name, count in (("linear_prompt", 10), ("linear_step", 9), ("beam_select", 6), ("copy_pages", 4), ("fork_pages", 10), ("resize_pages", 8), ("keep_drafted", 7)):
        for n in (0, count - 1, count + 1):
            with pytest.raises(TypeError):
                getattr(nx.calls(), name)(*[None] * n)
        with pytest.raises(TypeError):
            getattr(nx.calls(), name)(*["not a tensor"] * count)


def test_linear_attention_statement():
    gen = torch.Generator().manual_seed(0)
    lens, H, KV, D = (1, 0, 40), 4, 2, 64
    q, k, v = (torch.randn(43, n, D, generator=gen).to(torch.bfloat16) for n in (H, KV, KV))
    g, pool = torch.tensor([0.0, -0.1, -2.0, -float("inf")]), torch.randn(5, H, D, D, generator=gen)
    state = pool.clone()
    out = linear_attention_torch(q, k, v, torch.tensor([0, 1, 1, 41]), g, 0.1, state, torch.tensor([3, -1, 4]), torch.tensor([1, 2, 4]))
    starts = torch.stack([pool[3], torch.zeros_like(pool[0]), pool[4]])
    want, ends = linear64(q, k, v, lens, g, 0.1, starts)
    rows, states = bounds(q, k, v, lens, g, 0.1, starts)
    assert ((out.double() - want).abs()[:41] <= rows[:41]).all() and (out[41:] == 0).all()
    assert ((state[[1, 2, 4]].double() - ends).abs() <= states).all() and torch.equal(state[[0, 3]], pool[[0, 3]])


def test_beam_statement():
    gen = torch.Generator().manual_seed(1)
    logits, scores = torch.randn(6, 11, generator=gen), torch.randn(6, generator=gen)
    logits[1, 3:] = -torch.inf
    scores[2] = -torch.inf
    logits[3:5] = logits[3]
    scores[4] = scores[3]
    best, parents, tokens = beam_select_torch(logits, scores, 3, 9)
    for r in range(2):
        every = []
        for b in range(3 * r, 3 * r + 3):
            total = math.log(sum(math.exp(x) for x in logits[b].tolist()))
            every += [(-(float(scores[b]) + x - total), b, t) for t, x in enumerate(logits[b].tolist()) if x != -math.inf and scores[b] != -torch.inf]
        every.sort()
        assert parents[r].tolist() == [x[1] for x in every[:9]] and tokens[r].tolist() == [x[2] for x in every[:9]]
        assert torch.allclose(best[r].double(), torch.tensor([-x[0] for x in every[:9]], dtype=torch.float64), rtol=0, atol=2e-6)
    assert beam_select_torch(logits[2:3], scores[2:3], 1, 2)[1].tolist() == [[-1, -1]]


@pytest.mark.parametrize("score", [float("nan"), float("inf")])
def test_beam_statement_of_a_score_without_tokens(score):
    logits = torch.full((2, 5), -torch.inf)
    logits[0] = 1.0
    best, parents, tokens = beam_select_torch(logits, torch.tensor([0.0, score]), 2, 3)
    assert best.isnan().all() and parents.eq(-1).all() and tokens.eq(-1).all()


def test_page_statements():
    ints = lambda x: torch.tensor(x, dtype=torch.int32)
    cache = torch.arange(8.0).view(8, 1, 1).repeat(1, 4, 1)
    table, refs = ints([[5, 2], [5, 3]]), ints([0, 0, 1, 1, 0, 2, 0, 0])
    new, lens, counts, missing = fork_pages_torch([cache], table, ints([6, 8]), ints([0, 0, 1, -1]), refs, 4)
    assert new.tolist() == [[5, 2], [5, 0], [5, 3], [-1, -1]] and lens.tolist() == [6, 6, 8, 0] and missing == 0
    assert counts.tolist() == [1, 0, 1, 1, 0, 3, 0, 0] and cache[0, 0, 0] == 2
    grown, counts, missing = resize_pages_torch(new[:, :2], lens, ints([4, 9, 0, 8]), counts, 4)
    assert grown.tolist() == [[5, -1], [5, 0], [-1, -1], [1, 4]] and counts.tolist() == [1, 1, 0, 0, 1, 2, 0, 0] and missing == 0
    rows = torch.arange(16.0).view(4, 4, 1)
    out = keep_drafted_torch([rows], ints([[2, 0]]), ints([7]), ints([0, 5]), torch.tensor([0b10101]), 4)
    assert out.tolist() == [5] and rows[2, :, 0].tolist() == [8, 9, 10, 0] and rows[0, :, 0].tolist() == [2, 1, 2, 3]
