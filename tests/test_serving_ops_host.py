"""CPU checks of prompt attention, the 8-bit cache and tree decoding: what the entry points refuse, before anything is
launched, and the torch statements against float64."""
import pytest
import torch

from attention64 import attend64, check
from vllm_exact import _native as nx
from vllm_exact.int8_cache import dequantize_torch, make_cache, quantize_torch, read_cache, write_cache
from vllm_exact.prompt_attn import prompt_attention, prompt_attention_torch
from vllm_exact.tree_attn import tree_decode, tree_decode_torch

FAKE = 1 << 20  # never dereferenced: validation fails first
BF, F32, F16 = nx.VXA_BF16, nx.VXA_F32, nx.VXA_F16


def calls(fn, defaults):
    return lambda **over: getattr(nx.lib(), fn)(*dict(defaults, **over).values())


def test_prompt_attention_refusals():
    call = calls("vxa_prompt_attention", dict(
        q=FAKE, sqt=1024, sqh=128, k=FAKE, skt=256, skh=128, v=FAKE, svt=256, svh=128, dtype=BF, cu=FAKE, n=2, tokens=100,
        scale=0.1, out=FAKE, od=BF, sot=1024, soh=128, H=8, KV=2, D=128, st=None))
    assert call(n=0) == nx.VXA_OK and call(tokens=0, q=None) == nx.VXA_OK
    for bad in (dict(n=-1), dict(tokens=-1), dict(H=0), dict(KV=0), dict(D=0), dict(H=7), dict(dtype=F32), dict(dtype=9),
                dict(od=9), dict(q=None), dict(k=None), dict(v=None), dict(cu=None), dict(out=None)):
        assert call(**bad) == nx.VXA_ERR_ARG, bad
    for bad in (dict(D=96), dict(q=FAKE + 2), dict(k=FAKE + 8), dict(v=FAKE + 8), dict(sqt=1020), dict(skh=4), dict(svt=2),
                dict(tokens=1 << 40), dict(n=1 << 40), dict(tokens=1 << 30, H=1 << 16, KV=1)):
        assert call(**bad) == nx.VXA_ERR_UNSUPPORTED, bad


CACHE = dict(kc=FAKE, skcb=8192, skcp=256, skch=4096, vc=FAKE, svcb=8192, svcp=256, svch=4096, ks=FAKE, sksb=64, sksp=2,
             sksh=32, vs=FAKE, svsb=64, svsp=2, svsh=32)


def test_int8_cache_refusals():
    write = calls("vxa_int8_cache_write", dict(
        k=FAKE, skt=256, skh=128, v=FAKE, svt=256, svh=128, dtype=BF, tokens=10, KV=2, D=128, **CACHE, blocks=8, page=16,
        slots=FAKE, st=None))
    read = calls("vxa_int8_cache_read", dict(
        **CACHE, blocks=8, page=16, bt=FAKE, sbt=4, cols=4, cu=FAKE, first=None, n=2, tokens=10, KV=2, D=128, k=FAKE, skt=256,
        skh=128, v=FAKE, svt=256, svh=128, dtype=BF, st=None))
    assert write(tokens=0) == nx.VXA_OK and write(blocks=0) == nx.VXA_OK
    assert read(tokens=0) == nx.VXA_OK and read(n=0) == nx.VXA_OK
    for call in (write, read):
        for bad in (dict(tokens=-1), dict(KV=0), dict(D=0), dict(blocks=-1), dict(page=0), dict(dtype=7), dict(k=None), dict(v=None),
                    dict(kc=None), dict(vc=None), dict(ks=None), dict(vs=None)):
            assert call(**bad) == nx.VXA_ERR_ARG, bad
        for bad in (dict(D=80), dict(kc=FAKE + 8), dict(vc=FAKE + 4), dict(skcb=8200), dict(svcp=8), dict(skch=4),
                    dict(blocks=1 << 28), dict(KV=1 << 30)):
            assert call(**bad) == nx.VXA_ERR_UNSUPPORTED, bad
    assert write(slots=None) == nx.VXA_ERR_ARG and read(bt=None) == nx.VXA_ERR_ARG and read(cu=None) == nx.VXA_ERR_ARG
    assert read(n=-1) == nx.VXA_ERR_ARG and read(cols=-1) == nx.VXA_ERR_ARG
    for bad in (dict(cols=1 << 28), dict(k=FAKE + 2), dict(svt=100), dict(dtype=F32, skt=2)):
        assert read(**bad) == nx.VXA_ERR_UNSUPPORTED, bad


def test_tree_decode_refusals():
    call = calls("vxa_tree_decode", dict(
        q=FAKE, sqt=1024, sqh=128, qd=BF, **CACHE, blocks=8, page=16, bt=FAKE, sbt=40, cols=40, sl=FAKE, qsl=FAKE, mask=None,
        scale=0.1, out=FAKE, od=BF, sot=1024, soh=128, n=2, tokens=10, H=8, KV=2, D=128, nodes=5, longest=500, ws=None, wsb=0,
        st=None))
    assert call(n=0) == nx.VXA_OK and call(tokens=0) == nx.VXA_OK and call(nodes=0) == nx.VXA_OK
    for bad in (dict(n=-1), dict(tokens=-1), dict(H=0), dict(KV=0), dict(D=0), dict(H=7), dict(qd=F32), dict(od=5), dict(page=0),
                dict(blocks=-1), dict(blocks=0), dict(cols=-1), dict(nodes=-1), dict(longest=-1), dict(ks=None), dict(vs=None),
                dict(q=None), dict(kc=None), dict(vc=None), dict(bt=None), dict(sl=None), dict(qsl=None), dict(out=None)):
        assert call(**bad) == nx.VXA_ERR_ARG, bad
    for bad in (dict(D=96), dict(nodes=65), dict(q=FAKE + 8), dict(kc=FAKE + 8), dict(sqt=1020), dict(skcb=8), dict(svch=8),
                dict(skcp=12, ks=None, vs=None), dict(longest=1 << 31), dict(tokens=1 << 40), dict(n=1 << 40)):
        assert call(**bad) == nx.VXA_ERR_UNSUPPORTED, bad
    assert call(longest=600) == nx.VXA_ERR_WORKSPACE
    assert call(longest=600, ws=FAKE, wsb=nx.tree_workspace(10, 8, 128, 600) - 1) == nx.VXA_ERR_WORKSPACE
    assert nx.tree_workspace(10, 8, 128, 512) == 0 and nx.tree_workspace(10, 8, 128, 513) == 10 * 8 * 2 * 130 * 4
    with pytest.raises(ValueError):
        nx.tree_workspace(-1, 8, 128, 512)


def test_cpu_tensors_are_refused():
    q, k, cu = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, 1, 64, dtype=torch.bfloat16), torch.tensor([0, 3]).int()
    cache = make_cache(2, 16, 1, 64, "cpu")
    with pytest.raises(ValueError, match="prompt_attention_torch"):
        prompt_attention(q, k, k, cu, 1.0, q.clone())
    with pytest.raises(ValueError, match="quantize_torch"):
        write_cache(k, k, *cache, torch.arange(3))
    with pytest.raises(ValueError, match="dequantize_torch"):
        read_cache(*cache, torch.zeros(1, 1).int(), cu, k, k.clone())
    with pytest.raises(ValueError, match="tree_decode_torch"):
        tree_decode(q, *cache[:2], torch.zeros(1, 1).int(), torch.tensor([3]).int(), cu, None, 1.0, q.clone(), 3, 16,
                    key_scale=cache[2], value_scale=cache[3])


def test_cache_layout():
    k, v, ks, vs = make_cache(5, 16, 3, 64, "cpu")
    assert k.shape == v.shape == (5, 16, 3, 64) and ks.shape == vs.shape == (5, 16, 3)
    assert k.stride() == (3 * 16 * 128, 128, 16 * 128, 1) and v.storage_offset() == 64 and vs.storage_offset() == 1


def test_quantisation_statement():
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(50, 3, 64, generator=g) * 100).to(torch.bfloat16)
    x[0, 0] = 0
    q, s = quantize_torch(x)
    top = x.double().abs().amax(-1)
    want = torch.round(127 * x.double() / torch.where(top > 0, top, 1)[..., None])
    assert torch.equal(q.double(), want) and ((s.double() - top / 127).abs() <= top / 127 * 2.0 ** -24).all()
    assert ((dequantize_torch(q, s).double() - x.double()).abs() <= (top / 254 * 1.001)[..., None]).all()
    x[1, 1, 5] = float("nan")
    q, s = quantize_torch(x)
    assert (q[1, 1] == 0).all() and torch.isnan(s[1, 1]) and torch.isfinite(s[1, 0])


@pytest.mark.parametrize("lens", [(1,), (0, 5, 33), (70, 2)])
def test_prompt_statement(lens):
    g = torch.Generator().manual_seed(1)
    T = sum(lens) + 2
    q, k, v = (torch.randn(T, n, 64, generator=g).to(torch.bfloat16) for n in (4, 2, 2))
    cu = torch.tensor([0] + list(lens)).cumsum(0).int()
    out = prompt_attention_torch(q, k, v, cu, 0.125)
    for lo, hi in zip(cu.tolist(), cu.tolist()[1:]):
        for h in range(4):
            if hi > lo:
                want, bound = attend64(q[lo:hi, h], k[lo:hi, h // 2], v[lo:hi, h // 2],
                                       torch.ones(hi - lo, hi - lo, dtype=torch.bool).tril(), 0.125, 0.0, 0.0)
                check(out[lo:hi, h], want, bound)
    assert (out[-2:] == 0).all()


@pytest.mark.parametrize("int8", [True, False])
def test_tree_statement(int8):
    g = torch.Generator().manual_seed(2)
    pool = torch.randn(9, 16, 2, 64, generator=g).to(torch.bfloat16), torch.randn(9, 16, 2, 64, generator=g).to(torch.bfloat16)
    scales = (None, None)
    keys, vals = pool
    if int8:
        (kq, ks), (vq, vs) = map(quantize_torch, pool)
        pool, scales = (kq, vq), (ks, vs)
        keys, vals = dequantize_torch(kq, ks), dequantize_torch(vq, vs)
    q = torch.randn(6, 4, 64, generator=g).to(torch.bfloat16)
    bt, sl, qsl = torch.tensor([[3, 1, 7], [2, 8, 0]]).int(), torch.tensor([4, 40]).int(), torch.tensor([0, 4, 6]).int()
    mask = torch.tensor([1, 0, 0b101, 0b1010, 0b01, 0b10])
    out = tree_decode_torch(q, *pool, bt, sl, qsl, mask, 0.125, *scales)
    assert (out[1] == 0).all()
    for b, (lo, hi, n) in enumerate(((0, 4, 4), (4, 6, 40))):
        rows = [(int(bt[b, t // 16]), t % 16) for t in range(n)]
        kk, vv = (torch.stack([x[r] for r in rows]) for x in (keys, vals))
        seen = torch.ones(hi - lo, n, dtype=torch.bool)
        for i in range(hi - lo):
            for j in range(hi - lo):
                seen[i, n - (hi - lo) + j] = bool(int(mask[lo + i]) >> j & 1)
        for h in range(4):
            check(out[lo:hi, h], *attend64(q[lo:hi, h], kk[:, h // 2], vv[:, h // 2], seen, 0.125, 0.0, 0.0))
