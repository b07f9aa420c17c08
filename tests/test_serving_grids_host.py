"""CPU checks that a serving operator refuses what needs more threads than one launch has, before anything is launched."""
import pytest

from vllm_exact import _native as nx

import test_serving_ops_host as ops

FAKE, BF = ops.FAKE, ops.BF


def test_prompt_attention():
    call = ops.calls("vxa_prompt_attention", dict(
        q=FAKE, sqt=4096, sqh=128, k=FAKE, skt=1024, skh=128, v=FAKE, svt=1024, svh=128, dtype=BF, cu=FAKE, n=2, tokens=100,
        scale=0.1, out=FAKE, od=BF, sot=4096, soh=128, H=32, KV=8, D=128, st=None))
    assert call(tokens=1 << 28) == nx.VXA_ERR_UNSUPPORTED  # 2^23 tiles of 32 rows, 8 groups of heads, 256 threads


def test_int8_cache():
    write = ops.calls("vxa_int8_cache_write", dict(
        k=FAKE, skt=2048, skh=256, v=FAKE, svt=2048, svh=256, dtype=BF, tokens=1 << 24, KV=8, D=256, **ops.CACHE, blocks=8, page=16,
        slots=FAKE, st=None))
    assert write() == nx.VXA_ERR_UNSUPPORTED  # a workgroup of 256 for each token


@pytest.mark.parametrize("over", [dict(n=1 << 12, longest=1 << 20, nodes=1), dict(n=(1 << 31) - 1, longest=1 << 30, nodes=64, H=1 << 16, KV=1 << 16),
                                  dict(n=1 << 12, longest=1 << 20, nodes=64)])
def test_tree_decode(over):
    call = ops.calls("vxa_tree_decode", dict(
        q=FAKE, sqt=1024, sqh=128, qd=BF, **ops.CACHE, blocks=8, page=16, bt=FAKE, sbt=40, cols=40, sl=FAKE, qsl=FAKE, mask=None,
        scale=0.1, out=FAKE, od=BF, sot=1024, soh=128, n=2, tokens=10, H=32, KV=8, D=128, nodes=5, longest=500, ws=FAKE, wsb=(1 << 63) - 1,
        st=None))
    assert call(**over) == nx.VXA_ERR_UNSUPPORTED
