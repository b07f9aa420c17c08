"""GPU checks of the serving operators' calls on tensors whose memory the module may not touch."""
import pytest
import torch

from vllm_exact.int8_cache import make_cache, read_cache, write_cache
from vllm_exact.prompt_attn import prompt_attention
from vllm_exact.tree_attn import tree_decode

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_vmap_is_an_error():
    """The tensors that torch.vmap passes have no memory of their own."""
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    q, k, cu, slots = bf(2, 3, 2, 64), bf(2, 3, 1, 64), ints(0, 3), torch.arange(3, device=DEV)
    cache = make_cache(2, 16, 1, 64, DEV)
    bt, sl = ints(0, 1).view(1, 2), ints(3)
    for call, over in ((lambda x: prompt_attention(x, k[0], k[0], cu, 1.0, q[0].clone()), q),
                       (lambda x: write_cache(x, x, *cache, slots), k),
                       (lambda x: read_cache(*cache, bt, cu, x, x), k),
                       (lambda x: tree_decode(x, *cache[:2], bt, sl, cu, None, 1.0, q[0].clone(), 3, 16, *cache[2:]), q)):
        for _ in range(2):
            with pytest.raises(RuntimeError):
                torch.vmap(call)(over)
    out = torch.empty(3, 2, 64, device=DEV)
    assert torch.equal(prompt_attention(q[0], k[0], k[0], cu, 1.0, out), torch.zeros_like(out))


def test_a_workspace_that_does_not_fit():
    """Lengths up to 2^30 of many nodes: more than any memory. torch's own exception, as from a tensor of that size."""
    n, nodes, H, D = 300, 64, 64, 64
    q = torch.zeros(n * nodes, H, D, dtype=torch.bfloat16, device=DEV)
    cache = make_cache(2, 16, H, D, DEV)
    bt, sl = torch.zeros(n, 4, dtype=torch.int32, device=DEV), torch.full((n,), nodes, dtype=torch.int32, device=DEV)
    qsl, out = torch.arange(0, n * nodes + 1, nodes, dtype=torch.int32, device=DEV), torch.empty_like(q)
    call = lambda longest: tree_decode(q, *cache[:2], bt, sl, qsl, None, 1.0, out, nodes, longest, *cache[2:])
    with pytest.raises(torch.OutOfMemoryError):
        call(1 << 30)
    call(64)
    assert (out == 0).all()
