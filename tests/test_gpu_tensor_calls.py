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
