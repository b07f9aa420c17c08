"""CPU checks that tensors without memory are an error of the calls on tensors, raised with the interpreter lock held: their
pointers are asked for before anything that needs a GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from vllm_exact.int8_cache import make_cache, read_cache, write_cache
from vllm_exact.prompt_attn import prompt_attention
from vllm_exact.tree_attn import tree_decode


def test_tensors_without_memory_are_an_error():
    """The tensors that torch.vmap passes, of a GPU that need not be there."""
    with FakeTensorMode():
        bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
        ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
        q, k, cu, slots = bf(2, 3, 2, 64), bf(2, 3, 1, 64), ints(2, 2), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
        cache, table, lens = make_cache(2, 16, 1, 64, "cuda"), ints(2, 1, 1), ints(2, 1)
        for call, over in ((lambda q, k, cu: prompt_attention(q, k, k, cu, 1.0, q), (q, k, cu)),
                           (lambda k, slots: write_cache(k, k, *cache, slots), (k, slots)),
                           (lambda table, cu, k, first: read_cache(*cache, table, cu, k, k, first=first), (table, cu, k, lens)),
                           (lambda q, table, lens, cu, mask: tree_decode(q, *cache[:2], table, lens, cu, mask, 1.0, q, 3, 16, *cache[2:]),
                            (q, table, lens, cu, slots))):
            for _ in range(2):  # the second call: the first has left the interpreter as it was
                with pytest.raises(RuntimeError, match="doesn't have storage"):
                    torch.vmap(call)(*over)
