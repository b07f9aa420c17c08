"""CPU checks of the serving operators' calls on tensors (csrc/tensor_calls.cpp): what is refused before a GPU is needed, and
that no C++ exception passes the module."""
import ctypes

import pytest
import torch

from vllm_exact import _native as nx
from vllm_exact.int8_cache import make_cache, read_cache, write_cache
from vllm_exact.prompt_attn import prompt_attention
from vllm_exact.tree_attn import tree_decode


def test_the_module_is_bound_to_the_loaded_library():
    assert nx.calls() is nx.calls()
    with pytest.raises(TypeError):
        nx.calls().bind(1)
    with pytest.raises((TypeError, ValueError)):
        nx.calls().bind(0, 0, 0, 0, 0)
    address = ctypes.cast(nx.lib().vxa_tree_decode, ctypes.c_void_p).value
    with pytest.raises(TypeError):
        nx.calls().bind(address, address, address, address, "x")


def test_wrong_counts_and_kinds_of_arguments():
    calls = nx.calls()
    for name, count in (("prompt_attention", 6), ("write_cache", 7), ("read_cache", 9), ("tree_decode", 13)):
        for n in (0, count - 1, count + 1):
            with pytest.raises(TypeError):
                getattr(calls, name)(*[None] * n)
        with pytest.raises(TypeError):
            getattr(calls, name)(*["not a tensor"] * count)


def test_tensors_without_gpu_memory_are_refused():
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    k, cu = q[:, :1], torch.tensor([0, 3]).int()
    cache = make_cache(2, 16, 1, 64, "cpu")
    table, lens = torch.zeros(1, 1).int(), torch.tensor([3]).int()
    for where in ("cpu", "meta"):
        move = lambda *ts: [t.to(where) for t in ts]
        with pytest.raises(ValueError, match="GPU tensors"):
            prompt_attention(*move(q, k, k, cu), 1.0, *move(q))
        with pytest.raises(ValueError, match="GPU tensors"):
            write_cache(*move(k, k, *cache, torch.arange(3)))
        with pytest.raises(ValueError, match="GPU tensors"):
            read_cache(*move(*cache, table, cu, k, k), first=lens.to(where))
        with pytest.raises(ValueError, match="GPU tensors"):
            tree_decode(*move(q, *cache[:2], table, lens, cu), None, 1.0, *move(q), 3, 16)
    with pytest.raises((TypeError, AttributeError)):
        tree_decode(None, *cache[:2], table, lens, cu, None, 1.0, q, 3, 16)
