"""CPU check that errors of torch inside the calls on tensors are torch's own Python exceptions."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from vllm_exact.prompt_attn import prompt_attention


def test_errors_of_torch_are_its_python_exceptions():
    """Their messages are one statement, without a listing of C++ frames."""
    with FakeTensorMode():
        q, cu = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        with pytest.raises(RuntimeError) as e:
            torch.vmap(lambda q: prompt_attention(q, q, q, cu, 1.0, q))(q)
    assert "storage" in str(e.value) and "frame #" not in str(e.value)
