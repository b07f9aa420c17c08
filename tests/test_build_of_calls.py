"""CPU checks of when the module of the calls on tensors is built: again where torch has changed, and not where there is no torch,
which the C entry points do not need."""
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

PACKAGE = Path(__file__).resolve().parents[1] / "vllm-exact_amd"
pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="no make")


def planned(*args):
    return subprocess.run(["make", "-n", "-C", str(PACKAGE), *args], check=True, capture_output=True, text=True).stdout


def test_built_again_with_another_torch():
    assert "csrc/tensor_calls.cpp" in planned("-W", str(Path(torch.__file__).parent / "version.py"))


def test_the_library_alone_without_torch():
    plan = planned("-B", "TORCH=")
    assert "libvllm_exact_amd.so" in plan and "csrc/tensor_calls.cpp" not in plan
    assert "csrc/tensor_calls.cpp" in planned("-B")
