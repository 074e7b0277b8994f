"""Calls at the edges of what the operators for many tokens take (vllm_expert_cache/ops.py and their C
entry points), checked without a GPU: none of them launches a kernel."""
from __future__ import annotations

import ctypes

import pytest
import torch

from vllm_expert_cache import _lib, ops

BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


@pytest.fixture
def no_kernels(monkeypatch):
    """Lets CPU tensors past the device check, and calls that every check lets through end without
    a device."""
    calls = []
    monkeypatch.setattr(ops, "_on_gpu", lambda *t: t[0].device)
    monkeypatch.setattr(ops, "_on_device", lambda device, call, *args: calls.append(args) or 0)
    return calls


# ---- no tokens ----------------------------------------------------------------------------

# few and many outputs, of lengths that are cut where tokens are few (6017 on) and that aren't
@pytest.mark.parametrize("H", [16, 6000, 6017, 131056])
@pytest.mark.parametrize("O", [1, 8191, 8192, 2 ** 24])
def test_a_projection_of_no_tokens(lib, no_kernels, O, H):
    size = ctypes.c_long(-5)
    l = _lib.Linear(O, H, -(-H // 16) * 16, 16, 16, None)
    for kind in (1, 2, 3):
        size.value = -5
        assert lib.expert_cache_linear8_workspace(ctypes.addressof(l), kind, 0,
                                                  ctypes.addressof(size)) == 0
        assert size.value == 0
    if O == 8192 and H < 10000:
        lin = ops.Linear8(torch.zeros((O, H), dtype=I8), torch.ones(O))
        assert lin(torch.empty((0, H), dtype=BF16)).shape == (0, O)
        assert lin(torch.empty((0, H), dtype=I8), torch.empty(0)).shape == (0, O)


def test_a_layer_of_no_tokens(lib):
    size = ctypes.c_long(-5)
    for S, H, I in ((1, 16, 16), (1024, 131056, 16)):
        e = _lib.Experts(S, H, I, 1, 3, 16, 16, 16, 16)
        assert lib.expert_cache_moe8_workspace(ctypes.addressof(e), 0, 8, ctypes.addressof(size)) == 0
