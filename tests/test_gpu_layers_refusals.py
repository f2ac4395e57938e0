"""Refusals of the layers that come before memory is taken."""

import pytest
import torch

import fuselse_amd
from fuselse_amd import ext, layers
from test_gpu_followed_calls import _None

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("experts", [1025, 1 << 40, 1 << 62, 1 << 70])
def test_too_many_experts(cuda, monkeypatch, experts, python):
    """Refused by their number, not by the allocation of their counts."""
    if python:
        monkeypatch.setattr(layers, "_common", _None())
    index = torch.zeros(3, 2, dtype=torch.int64, device=cuda)
    with pytest.raises(RuntimeError, match="1024 experts"):
        fuselse_amd.expert_order(index, experts)
    with pytest.raises(RuntimeError, match="1024 experts"):
        ext.expert_order(index, experts)
