"""Dense layers of weights that come as parameters: the layer keeps copies of its own."""

import copy
import pickle

import pytest
import torch

from sgl_asap_amd.moe import linear as L


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_scales_given_as_a_parameter(monkeypatch, kind):
    monkeypatch.setattr(L, "need_gpu", lambda *a: None)
    monkeypatch.setattr(L, "launch", lambda *a: None)
    if kind == "int8":
        scales = torch.nn.Parameter(torch.ones(24, 1))
        layer = L.Int8Linear(torch.zeros(24, 16, dtype=torch.int8), scales)
    else:
        scales = torch.nn.Parameter(torch.ones(1, 1))
        layer = L.Fp8BlockLinear(torch.zeros(24, 16, dtype=torch.uint8), scales)
    assert not layer.scales.requires_grad and layer.scales.is_leaf
    assert layer.scales.data_ptr() != scales.data_ptr() and not list(layer.parameters())
    for other in (copy.deepcopy(layer), pickle.loads(pickle.dumps(layer))):
        assert torch.equal(other.scales.view(-1), scales.detach().view(-1))
        assert other._weights.scales == other.scales.data_ptr()
