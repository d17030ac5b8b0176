"""The MoE modules as parts of a model: casts, copies and hooks (on the CPU, with the launches left out)."""

import copy
import pickle

import pytest
import torch

from sgl_asap_amd.moe import topk as T


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.bfloat16(),
                                  lambda m: m.to("cpu", torch.bfloat16)])
def test_a_cast_of_the_model_leaves_the_correction_bias(cast):
    """Its small differences decide between experts; the entry point takes it in fp32 alone."""
    bias = torch.randn(16) * 1e-3
    model = torch.nn.Sequential(torch.nn.Linear(4, 16), T.TopK(2, correction_bias=bias.clone()), T.TopK(2))
    cast(model)
    assert model[0].weight.dtype != torch.float32
    assert model[1].correction_bias.dtype == torch.float32 and torch.equal(model[1].correction_bias, bias)
    assert model[2].correction_bias is None
    assert torch.equal(model.state_dict()["1.correction_bias"], bias)


def test_the_correction_bias_moves_with_the_model():
    topk = T.TopK(2, correction_bias=torch.zeros(16))
    for move in (lambda m: m.to("meta"), lambda m: m.to("meta", torch.bfloat16)):
        there = move(copy.deepcopy(topk)).correction_bias
        assert there.device.type == "meta" and there.dtype == torch.float32
