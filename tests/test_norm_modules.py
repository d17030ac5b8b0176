"""A block's norms as a module, and a single token's gate, on the host."""

import pytest
import torch

from sgl_asap_amd.moe.norm import BlockNorms, residual_norm


def test_given_parameters_are_the_module_s():
    """What an optimizer holds is what gets the gradients."""
    w, p, g = (torch.nn.Parameter(torch.ones(8)) for _ in range(3))
    g.requires_grad_(False)
    norms = BlockNorms(w, p, g)
    assert norms.input_weight is w and norms.post_weight is p and norms.gate is g
    assert [k for k, _ in norms.named_parameters()] == ["input_weight", "post_weight", "gate"]
    assert not norms.gate.requires_grad
    plain = BlockNorms(torch.ones(8), torch.ones(8))
    assert all(isinstance(t, torch.nn.Parameter) and t.requires_grad for t in plain.parameters())
    assert plain.gate is None


def test_a_gate_of_one_token():
    """[1] beside y [hidden] is a gate per token: its shape passes."""
    y = torch.zeros(8)
    for gate in (torch.ones(1), torch.ones(8)):
        with pytest.raises(ValueError, match="GPU"):
            residual_norm(y, y, gate=gate)
    for gate in (torch.ones(2), torch.ones(0), torch.ones(9)):
        with pytest.raises(ValueError, match="gate must be"):
            residual_norm(y, y, gate=gate)
