"""A block's norms as a module, on the host."""

import torch

from sgl_asap_amd.moe.norm import BlockNorms


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
