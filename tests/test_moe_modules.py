"""The MoE modules as parts of a model: casts, copies and hooks (on the CPU, with the launches left out; on the GPU their
results)."""

import copy
import io

import pytest
import torch

from sgl_asap_amd.moe import linear as L
from sgl_asap_amd.moe import topk as T
from sgl_asap_amd.moe.shared import Fp8SharedExpertMLP


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


def test_a_correction_bias_of_another_type_can_be_cast_to_the_one_it_needs():
    topk = T.TopK(2, correction_bias=torch.ones(16, dtype=torch.bfloat16))
    assert topk.float().correction_bias.dtype == torch.float32
    assert topk.bfloat16().correction_bias.dtype == torch.float32


@pytest.fixture
def no_launches(monkeypatch):
    monkeypatch.setattr(L, "need_gpu", lambda *a: None)
    monkeypatch.setattr(L, "launch", lambda *a: None)


def addresses(layer):
    w = layer._weights_ref._obj
    return w.n_out, w.k_in, w.image, w.scales


def copies(layer):
    """A deep copy, and one through a file."""
    file = io.BytesIO()
    torch.save(layer, file)
    file.seek(0)
    return copy.deepcopy(layer), torch.load(file, weights_only=False)


def test_copies_of_a_layer_hold_weights_of_their_own(no_launches):
    layer = L.Fp8BlockLinear(torch.zeros(20, 130, dtype=torch.uint8), torch.rand(1, 2))
    layer.image.random_(0, 255)
    before = addresses(layer)
    for other in copies(layer):
        assert addresses(other) == (20, 130, other.image.data_ptr(), other.scales.data_ptr())
        assert other.image.data_ptr() != layer.image.data_ptr() and other.scales.data_ptr() != layer.scales.data_ptr()
        assert torch.equal(other.image, layer.image) and torch.equal(other.scales, layer.scales)
        assert (other.out_features, other.in_features) == (20, 130)
    assert addresses(layer) == before == (20, 130, layer.image.data_ptr(), layer.scales.data_ptr())
    model = copy.deepcopy(torch.nn.Sequential(layer))
    assert addresses(model[0])[2] == model[0].image.data_ptr()


@pytest.mark.parametrize("inter", [1, 12, 131])
def test_an_mlp_of_any_intermediate_size_is_its_two_layers(no_launches, monkeypatch, inter):
    """As wide as its layers are, and calls them as modules, so that hooks on either run."""
    calls, seen = [], []
    monkeypatch.setattr(L, "launch", lambda name, *a: calls.append(name))
    ceil = lambda a: -(-a // 128)
    codes = lambda *shape: torch.zeros(*shape, dtype=torch.uint8)
    mlp = Fp8SharedExpertMLP(codes(2 * inter, 40), torch.zeros(ceil(2 * inter), 1), codes(40, inter), torch.zeros(1, ceil(inter)))
    calls.clear()
    for name, layer in mlp.named_children():
        layer.register_forward_pre_hook(lambda m, args, name=name: seen.append((name, tuple(args[0].shape))))
        layer.register_forward_hook(lambda m, args, y, name=name: seen.append((name, tuple(y.shape))))
    assert mlp(torch.zeros(3, 40, dtype=torch.bfloat16)).shape == (3, 40)
    assert calls == ["afd_linear", "afd_linear_silu_mul"]
    assert seen == [("gate_up", (3, 40)), ("gate_up", (3, 2 * inter)), ("down", (3, 2 * inter)), ("down", (3, 40))]
    with pytest.raises(TypeError):
        mlp.down(torch.zeros(3, 2 * inter, dtype=torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,inter", [(384, 131), (130, 12), (256, 1)])
def test_odd_mlps_and_their_copies_give_the_same_bits(hidden, inter):
    """An intermediate size that the activation's own kernel does not take, against the layers padded to one that it does."""
    from gpu_util import dev, say
    from sgl_asap_amd.moe.shared import silu_mul

    g = torch.Generator().manual_seed(inter)
    ceil = lambda a: -(-a // 128)
    e4m3 = lambda *shape: (torch.randn(*shape, generator=g) * 50).clamp(-448, 448).to(torch.float8_e4m3fn)
    w_gu, w_d = e4m3(2 * inter, hidden), e4m3(hidden, inter)
    s_gu = torch.rand(ceil(2 * inter), ceil(hidden), generator=g) * 2e-3
    s_d = torch.rand(ceil(hidden), ceil(inter), generator=g) * 2e-3
    mlp = Fp8SharedExpertMLP(*(t.to(dev()) for t in (w_gu, s_gu, w_d, s_d)))
    pad = -(-inter // 8) * 8
    others = (*copies(mlp), Fp8SharedExpertMLP(w_gu, s_gu, w_d, s_d, device=dev()))
    for n in (1, 7, 40, 150):
        say(f"odd MLP n={n} hidden={hidden} inter={inter}")
        x = torch.randn(n, hidden, generator=g).to(torch.bfloat16).to(dev())
        gate_up = L.Fp8BlockLinear(w_gu.to(dev()), s_gu.to(dev()))(x)
        wide = torch.zeros(n, 2, pad, dtype=torch.bfloat16, device=dev())
        wide[:, :, :inter] = gate_up.view(n, 2, inter)
        h = silu_mul(wide.view(n, 2 * pad))[:, :inter]
        want = L.Fp8BlockLinear(w_d.to(dev()), s_d.to(dev()))(h)
        assert torch.isfinite(want).all() and (want != 0).any()
        for m in (mlp, *others):
            assert torch.equal(m(x), want)
