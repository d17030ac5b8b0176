"""GPU: a block's norms at the ends of their range: sums of squares past fp32, workgroups past 2^20, rows of any
alignment, a gate of one value for a single token."""

import pytest
import torch

from error_bounds import Bounded
from gpu_util import dev, say
from sgl_asap_amd.moe.norm import residual_norm, rms_norm
from test_gpu_norm import EPS, backward, make

pytestmark = pytest.mark.gpu


def unit(v, eps):
    r = (v * v).mean().over_root(eps)
    return v * r, r


def large(n, hidden, size, seed):
    """Rows of values up to about 4 ``size``, one of them ordinary."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, hidden, generator=g) * size).clamp(-4 * size, 4 * size)
    x[1] = torch.randn(hidden, generator=g)
    return x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hidden", [100, 512, 1024, 4096, 5001, 16384])
@pytest.mark.parametrize("size", [1e18, 8e18, 1e30, 2e37])
def test_rows_whose_squares_add_up_past_fp32(dtype, hidden, size):
    n, eps = 5, 1e-6
    x = large(n, hidden, size, hidden).to(dtype)
    g = torch.Generator().manual_seed(1)
    w = 1 + 0.3 * torch.randn(hidden, generator=g)
    dn = torch.randn(n, hidden, generator=g).to(dtype)
    say(f"large rows {dtype} hidden={hidden} size={size}")
    xd, wd = x.to(dev()).requires_grad_(), w.to(dev()).requires_grad_()
    out = rms_norm(xd, wd, eps=eps)
    dx, dw = torch.autograd.grad(out, (xd, wd), dn.to(dev()))
    v, r = unit(Bounded(x), eps)
    assert (v * Bounded(w)).held(dtype).holds(out.detach())
    assert float(out.detach()[0].abs().max()) > 1
    q = Bounded(dn) * Bounded(w)
    d = r * (q - v * (q * v).mean())
    # a gradient below the floats' least normal number is rounded to its steps of 2^-149, some times over
    d.e += 8 * 2.0**-149
    assert d.held(dtype).holds(dx)
    assert (Bounded(dn) * v).sum(0).held(torch.float32).holds(dw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hidden", [384, 4096, 9000])
def test_large_outputs_and_residuals(dtype, hidden):
    """Both norms' sums past fp32, one after the other and each alone."""
    n, eps = 5, 1e-5
    g = torch.Generator().manual_seed(hidden)
    w_post, w_next = (1 + 0.3 * torch.randn(hidden, generator=g) for _ in range(2))
    say(f"large blocks {dtype} hidden={hidden}")
    for size_y, size_r in ((1e19, 1e19), (1e19, 1.0), (1.0, 1e19), (1e30, 1e25)):
        y, res = large(n, hidden, size_y, 1).to(dtype), large(n, hidden, size_r, 2).to(dtype)
        h, normed = residual_norm(y.to(dev()), res.to(dev()), post_weight=w_post.to(dev()), next_weight=w_next.to(dev()), eps=eps)
        want = Bounded(res) + unit(Bounded(y), eps)[0] * Bounded(w_post)
        assert want.held(dtype).holds(h)
        assert (unit(want, eps)[0] * Bounded(w_next)).held(dtype).holds(normed)
        assert float(normed[0].abs().max()) > 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
@pytest.mark.parametrize("hidden", [384, 4096, 9000])
def test_gradients_of_large_outputs_and_residuals(dtype, gate, hidden):
    n = 5
    say(f"gradients of large blocks {dtype} {gate} hidden={hidden}")
    for size_y, size_r in ((1e19, 1e19), (1e19, 1.0), (1.0, 1e19), (1e30, 1e25)):
        d = make(n, hidden, dtype, True, gate, hidden)
        d["y"], d["res"] = large(n, hidden, size_y, 1).to(dtype), large(n, hidden, size_r, 2).to(dtype)
        leaves = {k: d[k].to(dev()).requires_grad_() for k in ("y", "res", "gate", "post", "next") if d[k] is not None}
        outs = residual_norm(leaves["y"], leaves["res"], post_weight=leaves["post"], gate=leaves.get("gate"), scale=0.5,
                             next_weight=leaves["next"], eps=EPS)
        grads = torch.autograd.grad(outs, list(leaves.values()), (d["dh"].to(dev()), d["dn"].to(dev())))
        want = backward(d, True, True, 0.5)
        for name, got in zip(leaves, grads):
            assert want[name].holds(got), (name, size_y, size_r)


def test_infinite_rows_stay_as_they_were():
    x = torch.ones(4, 600)
    x[0, 3], x[1, 5], x[2] = float("inf"), float("nan"), 3e38
    w = torch.ones(600)
    say("infinite rows")
    out = rms_norm(x.to(dev()), w.to(dev())).cpu()
    assert out[0, 3].isnan() and (out[0, :3] == 0).all() and out[1].isnan().all()
    # (one over 3e38 is not a normal number: 2^-149 of 2^-128)
    assert ((out[2] - 1).abs() <= 2.0**-20).all() and ((out[3] - 1).abs() <= 2.0**-19).all()


@pytest.mark.parametrize("n,hidden", [(1_100_003, 520), (4_300_003, 16)])
def test_more_than_two_to_the_twenty_workgroups(n, hidden):
    """The launch has two dimensions: rows at both ends and around workgroup 2^20 against small calls."""
    say(f"{n} rows of {hidden}")
    g = torch.Generator(device=dev()).manual_seed(0)
    y = torch.randn(n, hidden, generator=g, device=dev(), dtype=torch.bfloat16)
    res = torch.randn(n, hidden, generator=g, device=dev(), dtype=torch.bfloat16)
    w = torch.rand(hidden, generator=g, device=dev())
    gate = torch.rand(n, 1, generator=g, device=dev())
    normed = rms_norm(y, w)
    out = residual_norm(y, res, post_weight=w, gate=gate, next_weight=w)
    rows = 4 if hidden <= 512 else 1  # of a workgroup
    for at in (0, n // 2, rows * 2**20 - 60, n - 100):
        part = slice(at, at + 100)
        assert torch.equal(rms_norm(y[part], w), normed[part])
        small = residual_norm(y[part], res[part], post_weight=w, gate=gate[part], next_weight=w)
        assert torch.equal(small.hidden, out.hidden[part]) and torch.equal(small.normed, out.normed[part])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["none", "channel", "token", "element"])
@pytest.mark.parametrize("n,hidden", [(30, 40), (700, 512), (600, 1000), (30, 133), (9, 2048), (40, 3001), (6, 4096), (3, 9000)])
def test_rows_of_any_alignment_have_the_same_bits(dtype, kind, n, hidden):
    """A lane holds the same values whatever the rows' alignment, so sums have one order."""
    g = torch.Generator().manual_seed(n + hidden)
    y, res, dh, dn = (torch.randn(n, hidden, generator=g).to(dtype) for _ in range(4))
    w_post, w_next = (1 + 0.3 * torch.randn(hidden, generator=g) for _ in range(2))
    shape = {"none": None, "channel": (hidden,), "token": (n, 1), "element": (n, hidden)}[kind]
    gate = None if shape is None else torch.tanh(torch.randn(*shape, generator=g)).to(dev())
    say(f"alignment {dtype} {kind} n={n} hidden={hidden}")
    results = []
    for left, right in ((0, 0), (0, 8 - hidden % 8), (1, 6), (3, 2), (8, 8)):
        def placed(t):
            wide = torch.full((t.shape[0], left + hidden + right), 3.0, dtype=t.dtype, device=dev())
            wide[:, left : left + hidden] = t.to(dev())
            return wide[:, left : left + hidden].requires_grad_()

        leaves = [placed(y), placed(res), placed(w_post[None]), placed(w_next[None])]
        if gate is not None:
            leaves.append(gate.clone().requires_grad_())
        ys, rs, wp, wn = leaves[:4]
        outs = residual_norm(ys, rs, post_weight=wp[0], gate=leaves[4] if gate is not None else None, scale=0.3, next_weight=wn[0])
        results.append([t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, (dh.to(dev()), dn.to(dev())))))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("hidden", [1, 7, 64])
def test_one_token_and_its_gate(hidden):
    """y [hidden], a gate per token of [1], per channel of [hidden]."""
    g = torch.Generator().manual_seed(2)
    y, res, gate = torch.randn(hidden, generator=g), torch.randn(hidden, generator=g), torch.randn(1, generator=g)
    say(f"one token hidden={hidden}")
    leaves = [t.to(dev()).requires_grad_() for t in (y, res, gate)]
    out = residual_norm(leaves[0], leaves[1], gate=leaves[2], scale=0.5)
    rows = [t.to(dev()).view(1, -1).requires_grad_() for t in (y, res, gate)]
    want = residual_norm(rows[0], rows[1], gate=rows[2], scale=0.5)
    assert out.hidden.shape == (hidden,) and torch.equal(out.hidden, want.hidden[0])
    g_out = torch.randn(hidden, generator=g).to(dev())
    for got, exp, leaf in zip(torch.autograd.grad(out.hidden, leaves, g_out), torch.autograd.grad(want.hidden, rows, g_out[None]), leaves):
        assert got.shape == leaf.shape and torch.equal(got.view(-1), exp.view(-1))
