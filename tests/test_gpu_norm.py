"""GPU parity of the norms before and after a block with its gate and residual scale (afd_residual_norm and its gradient).

Against 64 bits, within what fp32's operations and the results' types may be off (``error_bounds``): the bounds follow the
formulas, with the sums over a row and over the tokens in any order."""

import pytest
import torch

from error_bounds import Bounded
from gpu_util import dev, say
from sgl_asap_amd.moe.norm import BlockNorms, residual_norm, rms_norm

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5


def make(n, hidden, dtype, wide, gate, seed, shape=None):
    g = torch.Generator().manual_seed(seed)
    held = torch.float32 if wide else dtype
    shape = shape or (n,)
    d = dict(y=torch.randn(*shape, hidden, generator=g) * torch.exp(torch.randn(*shape, 1, generator=g)),
             res=2 * torch.randn(*shape, hidden, generator=g))
    d = {k: v.to(dtype) for k, v in d.items()}
    size = {"none": None, "channel": (hidden,), "token": (*shape, 1), "element": (*shape, hidden)}[gate]
    d["gate"] = None if size is None else torch.tanh(torch.randn(*size, generator=g)).to(held)
    d["post"], d["next"] = ((1 + 0.3 * torch.randn(hidden, generator=g)).to(held) for _ in range(2))
    d["dh"], d["dn"] = (torch.randn(*shape, hidden, generator=g).to(dtype) for _ in range(2))
    return d


def on_gpu(d, *names, grad=True):
    return [None if d[k] is None else d[k].to(dev()).requires_grad_(grad) for k in names]


def unit(v, eps=EPS):
    r = (v * v).mean().over_root(eps)
    return v * r, r


def forward(d, post, nxt, scale):
    """(h before it is rounded, h, normed) with bounds."""
    y = Bounded(d["y"])
    if post:
        y = unit(y)[0] * Bounded(d["post"])
    f = y * scale
    if d["gate"] is not None:
        f = f * Bounded(d["gate"])
    h = Bounded(d["res"]) + f
    dtype = d["y"].dtype
    return h, h.held(dtype), (unit(h)[0] * Bounded(d["next"])).held(dtype) if nxt else None


def backward(d, post, nxt, scale, dh=True, dn=True):
    """{name: gradient with bounds}; h as it is before it is rounded."""
    dtype, out = d["y"].dtype, {}
    h = forward(d, post, nxt, scale)[0]
    g = Bounded(torch.zeros_like(d["y"])) if not dh else Bounded(d["dh"])
    if nxt and dn:
        r = unit(h)[1]
        u = h * r
        q = Bounded(d["dn"]) * Bounded(d["next"])
        out["next"] = (Bounded(d["dn"]) * u).sum(0).held(d["next"].dtype)
        g = g + r * (q - u * (q * u).mean())
    out["res"] = g.held(dtype)
    y = Bounded(d["y"])
    v, r = unit(y) if post else (y, None)
    f = v * Bounded(d["post"]) if post else v
    if d["gate"] is not None:
        e = g * f * scale
        gate = d["gate"]
        e = e.sum(0) if gate.dim() == 1 else e.sum(-1, True) if gate.shape[-1] == 1 and d["y"].shape[-1] > 1 else e
        out["gate"] = e.held(gate.dtype)
        g = g * Bounded(gate)
    g = g * scale
    if post:
        out["post"] = (g * v).sum(0).held(d["post"].dtype)
        g = g * Bounded(d["post"])
        g = r * (g - v * (g * v).mean())
    out["y"] = g.held(dtype)
    return out


SHAPES = [(1, 1), (3, 8), (5, 131), (70, 512), (9, 520), (33, 1111), (600, 640), (7, 2048), (5, 3001), (40, 4096), (3, 5000), (2, 8192),
          (3, 10001), (2, 16384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,hidden", SHAPES)
def test_before_a_block(dtype, n, hidden):
    for wide in (False, True):
        d = make(n, hidden, dtype, wide, "none", n + hidden)
        say(f"rms_norm {dtype} n={n} hidden={hidden} wide={wide}")
        x, w = on_gpu(d, "y", "next")
        out = rms_norm(x, w, eps=EPS)
        assert out.dtype == dtype
        v, r = unit(Bounded(d["y"]))
        assert (v * Bounded(d["next"])).held(dtype).holds(out.detach())
        dx, dw = torch.autograd.grad(out, (x, w), d["dn"].to(dev()))
        q = Bounded(d["dn"]) * Bounded(d["next"])
        assert (r * (q - v * (q * v).mean())).held(dtype).holds(dx)
        assert (Bounded(d["dn"]) * v).sum(0).held(w.dtype).holds(dw)
        assert torch.equal(out, rms_norm(x.detach(), w.detach(), eps=EPS))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
@pytest.mark.parametrize("post,nxt", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("n,hidden", [(5, 130), (50, 512), (700, 264), (33, 1111), (20, 2048), (9, 4096), (3, 9000)])
def test_after_a_block(dtype, gate, post, nxt, n, hidden):
    wide = (n + hidden) % 2 == 0
    d = make(n, hidden, dtype, wide, gate, n)
    scale = 0.22 if post else 1.5
    say(f"residual_norm {dtype} {gate} post={post} next={nxt} n={n} hidden={hidden}")
    y, res, g, w_post, w_next = on_gpu(d, "y", "res", "gate", "post", "next")
    w_post, w_next = w_post if post else None, w_next if nxt else None
    h, normed = residual_norm(y, res, post_weight=w_post, gate=g, scale=scale, next_weight=w_next, eps=EPS)
    _, want_h, want_n = forward(d, post, nxt, scale)
    assert h.dtype == dtype and want_h.holds(h.detach())
    assert (normed is None) if not nxt else want_n.holds(normed.detach())
    again = residual_norm(*(t.detach() for t in (y, res)), post_weight=None if w_post is None else w_post.detach(),
                          gate=None if g is None else g.detach(), scale=scale,
                          next_weight=None if w_next is None else w_next.detach(), eps=EPS)
    assert torch.equal(again.hidden, h) and (normed is None or torch.equal(again.normed, normed))
    leaves = {k: t for k, t in dict(y=y, res=res, gate=g, post=w_post, next=w_next).items() if t is not None}
    for with_h, with_n in ((True, True), (True, False), (False, True)):
        if with_n and not nxt and (not with_h or (with_h, with_n) == (True, True)):
            with_n = False
            if not with_h:
                continue
        outs, given = ([h] if with_h else []) + ([normed] if with_n else []), []
        given = ([d["dh"].to(dev())] if with_h else []) + ([d["dn"].to(dev())] if with_n else [])
        grads = torch.autograd.grad(outs, list(leaves.values()), given, retain_graph=True, allow_unused=True)
        want = backward(d, post, nxt, scale, with_h, with_n)
        for name, got in zip(leaves, grads):
            if name == "next" and not with_n:
                assert got is None
                continue
            assert got.dtype == leaves[name].dtype and got.shape == leaves[name].shape
            assert want[name].holds(got), (name, with_h, with_n)
        # each gradient alone is the same bits
        for name, got in zip(leaves, grads):
            if got is not None and with_h:
                (only,) = torch.autograd.grad(outs, leaves[name], given, retain_graph=True)
                assert torch.equal(only, got), name


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_tokens(dtype):
    """More tokens than slots of the sums, in each of the row's forms."""
    for n, hidden in ((5000, 96), (3001, 1030), (1300, 4096)):
        d = make(n, hidden, dtype, True, "channel", 5)
        say(f"many tokens {dtype} n={n} hidden={hidden}")
        leaves = on_gpu(d, "y", "res", "gate", "post", "next")
        y, res, g, w_post, w_next = leaves
        outs = residual_norm(y, res, post_weight=w_post, gate=g, scale=0.5, next_weight=w_next, eps=EPS)
        grads = torch.autograd.grad(outs, leaves, (d["dh"].to(dev()), d["dn"].to(dev())))
        want = backward(d, True, True, 0.5)
        for name, got in zip(("y", "res", "gate", "post", "next"), grads):
            assert want[name].holds(got), name


def test_gradient_against_differences():
    """fp32: a central difference of the kernel's own output in a random direction, h in 64 bits on the CPU."""
    n, hidden = 6, 48
    d = make(n, hidden, torch.float32, True, "channel", 3)
    leaves = on_gpu(d, "y", "res", "gate", "post", "next")
    say("differences")

    def loss(ts):
        h, m = residual_norm(ts[0], ts[1], post_weight=ts[3], gate=ts[2], scale=0.7, next_weight=ts[4], eps=EPS)
        return (h.double() * d["dh"].to(dev()).double()).sum() + (m.double() * d["dn"].to(dev()).double()).sum()

    grads = torch.autograd.grad(loss(leaves), leaves)
    gen = torch.Generator().manual_seed(4)
    step = 2.0**-7
    for i in range(5):
        way = torch.randn(leaves[i].shape, generator=gen).to(dev())
        way /= way.norm()
        a, b = ([t.detach() + (s * step * way if j == i else 0) for j, t in enumerate(leaves)] for s in (1, -1))
        diff = float((loss(a) - loss(b)) / (2 * step))
        exact = float((grads[i].double() * way.double()).sum())
        # outputs below 8, 2 x 288 of them, each off by 8 x 8 x 2^-24 at most, over 2 steps: 2^-4.4 were all off one way, as
        # random signs 2^-9; the third derivative's share is below step^2 x 100 = 2^-7
        assert abs(diff - exact) <= 2.0**-6, (i, diff, exact)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hidden", [64, 2000, 4100])
def test_zeros_infinities_and_nans_stay_in_their_rows(dtype, hidden):
    n = 40
    d = make(n, hidden, dtype, False, "element", 1)
    for k in ("y", "res"):
        d[k][3] = 0.0
    bad = {k: v.clone() for k, v in d.items()}
    bad["y"][5, 1], bad["res"][6, 0], bad["gate"][7, 2], bad["y"][8] = float("inf"), float("nan"), float("nan"), float("-inf")
    say(f"bad rows {dtype} hidden={hidden}")
    results = []
    for data in (d, bad):
        y, res, g, w_post, w_next = leaves = on_gpu(data, "y", "res", "gate", "post", "next")
        outs = residual_norm(y, res, post_weight=w_post, gate=g, next_weight=w_next, eps=EPS)
        dh, dn = data["dh"].to(dev()), data["dn"].to(dev())
        results.append([*outs, *torch.autograd.grad(outs, leaves[:3], (dh, dn))])
    keep = [i for i in range(n) if i not in (5, 6, 7, 8)]
    for a, b in zip(*results):
        assert torch.equal(a[keep], b[keep]) and a.isfinite().all()
        assert not b[[5, 6, 7, 8]].isfinite().all(1).any()
    # a row of zeros: h 0, normed 0
    assert (results[0][0][3] == 0).all() and (results[0][1][3] == 0).all()
    # without the norm after the block an infinite y does not reach its own gradient
    y, res = on_gpu(bad, "y", "res")
    scale = 0.5
    dy, dr = torch.autograd.grad(residual_norm(y, res, scale=scale).hidden, (y, res), d["dh"].to(dev()))
    assert torch.equal(dr.cpu(), d["dh"]) and torch.equal(dy.cpu(), d["dh"] * scale)
    g = d["gate"][0, :hidden].clone().to(dev()).requires_grad_()
    dy, dg = torch.autograd.grad(residual_norm(y, res, gate=g).hidden, (y, g), d["dh"].to(dev()))
    assert dy.isfinite().all() and not dg.isfinite().all()


def test_large_and_small_values():
    """Squares up to fp32's largest and rows far below eps."""
    say("large, small")
    x = torch.zeros(4, 256)
    x[0], x[1], x[2, 7] = 1e18, 1e-20, 1e18
    w = torch.ones(256)
    out = rms_norm(x.to(dev()), w.to(dev()), eps=1e-6)
    want = unit(Bounded(x), 1e-6)[0]
    assert want.held(torch.float32).holds(out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hidden", [40, 133, 1000, 4096])
def test_strides_shapes_and_broadcast_gradients(dtype, hidden):
    n = 30
    d = make(n, hidden, dtype, False, "token", 2)
    y, res, g, w_post, w_next = on_gpu(d, "y", "res", "gate", "post", "next", grad=False)
    kw = dict(post_weight=w_post, scale=0.3, next_weight=w_next, eps=EPS)
    want = residual_norm(y, res, gate=g, **kw)
    say(f"strides {dtype} hidden={hidden}")
    grads = None
    for left in (0, 3, 8):
        wide = torch.full((n, 2 * hidden + 40), float("nan"), dtype=dtype, device=dev())
        ys, rs = wide[:, left : left + hidden], wide[:, hidden + left + 16 : 2 * hidden + left + 16]
        ys.copy_(y)
        rs.copy_(res)
        ws = torch.zeros(hidden + 5, dtype=dtype, device=dev())[left : left + hidden] if left < 5 else w_post.clone()
        ws.copy_(w_post)
        ya, ra, ga, wa = (t.detach().requires_grad_() for t in (ys, rs, g, ws))
        got = residual_norm(ya, ra, gate=ga, **dict(kw, post_weight=wa))
        # (rows of other alignments are read in another order, so their sums may round otherwise)
        tight = 8 * torch.finfo(dtype).eps
        for a, b in zip(got, want):
            assert ((a - b).abs().double() <= tight * (1 + b.abs().double())).all()
        here = torch.autograd.grad((got.hidden.sum(), got.normed.sum()), (ya, ra, ga, wa))
        if grads is not None:
            for a, b in zip(here, grads):
                top = b.abs().double().max()
                assert ((a - b).abs().double() <= 16 * torch.finfo(dtype).eps * top).all()
        grads = here
    for shape in ((2, 15, hidden), (30, 1, 1, hidden)):
        got = residual_norm(y.view(shape), res.view(shape), gate=g.view(shape[:-1] + (1,)), **kw)
        assert got.hidden.shape == shape and got.normed.shape == shape
        assert torch.equal(got.hidden.view(n, hidden), want.hidden) and torch.equal(got.normed.view(n, hidden), want.normed)
    one = residual_norm(y[0], res[0], gate=g[:1, 0].expand(hidden) if hidden > 1 else None, **kw)
    assert one.hidden.shape == (hidden,)
    assert torch.equal(rms_norm(y[3], w_next, eps=EPS), rms_norm(y, w_next, eps=EPS)[3])
    t = y.t().contiguous().t()
    assert torch.equal(residual_norm(t, res, gate=g, **kw).hidden, want.hidden)
    # y and the residual the same tensor, and a residual that was broadcast
    x = y.detach().clone().requires_grad_()
    (dx,) = torch.autograd.grad(residual_norm(x, x).hidden, x, d["dh"].to(dev()))
    assert torch.equal(dx, d["dh"].to(dev()) + d["dh"].to(dev()))
    row = res[:1].detach().clone().requires_grad_()
    residual_norm(y, row.expand(n, hidden)).hidden.backward(torch.ones_like(y))
    assert torch.equal(row.grad, torch.full_like(row, float(n)))


def test_no_tokens():
    say("no tokens")
    y = torch.zeros(0, 64, device=dev(), requires_grad=True)
    w, g = (torch.ones(64, device=dev(), requires_grad=True) for _ in range(2))
    h, m = residual_norm(y, y, post_weight=w, gate=g, next_weight=w)
    assert h.shape == (0, 64) and m.shape == (0, 64)
    (h.sum() + m.sum()).backward()
    assert y.grad.shape == (0, 64) and (w.grad == 0).all() and (g.grad == 0).all()
    assert rms_norm(y.view(0, 2, 64), w).shape == (0, 2, 64)


def test_derivatives_that_are_refused():
    d = make(6, 32, torch.float32, True, "channel", 7)
    y, res, g, w_post, w_next = leaves = on_gpu(d, "y", "res", "gate", "post", "next")
    say("second derivatives")
    for i, leaf in enumerate(leaves):
        out = residual_norm(y, res, post_weight=w_post, gate=g, next_weight=w_next)
        (first,) = torch.autograd.grad(out.hidden.square().sum() + out.normed.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="no second"):
            first.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(y.detach(), torch.ones_like(y))
        for call in (lambda: rms_norm(dual, w_next), lambda: residual_norm(y, dual), lambda: residual_norm(dual, y)):
            with pytest.raises(NotImplementedError):
                call()
    out = residual_norm(y, res, next_weight=w_next)
    out.hidden.detach().add_(1.0)  # (not what the backward reads)
    (before,) = torch.autograd.grad(out.normed, y, y.detach(), retain_graph=True)
    (after,) = torch.autograd.grad(residual_norm(y, res, next_weight=w_next).normed, y, y.detach())
    assert torch.equal(before, after)
    with torch.no_grad():
        res.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        out.normed.sum().backward()


def test_captured_and_replayed():
    n, hidden = 300, 512
    d = make(n, hidden, torch.bfloat16, True, "channel", 7)
    buf = on_gpu(d, "y", "res", "gate", "post", "next", grad=False)
    dh = d["dh"].to(dev())
    say("captured")

    def step():
        y, res, g, w_post, w_next = leaves = [t.detach().requires_grad_() for t in buf]
        x = rms_norm(y, w_next)
        outs = residual_norm(x, res, post_weight=w_post, gate=g, scale=0.5, next_weight=w_next)
        return [*outs, *torch.autograd.grad(outs, leaves, (dh, dh))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(3):
        new = make(n, hidden, torch.bfloat16, True, "channel", 20 + i)
        for t, k in zip(buf, ("y", "res", "gate", "post", "next")):
            t.copy_(new[k].to(dev()))
        for graph, _ in graphs:
            graph.replay()
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def test_streams():
    say("streams")
    data = [on_gpu(make(200 + i, 1000, torch.bfloat16, True, "token", i), "y", "res", "gate", "post", "next") for i in range(3)]

    def step(ts):
        y, res, g, w_post, w_next = ts
        outs = residual_norm(y, res, post_weight=w_post, gate=g, next_weight=w_next)
        return [*outs, *torch.autograd.grad(outs, ts, (y.detach(), res.detach()))]

    want = [step(ts) for ts in data]
    torch.cuda.synchronize()
    side, got = [torch.cuda.Stream() for _ in data], []
    for _ in range(10):
        for st, ts in zip(side, data):
            with torch.cuda.stream(st):
                got.append(step(ts))
    torch.cuda.synchronize()
    for i, many in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(many, want[i % 3]))


def test_rows_past_32_bits():
    """Activations past 2^32 bytes: the ends against small calls."""
    n, hidden = 600_000, 4096
    say("600000 rows of 4096")
    g = torch.Generator(device=dev()).manual_seed(0)
    y = torch.randn(n, hidden, generator=g, device=dev(), dtype=torch.bfloat16).requires_grad_()
    res = torch.randn(n, hidden, generator=g, device=dev(), dtype=torch.bfloat16).requires_grad_()
    w = torch.rand(hidden, generator=g, device=dev())
    gate = torch.rand(n, 1, generator=g, device=dev())
    out = residual_norm(y, res, post_weight=w, gate=gate, next_weight=w)
    dy, dr = torch.autograd.grad(out, (y, res), (res.detach(), y.detach()))
    for at in (0, 262_100, 524_250, n - 100):
        part = slice(at, at + 100)
        a, b = (t[part].detach().requires_grad_() for t in (y, res))
        small = residual_norm(a, b, post_weight=w, gate=gate[part], next_weight=w)
        assert torch.equal(small.hidden, out.hidden[part]) and torch.equal(small.normed, out.normed[part])
        for s, full in zip(torch.autograd.grad(small, (a, b), (b.detach(), a.detach())), (dy, dr)):
            assert torch.equal(s, full[part])


def test_refusals_of_calls():
    d = make(6, 32, torch.bfloat16, False, "channel", 7)
    y, res, g, w_post, w_next = on_gpu(d, "y", "res", "gate", "post", "next", grad=False)
    say("refusals")
    with pytest.raises(ValueError):
        residual_norm(y, res, post_weight=w_post.cpu())
    with pytest.raises(ValueError):
        residual_norm(y, res.cpu())
    with pytest.raises(ValueError):
        residual_norm(y, res, gate=g.cpu())
    with pytest.raises(ValueError):
        rms_norm(torch.zeros(2, 16385, device=dev()), torch.zeros(16385, device=dev()))


def test_module():
    n, hidden = 12, 96
    d = make(n, hidden, torch.bfloat16, True, "channel", 9)
    y, res, g, w_post, w_next = on_gpu(d, "y", "res", "gate", "post", "next", grad=False)
    say("module")
    norms = BlockNorms(w_next, w_post, g, scale=0.25, eps=EPS)
    assert [k for k, _ in norms.named_parameters()] == ["input_weight", "post_weight", "gate"]
    assert torch.equal(norms.before(y), rms_norm(y, w_next, eps=EPS))
    kw = dict(post_weight=w_post, scale=0.25, eps=EPS)
    assert torch.equal(norms.after(y, res).hidden, residual_norm(y, res, gate=g, **kw).hidden)
    token = torch.rand(n, 1, device=dev())
    got = norms.after(y, res, gate=token, next_weight=w_next)
    want = residual_norm(y, res, gate=token, next_weight=w_next, **kw)
    assert torch.equal(got.hidden, want.hidden) and torch.equal(got.normed, want.normed)
    out = norms.after(norms.before(y), res)
    out.hidden.sum().backward()
    assert all(p.grad is not None and p.grad.shape == (hidden,) for p in norms.parameters())
    plain = BlockNorms(w_next)
    assert torch.equal(plain.after(y, res).hidden, residual_norm(y, res).hidden)
