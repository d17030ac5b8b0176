"""GPU parity of the dense FP8 block product (afd_linear) and the shared expert on it.

Exact cases: integers whose every partial sum fp32 holds, so the bf16 result has one right
answer. Random cases: against 64 bits on the same codes, within half a bf16 step (2^-8 of the value) plus the
fp32 sums' error: every addition is off by at most 2^-23 of what it adds up to, below sum |terms|, and a
result is made of 128-term block sums (at most 128 additions) and K / 128 folds."""

import numpy as np
import pytest
import torch

from gpu_util import bits16, dev, say
from oracle import formats as F
from sgl_asap_amd.moe.linear import Fp8BlockLinear
from sgl_asap_amd.moe.shared import Fp8SharedExpertMLP, silu_mul

pytestmark = pytest.mark.gpu


def e4m3(v):
    return v.to(torch.float8_e4m3fn)


def ceil(a, b):
    return -(-a // b)


def integers(n, k, n_out, seed):
    """x of integers in [-7, 7] with one 448 in each block of 128, so its scale is 1 and its codes are
    exact; weights of integers in [-3, 3], scales powers of two. |sums| < 2^24."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-7, 8, (n, k), generator=g).float()
    for b in range(ceil(k, 128)):
        at = b * 128 + torch.randint(0, min(128, k - b * 128), (n,), generator=g)
        x[torch.arange(n), at] = 448.0
    w = torch.randint(-3, 4, (n_out, k), generator=g).float()
    s = torch.pow(2.0, torch.randint(-1, 2, (ceil(n_out, 128), ceil(k, 128)), generator=g).float())
    return x, w, s


def widen(s, n_out, k):
    return s.repeat_interleave(128, 0)[:n_out].repeat_interleave(128, 1)[:, :k]


SIZES = [(1, 1, 1), (1, 128, 16), (1, 300, 77), (2, 4096, 130), (15, 65, 200), (16, 256, 15), (17, 129, 257), (31, 2048, 64),
         (33, 127, 33), (48, 512, 96), (64, 1000, 129), (65, 128, 128), (100, 640, 700), (127, 130, 1), (128, 384, 257),
         (200, 2000, 111), (257, 256, 4), (300, 72, 513), (1025, 500, 640)]


@pytest.mark.parametrize("n,k,n_out", SIZES)
def test_exact_integers(n, k, n_out):
    x, w, s = integers(n, k, n_out, n + k)
    say(f"exact n={n} k={k} n_out={n_out}")
    layer = Fp8BlockLinear(e4m3(w).to(dev()), s.to(dev()))
    y = layer(x.to(torch.bfloat16).to(dev()))
    want = (x.double() @ (w.double() * widen(s, n_out, k).double()).t()).float().to(torch.bfloat16)
    assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("n,n_out", [(4096, 4096), (4000, 4100), (8200, 2048)])
def test_exact_integers_large_tiles(n, n_out):
    k = 400
    x, w, s = integers(n, k, n_out, 5)
    say(f"exact, many tiles n={n} n_out={n_out}")
    layer = Fp8BlockLinear(e4m3(w).to(dev()), s.to(dev()))
    y = layer(x.to(torch.bfloat16).to(dev()))
    want = (x @ (w * widen(s, n_out, k)).t()).to(torch.bfloat16)  # exact in fp32 too
    assert torch.equal(y.cpu(), want)


def same(a, b):
    """The same bits (the random weights hold a few NaN codes)."""
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def close(y, want, mass, additions):
    """Within the tolerance above; NaN exactly where the definition says (a weight code that is NaN)."""
    tol = 2.0**-8 * want.abs() + additions * 2.0**-23 * mass
    nan = want.isnan()
    return torch.equal(y.isnan(), nan) and bool(((y - want).abs() <= tol)[~nan].all())


def random(n, k, n_out, seed):
    """Weights past 464 (about one in 300000) have no e4m3 number and become its NaN code."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(torch.bfloat16)
    w = e4m3(torch.randn(n_out, k, generator=g) * 100)
    s = torch.rand(ceil(n_out, 128), ceil(k, 128), generator=g) * 1e-3
    return x, w, s


def quantized(x):
    """x as the product reads it, through the oracle's 1x128 quantizer (short last block padded with 0)."""
    n, k = x.shape
    v = np.zeros((n, ceil(k, 128) * 128), dtype=np.float32)
    v[:, :k] = x.float().numpy()
    return torch.from_numpy(F.fp8_group_dequantize(*F.fp8_group_quantize(v))[:, :k].astype(np.float64))


@pytest.mark.parametrize("n,k,n_out", [(1, 4096, 512), (7, 777, 300), (24, 2048, 1000), (60, 1536, 64), (90, 1111, 500),
                                       (333, 3000, 250), (2048, 640, 8192)])
def test_random_against_64_bits(n, k, n_out):
    x, w, s = random(n, k, n_out, n)
    say(f"random n={n} k={k} n_out={n_out}")
    y = Fp8BlockLinear(w.to(dev()), s.to(dev()))(x.to(dev())).cpu().double()
    q = quantized(x)
    wd = w.double() * widen(s, n_out, k).double()
    want, mass = q @ wd.t(), q.abs() @ wd.abs().t()
    assert close(y, want, mass, 128 + k / 128)


@pytest.mark.parametrize("n", [3, 40, 150, 2600])
def test_scales_of_any_size(n):
    """Block scales of 0, tiny and huge: each block is folded by itself."""
    k, n_out = 512, 6400
    x, w, _ = integers(n, k, n_out, 9)
    s = torch.tensor([0.0, 2.0**-100, 2.0**60, 1.0]).repeat(50, 1)
    s[1] = torch.tensor([2.0**60, 0.0, 0.0, 0.0])
    s[2] = 0.0
    s[3] = torch.tensor([0.0, 2.0**-140, 0.0, 0.0])
    say(f"scales n={n}")
    y = Fp8BlockLinear(e4m3(w).to(dev()), s.to(dev()))(x.to(torch.bfloat16).to(dev())).cpu().double()
    want = x.double() @ (w.double() * widen(s, n_out, k).double()).t()
    mass = x.double().abs() @ (w.double() * widen(s, n_out, k).double()).abs().t()
    assert ((y - want).abs() <= 2.0**-8 * want.abs() + 8 * 2.0**-23 * mass + 2.0**-133).all()


@pytest.mark.parametrize("n", [5, 37, 140, 2600])
def test_rows_with_infinities_and_nans_stay_apart(n):
    k, n_out = 300, 6400
    x, w, s = integers(n, k, n_out, 2)
    bad = x.clone()
    bad[1, 5], bad[2, 290], bad[4, 130] = float("inf"), float("nan"), float("-inf")
    layer = Fp8BlockLinear(e4m3(w).to(dev()), s.to(dev()))
    say(f"bad rows n={n}")
    good, y = (layer(v.to(torch.bfloat16).to(dev())) for v in (x, bad))
    rows = [1, 2, 4]
    assert y[rows].isnan().all()
    keep = torch.ones(n, dtype=torch.bool)
    keep[rows] = False
    assert torch.equal(y[keep.to(dev())], good[keep.to(dev())])


def test_rows_of_zeros_and_of_small_numbers():
    x = torch.zeros(20, 256, dtype=torch.bfloat16)
    x[3:10] = 1e-30  # below the quantizer's least scale: codes 0
    x[10:] = torch.finfo(torch.bfloat16).max
    say("zeros, small, largest")
    w = torch.ones(32, 256)
    y = Fp8BlockLinear(e4m3(w).to(dev()), torch.full((1, 2), 2.0**-10, device=dev()))(x.to(dev())).cpu()
    assert (y[:10] == 0).all()
    want = quantized(x[10:]).sum(1) * 2.0**-10
    assert ((y[10:].double() - want[:, None]).abs() <= 2.0**-8 * want[:, None]).all()


@pytest.mark.parametrize("n,k,n_out", [(9, 200, 50), (70, 256, 40), (130, 130, 136)])
def test_strides_shapes_and_what_lies_between(n, k, n_out):
    x, w, s = integers(n, k, n_out, 1)
    layer = Fp8BlockLinear(e4m3(w).to(dev()), s.to(dev()))
    want = layer(x.to(torch.bfloat16).to(dev()))
    say(f"strides n={n} k={k} n_out={n_out}")
    for ldx, x0, ldy, y0 in ((k + 9, 3, n_out + 5, 1), (k + 8 - k % 8 + 8, 8, n_out + 8 - n_out % 8 + 8, 8)):
        wide = torch.full((n, ldx + x0), float("nan"), dtype=torch.bfloat16, device=dev())
        wide[:, x0 : x0 + k] = x.to(torch.bfloat16).to(dev())
        y = torch.full((n + 3, ldy + y0), 7.0, dtype=torch.bfloat16, device=dev())
        got = layer(wide[:, x0 : x0 + k], out=y[:n, y0 : y0 + n_out])
        assert got.data_ptr() == y[:, y0:].data_ptr() and torch.equal(got, want)
        y[:n, y0 : y0 + n_out] = 7.0
        assert (y == 7.0).all()
    t = x.to(torch.bfloat16).to(dev()).t().contiguous().t()
    assert torch.equal(layer(t), want)
    assert torch.equal(layer(x.to(torch.bfloat16).to(dev()).view(n, 1, 1, k)).view(n, n_out), want)
    assert torch.equal(layer(t[0]), want[0]) and layer(t[:0]).shape == (0, n_out)
    row = t[:1].expand(5, k)
    assert torch.equal(layer(row), want[:1].expand(5, n_out))


def test_same_bits_in_every_form_of_few_rows_and_on_other_streams():
    """A row's result does not depend on the rows beside it within one form, and repeated calls agree."""
    x, w, s = random(64, 2048, 512, 3)
    layer = Fp8BlockLinear(w.to(dev()), s.to(dev()))
    x = x.to(dev())
    say("few rows, streams")
    want = layer(x)
    for n in (1, 5, 16, 17, 32, 33, 50):
        assert same(layer(x[:n]), want[:n]), n
    side = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i, st in enumerate(side):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append([layer(x[: 20 + i]) for _ in range(20)])
    torch.cuda.synchronize()
    for i, many in enumerate(outs):
        assert all(same(y, want[: 20 + i]) for y in many)


def test_captured_and_replayed():
    x, w, s = random(200, 1024, 512, 8)
    layer = Fp8BlockLinear(w.to(dev()), s.to(dev()))
    say("captured")
    graphs = []
    for n in (3, 40, 200):
        buf = x[:n].to(dev()).clone()
        layer(buf)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(buf)
        graphs.append((graph, buf, out))
    for i in range(3):
        for graph, buf, out in graphs:
            buf.copy_(random(buf.shape[0], 1024, 512, 20 + i)[0].to(dev()))
            graph.replay()
            want = layer(buf.clone())
            torch.cuda.synchronize()
            assert same(out, want)


def test_rows_past_32_bits():
    """x, its codes and y past 2^32 bytes; rows at the ends and in between against small calls."""
    n, k, n_out, ldy = 1_100_000, 4096, 24, 2048
    say("1.1 M rows of 4096")
    g = torch.Generator(device=dev()).manual_seed(0)
    x = torch.randn(n, k, generator=g, device=dev(), dtype=torch.bfloat16)
    _, w, s = random(1, k, n_out, 4)
    layer = Fp8BlockLinear(w.to(dev()), s.to(dev()))
    y = torch.full((n, ldy), 5.0, dtype=torch.bfloat16, device=dev())
    layer(x, out=y[:, :n_out])
    for at in (0, 524_200, 1_048_500, n - 100):
        part = slice(at, at + 100)
        q = quantized(x[part].cpu())
        wd = w.double() * widen(s, n_out, k).double()
        want, mass = q @ wd.t(), q.abs() @ wd.abs().t()
        assert close(y[part, :n_out].cpu().double(), want, mass, 128 + k / 128)
    assert (y[:, n_out:] == 5.0).all()


def test_widest_layer():
    """65536 inputs, and 65536 outputs."""
    for n, k, n_out in ((3, 65536, 20), (70, 65536, 20), (2, 130, 65536), (300, 130, 65535)):
        x, w, s = random(n, k, n_out, 1)
        say(f"widest n={n} k={k} n_out={n_out}")
        y = Fp8BlockLinear(w.to(dev()), s.to(dev()))(x.to(dev())).cpu().double()
        q = quantized(x)
        wd = w.double() * widen(s, n_out, k).double()
        want, mass = q @ wd.t(), q.abs() @ wd.abs().t()
        assert close(y, want, mass, 128 + k / 128)


@pytest.mark.parametrize("n", [1, 20, 130])
def test_shared_expert(n):
    hidden, inter = 384, 200
    g = torch.Generator().manual_seed(6)
    wg, wd = e4m3(torch.randn(2 * inter, hidden, generator=g) * 50), e4m3(torch.randn(hidden, inter, generator=g) * 50)
    sg, sd = torch.rand(4, 3, generator=g) * 2e-3, torch.rand(3, 2, generator=g) * 2e-3
    x = torch.randn(n, hidden, generator=g).to(torch.bfloat16).to(dev())
    say(f"shared expert n={n}")
    mlp = Fp8SharedExpertMLP(*(t.to(dev()) for t in (wg, sg, wd, sd)))
    y = mlp(x)
    # its parts are the layer's own, so the whole is theirs bit for bit
    h = silu_mul(Fp8BlockLinear(wg.to(dev()), sg.to(dev()))(x))
    assert np.array_equal(bits16(y), bits16(Fp8BlockLinear(wd.to(dev()), sd.to(dev()))(h)))
    gu = quantized(x.cpu()) @ (wg.double() * widen(sg, 2 * inter, hidden).double()).t()
    gate, up = gu[:, :inter], gu[:, inter:]
    act = (gate * torch.sigmoid(gate) * up).float().to(torch.bfloat16)
    want = quantized(act) @ (wd.double() * widen(sd, hidden, inter).double()).t()
    # a code of h may be its neighbour (1/8 apart at most) where gate and up round to other bf16
    rel = float((y.cpu().double() - want).norm() / want.norm())
    assert rel <= 2.0**-5, rel


@pytest.mark.parametrize("n,n_out", [(65, 4096), (500, 4100), (1000, 4000), (1500, 4096), (2900, 4096), (70, 65000), (5000, 300),
                                     (5800, 4096), (2885, 4091), (3900, 3100)])
def test_exact_integers_every_tile_shape(n, n_out):
    """Calls that take each of the tile shapes, with rows and outputs that end inside a tile."""
    k = 700
    x, w, s = integers(n, k, n_out, n)
    say(f"exact, tile shapes n={n} n_out={n_out}")
    y = Fp8BlockLinear(e4m3(w).to(dev()), s.to(dev()))(x.to(torch.bfloat16).to(dev()))
    want = (x @ (w * widen(s, n_out, k)).t()).to(torch.bfloat16)  # exact in fp32 too
    assert torch.equal(y.cpu(), want)


def test_out_that_shares_elements_with_x_is_refused():
    n, k = 6, 256
    x, w, s = integers(n, k, k, 8)
    layer = Fp8BlockLinear(e4m3(w).to(dev()), s.to(dev()))
    buf = torch.zeros(n + 3, 3 * k, dtype=torch.bfloat16, device=dev())
    buf[:n, :k] = x.to(torch.bfloat16).to(dev())
    rows = buf[:n, :k]
    say("out over x")
    for out in (rows, buf[1 : n + 1, :k], buf[:n, 128 : 128 + k], buf[:n, k - 1 : 2 * k - 1]):
        with pytest.raises(ValueError, match="shares"):
            layer(rows, out=out)
    with pytest.raises(NotImplementedError):
        layer(rows.clone(), out=torch.zeros(n, k, dtype=torch.bfloat16, device=dev(), requires_grad=True))
    say("out beside x in one buffer")
    want = layer(rows.clone())
    for at in (k, 2 * k):
        out = buf[:n, at : at + k]
        assert layer(rows, out=out) is out and torch.equal(out, want)
    assert torch.equal(buf[:n, :k].cpu(), x.to(torch.bfloat16))


@pytest.mark.parametrize("n,inter,n_out", [(1, 256, 64), (3, 1536, 384), (20, 200, 100), (47, 131, 65), (64, 384, 260), (130, 128, 48),
                                           (700, 640, 513), (2600, 1536, 512), (9000, 2048, 40)])
def test_silu_mul_in_the_quantization(n, inter, n_out):
    """The same bits as the activation and the layer one after the other, from rows with a stride and into them."""
    g = torch.Generator().manual_seed(n + inter)
    w, s = e4m3(torch.randn(n_out, inter, generator=g) * 50), torch.rand(ceil(n_out, 128), ceil(inter, 128), generator=g) * 2e-3
    gu = (torch.randn(n, 2 * inter, generator=g) * 3).to(torch.bfloat16)
    gu[0, :5] = 100.0
    if n > 2:
        gu[1], gu[2, 7], gu[n - 1, inter] = 0.0, float("inf"), float("nan")
    layer = Fp8BlockLinear(w.to(dev()), s.to(dev()))
    say(f"silu n={n} inter={inter} n_out={n_out}")
    gu = gu.to(dev())
    want = layer(silu_mul_any(gu))
    got = layer.silu_mul(gu)
    assert np.array_equal(bits16(got), bits16(want))
    if n > 2:
        assert torch.isnan(got[2]).all() and torch.isnan(got[n - 1]).all() and torch.isfinite(got[0]).all()
    buf = torch.full((n, 2 * inter + 24), 7.0, dtype=torch.bfloat16, device=dev())
    buf[:, 8 : 8 + 2 * inter] = gu
    out = torch.full((n, n_out + 9), 5.0, dtype=torch.bfloat16, device=dev())
    layer.silu_mul(buf[:, 8 : 8 + 2 * inter], out=out[:, :n_out])
    assert np.array_equal(bits16(out[:, :n_out]), bits16(want)) and (out[:, n_out:] == 5).all()
    assert np.array_equal(bits16(layer.silu_mul(gu.view(1, n, 2 * inter))[0]), bits16(want))


def silu_mul_any(gate_up):
    """silu_mul of any number of columns: its kernel's rows padded to a multiple of 8."""
    n, inter = gate_up.shape[0], gate_up.shape[1] // 2
    pad = (inter + 7) // 8 * 8
    wide = torch.zeros(n, 2, pad, dtype=torch.bfloat16, device=gate_up.device)
    wide[:, :, :inter] = gate_up.view(n, 2, inter)
    return silu_mul(wide.view(n, 2 * pad))[:, :inter].contiguous()


def test_silu_mul_refusals_and_capture():
    g = torch.Generator().manual_seed(1)
    w, s = e4m3(torch.randn(96, 256, generator=g) * 50), torch.rand(1, 2, generator=g) * 2e-3
    layer = Fp8BlockLinear(w.to(dev()), s.to(dev()))
    gu = torch.randn(30, 512, generator=g).to(torch.bfloat16).to(dev())
    say("silu refusals, capture")
    with pytest.raises(TypeError):
        layer.silu_mul(gu[:, :256])
    with pytest.raises(TypeError):
        layer.silu_mul(gu.float())
    with pytest.raises(ValueError):
        layer.silu_mul(gu, out=gu[:, :96])
    with pytest.raises(NotImplementedError):
        layer.silu_mul(gu.clone().requires_grad_())
    assert layer.silu_mul(gu[:0]).shape == (0, 96)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.silu_mul(gu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.silu_mul(gu)
    for _ in range(3):
        gu.copy_(torch.randn(30, 512, generator=g).to(torch.bfloat16).to(dev()))
        graph.replay()
        assert torch.equal(y, layer(silu_mul(gu)))
