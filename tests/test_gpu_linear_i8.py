"""GPU parity of the dense int8 product (afd_linear_i8) and the shared expert on it.

The codes, the sums and every rounding are defined, so the result is one bit pattern: ``expected`` makes it on the CPU
from int64 sums. Against 64 bits the same results are within half a bf16 step (2^-8 of the value) and the three fp32
roundings (of the sum, of the scales' product and of their product: 3 x 2^-24)."""

import copy
import pickle

import numpy as np
import pytest
import torch

from gpu_util import bits16, dev, say
from sgl_asap_amd.moe.linear import Int8Linear
from sgl_asap_amd.moe.shared import Int8SharedExpertMLP, silu_mul

pytestmark = pytest.mark.gpu

REL = 2.0**-8 + 3 * 2.0**-24


def quantized(x):
    """(codes int64, scales fp32 [n, 1]) of bf16 x on the CPU; a row that is not finite: codes 0, scale NaN."""
    v = x.float().numpy()
    good = np.isfinite(v).all(1, keepdims=True)
    v = np.where(good, v, np.float32(0))
    s = np.maximum(np.abs(v).max(1, keepdims=True), np.float32(1e-10)) / np.float32(127)
    q = np.rint(v / s)
    assert np.abs(q).max(initial=0) <= 127
    return torch.from_numpy(q).long(), torch.from_numpy(np.where(good, s, np.float32("nan")).astype(np.float32))


def sums(q, w):
    """Exact integer products of codes, in fp64 (all below 2^53)."""
    return q.double() @ w.double().t()


def expected(x, w, s):
    q, sx = quantized(x)
    return (sums(q, w).float() * (sx * s[None])).to(torch.bfloat16)


def random(n, k, n_out, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, k, generator=g) * torch.exp(spread * torch.randn(n, 1, generator=g))).to(torch.bfloat16)
    w = torch.randint(-128, 128, (n_out, k), generator=g, dtype=torch.int8)
    return x, w, torch.rand(n_out, generator=g) * 1e-3 + 1e-5


def layer_of(w, s):
    return Int8Linear(w.to(dev()), s.to(dev()))


def same(a, b):
    return np.array_equal(bits16(a), bits16(b))


SIZES = [(1, 1, 1), (1, 128, 16), (1, 300, 77), (2, 4096, 130), (15, 65, 200), (16, 256, 15), (17, 129, 257), (31, 2048, 64),
         (33, 127, 33), (48, 512, 96), (64, 1000, 129), (65, 128, 128), (100, 640, 700), (127, 130, 1), (128, 384, 257),
         (200, 2000, 111), (257, 256, 4), (300, 72, 513), (1025, 500, 640), (1, 4096, 512), (7, 777, 300), (24, 2048, 1000),
         (60, 1536, 64), (90, 1111, 500), (333, 5000, 250), (40, 9000, 60), (70, 9001, 33)]


@pytest.mark.parametrize("n,k,n_out", SIZES)
def test_bits(n, k, n_out):
    x, w, s = random(n, k, n_out, n + k)
    say(f"int8 n={n} k={k} n_out={n_out}")
    y = layer_of(w, s)(x.to(dev())).cpu()
    assert same(y, expected(x, w, s))
    q, sx = quantized(x)
    want = sums(q, w) * sx.double() * s.double()
    assert ((y.double() - want).abs() <= REL * want.abs()).all()


@pytest.mark.parametrize("n,n_out", [(65, 4096), (500, 4100), (1000, 4000), (1500, 4096), (2900, 4096), (70, 65000), (5000, 300),
                                     (5800, 4096), (2885, 4091), (3900, 3100), (8200, 2048), (4096, 4096), (100, 130), (300, 1111),
                                     (1500, 1536), (2900, 1600), (3800, 2048), (2900, 4352), (66, 200), (300, 3000)])
def test_bits_of_every_tile_shape(n, n_out):
    """Calls that take each of the tile shapes, with rows and outputs that end inside a tile."""
    k = 700
    x, w, s = random(n, k, n_out, n)
    say(f"int8 tiles n={n} n_out={n_out}")
    y = layer_of(w, s)(x.to(dev())).cpu()
    q, sx = quantized(x)
    # sums of at most 700 x 127 x 128 < 2^24 are exact in fp32
    want = ((q.float() @ w.float().t()) * (sx * s[None])).to(torch.bfloat16)
    assert same(y, want)


def test_largest_sums():
    """Every product 127 x -128 over the widest row: the sum of 65536 x 16256 stays in 32 bits."""
    k = 65536
    w = torch.full((20, k), -128, dtype=torch.int8)
    w[3] = 127
    s = torch.full((20,), 2.0**-20)
    for n in (1, 5, 70, 300):
        x = torch.full((n, k), 127.0, dtype=torch.bfloat16)
        say(f"largest sums n={n}")
        y = layer_of(w, s)(x.to(dev())).cpu()
        assert same(y, expected(x, w, s))
        assert float(y[0, 0]) == -float(torch.tensor(127.0 * 128 * k * 2.0**-20).to(torch.bfloat16))


def test_widest_layer():
    for n, k, n_out in ((3, 65536, 20), (70, 65536, 20), (2, 130, 65536), (300, 130, 65535)):
        x, w, s = random(n, k, n_out, 1)
        say(f"widest n={n} k={k} n_out={n_out}")
        assert same(layer_of(w, s)(x.to(dev())), expected(x, w, s))


@pytest.mark.parametrize("n", [3, 40, 150, 2600])
def test_scales_of_any_size(n):
    """Channel scales of 0, tiny, huge, negative, infinite and NaN, each its own channel's matter."""
    k, n_out = 256, 1300
    x, w, s = random(n, k, n_out, 9, spread=20.0)
    x[0] = 3e38
    x[1] = 1e-38
    odd = torch.tensor([0.0, 2.0**-100, 2.0**-126, 2.0**-140, 2.0**60, 2.0**100, -0.5, -(2.0**-120), float("inf"), float("nan"),
                        2.0**-85, 2.0**6, 3.4e38])
    s[100 : 100 + len(odd)] = odd
    s[1287:] = odd
    say(f"scales n={n}")
    y = layer_of(w, s)(x.to(dev())).cpu().double()
    q, sx = quantized(x)
    total = sums(q, w)
    want = total * (sx.double() * s.double())
    nan = want.isnan()
    assert nan[:, 1296].all() and torch.equal(y.isnan(), nan)
    # infinite channels, and results that leave bf16, are infinite; the rest within the bound and half of bf16's least step
    top = float(torch.finfo(torch.bfloat16).max)
    big = want.abs() > top * (1 + 2.0**-8)
    assert torch.equal(y[big], want[big].sign() * float("inf"))
    near = ~nan & (want.abs() <= top)
    assert ((y - want).abs()[near] <= (REL * want.abs() + 2.0**-134)[near]).all()


@pytest.mark.parametrize("n", [5, 37, 140, 2600])
def test_rows_with_infinities_and_nans_stay_apart(n):
    k, n_out = 300, 1500
    x, w, s = random(n, k, n_out, 2)
    bad = x.clone()
    bad[1, 5], bad[2, 290], bad[4, 130] = float("inf"), float("nan"), float("-inf")
    layer = layer_of(w, s)
    say(f"bad rows n={n}")
    good, y = layer(x.to(dev())), layer(bad.to(dev()))
    rows = [1, 2, 4]
    assert y[rows].isnan().all()
    keep = torch.ones(n, dtype=torch.bool, device=dev())
    keep[rows] = False
    assert same(y[keep], good[keep])


def test_rows_of_zeros_and_of_small_numbers():
    x = torch.zeros(20, 256, dtype=torch.bfloat16)
    x[3:10] = 1e-30  # below the least scale: codes 0
    x[10:] = torch.finfo(torch.bfloat16).max
    w, s = torch.ones(32, 256, dtype=torch.int8), torch.full((32,), 2.0**-10)
    say("zeros, small, largest")
    y = layer_of(w, s)(x.to(dev())).cpu()
    assert (y[:10] == 0).all() and same(y, expected(x, w, s))


@pytest.mark.parametrize("n,k,n_out", [(9, 200, 50), (70, 256, 40), (130, 130, 136)])
def test_strides_shapes_and_what_lies_between(n, k, n_out):
    x, w, s = random(n, k, n_out, 1)
    layer = layer_of(w, s)
    xd = x.to(dev())
    want = layer(xd)
    say(f"strides n={n} k={k} n_out={n_out}")
    for ldx, x0, ldy, y0 in ((k + 9, 3, n_out + 5, 1), (k + 8 - k % 8 + 8, 8, n_out + 8 - n_out % 8 + 8, 8)):
        wide = torch.full((n, ldx + x0), float("nan"), dtype=torch.bfloat16, device=dev())
        wide[:, x0 : x0 + k] = xd
        y = torch.full((n + 3, ldy + y0), 7.0, dtype=torch.bfloat16, device=dev())
        got = layer(wide[:, x0 : x0 + k], out=y[:n, y0 : y0 + n_out])
        assert got.data_ptr() == y[:, y0:].data_ptr() and torch.equal(got, want)
        y[:n, y0 : y0 + n_out] = 7.0
        assert (y == 7.0).all()
    t = xd.t().contiguous().t()
    assert torch.equal(layer(t), want)
    assert torch.equal(layer(xd.view(n, 1, 1, k)).view(n, n_out), want)
    assert torch.equal(layer(t[0]), want[0]) and layer(t[:0]).shape == (0, n_out)
    assert torch.equal(layer(t[:1].expand(5, k)), want[:1].expand(5, n_out))


def test_a_row_does_not_depend_on_the_rows_beside_it():
    """The sums are exact: the same bits from every form, on every stream."""
    x, w, s = random(700, 2048, 512, 3)
    layer = layer_of(w, s)
    x = x.to(dev())
    say("same bits, streams")
    want = layer(x)
    for n in (1, 5, 16, 17, 32, 33, 50, 64, 65, 300):
        assert same(layer(x[:n]), want[:n]), n
    side = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i, st in enumerate(side):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append([layer(x[: 20 + 100 * i]) for _ in range(20)])
    torch.cuda.synchronize()
    for i, many in enumerate(outs):
        assert all(same(y, want[: 20 + 100 * i]) for y in many)


def test_captured_and_replayed():
    x, w, s = random(200, 1024, 512, 8)
    layer = layer_of(w, s)
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
    layer = layer_of(w, s)
    y = torch.full((n, ldy), 5.0, dtype=torch.bfloat16, device=dev())
    layer(x, out=y[:, :n_out])
    for at in (0, 524_200, 1_048_500, n - 100):
        part = slice(at, at + 100)
        assert same(y[part, :n_out], expected(x[part].cpu(), w, s))
    assert (y[:, n_out:] == 5.0).all()


@pytest.mark.parametrize("n", [1, 20, 130])
def test_shared_expert(n):
    hidden, inter = 384, 200
    g = torch.Generator().manual_seed(6)
    wg = torch.randint(-127, 128, (2 * inter, hidden), generator=g, dtype=torch.int8)
    wd = torch.randint(-127, 128, (hidden, inter), generator=g, dtype=torch.int8)
    sg, sd = torch.rand(2 * inter, generator=g) * 1e-3, torch.rand(hidden, 1, generator=g) * 1e-3
    x = torch.randn(n, hidden, generator=g).to(torch.bfloat16)
    say(f"shared expert n={n}")
    y = Int8SharedExpertMLP(*(t.to(dev()) for t in (wg, sg, wd, sd)))(x.to(dev()))
    h = silu_mul(layer_of(wg, sg)(x.to(dev())))
    assert same(y, layer_of(wd, sd)(h))
    # gate and up as their bits are; the activation may round to the other bf16, which may move a code by one of 127
    gate, up = expected(x, wg, sg).double().chunk(2, dim=1)
    q, sx = quantized((gate * torch.sigmoid(gate) * up).to(torch.bfloat16))
    want = sums(q, wd) * (sx.double() * sd.double().t())
    rel = float((y.cpu().double() - want).norm() / want.norm())
    assert rel <= 2.0**-6, rel


@pytest.mark.parametrize("n,inter,n_out", [(1, 256, 64), (3, 1536, 384), (20, 200, 100), (47, 131, 65), (64, 384, 260), (130, 128, 48),
                                           (700, 640, 513), (2600, 1536, 512), (9000, 2048, 40), (50, 9000, 40), (30, 6000, 70)])
def test_silu_mul_in_the_quantization(n, inter, n_out):
    """The same bits as the activation and the layer one after the other, from rows with a stride and into them."""
    g = torch.Generator().manual_seed(n + inter)
    w = torch.randint(-128, 128, (n_out, inter), generator=g, dtype=torch.int8)
    s = torch.rand(n_out, generator=g) * 1e-3
    gu = (torch.randn(n, 2 * inter, generator=g) * 3).to(torch.bfloat16)
    gu[0, :5] = 100.0
    if n > 2:
        gu[1], gu[2, 7], gu[n - 1, inter] = 0.0, float("inf"), float("nan")
    layer = layer_of(w, s)
    say(f"silu n={n} inter={inter} n_out={n_out}")
    gu = gu.to(dev())
    want = layer(silu_mul_any(gu))
    got = layer.silu_mul(gu)
    assert same(got, want)
    if n > 2:
        assert torch.isnan(got[2]).all() and torch.isnan(got[n - 1]).all() and torch.isfinite(got[0]).all()
    buf = torch.full((n, 2 * inter + 24), 7.0, dtype=torch.bfloat16, device=dev())
    buf[:, 8 : 8 + 2 * inter] = gu
    out = torch.full((n, n_out + 9), 5.0, dtype=torch.bfloat16, device=dev())
    layer.silu_mul(buf[:, 8 : 8 + 2 * inter], out=out[:, :n_out])
    assert same(out[:, :n_out], want) and (out[:, n_out:] == 5).all()
    assert same(layer.silu_mul(gu.view(1, n, 2 * inter))[0], want)


def silu_mul_any(gate_up):
    """silu_mul of any number of columns: its kernel's rows padded to a multiple of 8."""
    n, inter = gate_up.shape[0], gate_up.shape[1] // 2
    pad = (inter + 7) // 8 * 8
    wide = torch.zeros(n, 2, pad, dtype=torch.bfloat16, device=gate_up.device)
    wide[:, :, :inter] = gate_up.view(n, 2, inter)
    return silu_mul(wide.view(n, 2 * pad))[:, :inter].contiguous()


def test_refusals_of_calls():
    x, w, s = random(6, 256, 256, 8)
    layer = layer_of(w, s)
    buf = torch.zeros(9, 512, dtype=torch.bfloat16, device=dev())
    rows = buf[:6, :256]
    say("refusals")
    for bad in (rows.float(), rows[:, :255], torch.zeros((), dtype=torch.bfloat16, device=dev())):
        with pytest.raises(TypeError):
            layer(bad)
    with pytest.raises(ValueError):
        layer(x)
    with pytest.raises(NotImplementedError, match="Int8Linear"):
        layer(rows.clone().requires_grad_())
    with pytest.raises(TypeError):
        layer.silu_mul(rows)
    for out in (rows, buf[1:7, :256], buf[:6, 128:384]):
        with pytest.raises(ValueError, match="shares"):
            layer(rows, out=out)
    for out in (buf[:6, 256:511], buf[:5, 256:], torch.empty(6, 256, device=dev())):
        with pytest.raises(ValueError):
            layer(rows, out=out)
    assert layer(rows, out=buf[:6, 256:]).shape == (6, 256)


def test_copied_and_pickled():
    x, w, s = random(20, 300, 100, 5)
    layer = layer_of(w, s[:, None])
    say("copied, pickled")
    want = layer(x.to(dev()))
    assert same(want, expected(x, w, s))
    for other in (copy.deepcopy(layer), pickle.loads(pickle.dumps(layer)), layer.to(torch.float16)):
        assert same(other(x.to(dev())), want)
