"""GPU: the dense FP8 block product where an activation scale times a weight scale leaves fp32, and the result does not.

Against 64 bits on the same codes and scales. The codes' products are whole multiples of a number above 2^-13 of the largest,
which the matrix instruction adds up exactly; what is left is a fold per K block, off by at most 2^-23 of what it adds up to,
and the rounding to bf16: half a step, 2^-8 of the value (2^-134 among its denormals)."""

import math

import numpy as np
import pytest
import torch

from gpu_util import dev, say
from oracle import formats as F
from sgl_asap_amd.moe.linear import Fp8BlockLinear
from sgl_asap_amd.moe.shared import silu_mul

pytestmark = pytest.mark.gpu

# a call of each form: rows that quantize themselves, few rows, and tiles of every shape
FORMS = [(1, 384, 40), (3, 640, 100), (20, 1024, 36), (9, 4096, 50), (40, 4096, 33), (64, 2048, 48), (65, 384, 130),
         (500, 256, 4100), (1000, 256, 4000), (1500, 384, 4096), (2885, 256, 4091), (8200, 256, 2048)]


def ceil(a, b):
    return -(-a // b)


def parts(x):
    """Codes and scales of x in 64 bits, [n, kb, 128] and [n, kb]."""
    n, k = x.shape
    v = np.zeros((n, ceil(k, 128) * 128), dtype=np.float32)
    v[:, :k] = x.float().numpy()
    q, s = F.fp8_group_quantize(v)
    return torch.from_numpy(F.e4m3_decode(q).astype(np.float64)).view(n, -1, 128), torch.from_numpy(s.astype(np.float64))


def product(x, w, s):
    """(y, sum of |terms|) in 64 bits; w: e4m3 as float [n_out, k], s its block scales."""
    q, sx = parts(x)
    n_out, k = w.shape
    wide = torch.zeros(n_out, q.shape[1] * 128, dtype=torch.float64)
    wide[:, :k] = w.double()
    rows = torch.arange(n_out) // 128
    y, mass = (torch.zeros(x.shape[0], n_out, dtype=torch.float64) for _ in range(2))
    for b in range(q.shape[1]):
        part = wide[:, b * 128 : (b + 1) * 128]
        both = sx[:, b : b + 1] * s.double()[rows, b][None]
        y += (q[:, b] @ part.t()) * both
        mass += (q[:, b].abs() @ part.abs().t()) * both.abs()
    return y, mass


def check(y, want, mass, k):
    y = y.cpu().double()
    assert torch.isfinite(want).all() and float(want.abs().max()) < 3e38
    tol = 2.0**-8 * want.abs() + (2 + k / 128) * 2.0**-23 * mass + 2.0**-133
    assert torch.isfinite(y).all()
    assert ((y - want).abs() <= tol).all(), float(((y - want).abs() / tol).max())


def whole(shape, most, g):
    return torch.randint(-most, most + 1, shape, generator=g).float()


def rows_of_scale(n, k, sx, step, g):
    """x = sx times multiples of step up to 7 step, and one 448 in each block: its scale is sx, its codes are exact."""
    x = whole((n, k), 7, g) * step
    x[:, torch.arange(ceil(k, 128)) * 128 + 5] = 448.0
    return x * sx


@pytest.mark.parametrize("n,k,n_out", FORMS)
def test_products_of_scales_past_the_largest_float(n, k, n_out):
    """Each block has an x of 448 2^119 where the weights are 0: sx = 2^119, weight scales past 2^9, results from the rest."""
    g = torch.Generator().manual_seed(n + k)
    x = rows_of_scale(n, k, 2.0**119, 1.0, g)
    w = whole((n_out, k), 3, g) * 2.0**-9 * (torch.rand(n_out, k, generator=g) < 0.02)
    w[:, torch.arange(ceil(k, 128)) * 128 + 5] = 0.0
    w[::3] = 0.0  # outputs that are 0, not 0 times infinity
    s = 700.0 + 300.0 * torch.rand(ceil(n_out, 128), ceil(k, 128), generator=g)
    if n > 2:
        x[1] = rows_of_scale(1, k, 1.0, 1.0, g)[0]  # an ordinary row beside them
    x = x.to(torch.bfloat16)
    say(f"huge products n={n} k={k} n_out={n_out}")
    y = Fp8BlockLinear(w.to(torch.float8_e4m3fn).to(dev()), s.to(dev()))(x.to(dev()))
    want, mass = product(x, w, s)
    assert (want[:, ::3] == 0).all() and (want != 0).any()
    check(y, want, mass, k)


@pytest.mark.parametrize("n,k,n_out", FORMS)
def test_products_of_scales_among_the_denormals(n, k, n_out):
    """sx sw around 2^-143 and block sums around 2^19: the result is a normal number."""
    g = torch.Generator().manual_seed(n + k)
    x = rows_of_scale(n, k, 2.0**-32, 32.0, g)
    w = whole((n_out, k), 3, g) * 64.0
    s = 2.0**-111 * (0.5 + torch.rand(ceil(n_out, 128), ceil(k, 128), generator=g))
    if n_out > 128:
        s[0] = 1e-3  # a block of ordinary scales
    if k > 256:
        s[:, 1] = 0.0
    if n > 2:
        x[1] = rows_of_scale(1, k, 1.0, 32.0, g)[0]
    x = x.to(torch.bfloat16)
    say(f"tiny products n={n} k={k} n_out={n_out}")
    y = Fp8BlockLinear(w.to(torch.float8_e4m3fn).to(dev()), s.to(dev()))(x.to(dev()))
    want, mass = product(x, w, s)
    assert float(want[0].abs().max()) > 2.0**-126
    check(y, want, mass, k)


@pytest.mark.parametrize("n,k,n_out", [(2, 384, 140), (40, 2048, 133), (130, 304, 140), (700, 304, 2000)])
def test_both_in_one_call_from_strided_rows_and_the_activation(n, k, n_out):
    g = torch.Generator().manual_seed(n)
    w = whole((n_out, k), 3, g) * 64.0
    s = 2.0**-111 * (0.5 + torch.rand(ceil(n_out, 128), ceil(k, 128), generator=g))
    s[1] = 900.0
    x = rows_of_scale(n, k, 2.0**-32, 32.0, g)
    x[1::2] = rows_of_scale(x[1::2].shape[0], k, 2.0**-5, 32.0, g)
    x = x.to(torch.bfloat16)
    layer = Fp8BlockLinear(w.to(torch.float8_e4m3fn).to(dev()), s.to(dev()))
    say(f"both n={n} k={k} n_out={n_out}")
    wide = torch.full((n, k + 5), 3.0, dtype=torch.bfloat16, device=dev())
    wide[:, 3 : 3 + k] = x.to(dev())
    out = torch.full((n + 1, n_out + 3), 7.0, dtype=torch.bfloat16, device=dev())
    layer(wide[:, 3 : 3 + k], out=out[:n, 1 : 1 + n_out])
    check(out[:n, 1 : 1 + n_out], *product(x, w, s), k)
    out[:n, 1 : 1 + n_out] = 7.0
    assert (out == 7.0).all()
    gu = torch.randn(n, 2 * k, generator=g)
    gu[::2, k:] *= 1e-9
    gu = gu.to(torch.bfloat16).to(dev())
    assert torch.equal(layer.silu_mul(gu), layer(silu_mul(gu)))


@pytest.mark.parametrize("n,k,n_out", [(2, 384, 40), (40, 2048, 33), (130, 300, 140)])
def test_infinite_and_nan_weight_scales_stay_in_their_block(n, k, n_out):
    """0 times infinity is NaN, anything else times it infinite; a tiny scale beside it changes nothing in other blocks."""
    g = torch.Generator().manual_seed(n)
    n_out = max(n_out, 140)
    x = torch.randint(1, 5, (n, k), generator=g).to(torch.bfloat16)  # (codes are multiples of 1 with a 4 in each block)
    x[:, ::128] = 4.0
    w = torch.ones(n_out, k)
    w[5] = 0.0
    s = torch.full((ceil(n_out, 128), ceil(k, 128)), 2.0**-4)
    s[0, 0], s[0, 1] = math.inf, 2.0**-120
    say(f"infinite scales n={n}")
    y = Fp8BlockLinear(w.to(torch.float8_e4m3fn).to(dev()), s.to(dev()))(x.to(dev())).cpu().double()
    assert y[:, 5].isnan().all() and (y[:, :5] == math.inf).all()
    want, mass = product(x, w[128:], s[1:])
    check(y[:, 128:], want, mass, k)
    s[0, 0] = math.nan
    y = Fp8BlockLinear(w.to(torch.float8_e4m3fn).to(dev()), s.to(dev()))(x.to(dev())).cpu().double()
    assert y[:, :128].isnan().all()
    check(y[:, 128:], want, mass, k)
