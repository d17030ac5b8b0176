"""GPU: int8 products whose channels' scales are of ordinary and of odd sizes side by side: each channel's result is its own."""

import pytest
import torch

from gpu_util import bits16, dev, say
from sgl_asap_amd.moe.linear import Int8Linear

pytestmark = pytest.mark.gpu


def scales(n_out, every, seed):
    """Of about 1e-4, every ``every``-th far below or above what an fp32 product of scales is sure to hold."""
    s = torch.rand(n_out, generator=torch.Generator().manual_seed(seed)) * 1e-3 + 1e-5
    odd = torch.tensor([2.0**-100, 2.0**-90, 2.0**20, -(2.0**-110), 2.0**40])
    s[1::every] = odd.repeat(-(-n_out // 5))[: s[1::every].numel()]
    return s


@pytest.mark.parametrize("n,k,n_out,every", [(2048, 700, 1536, 8), (2048, 520, 1531, 5), (6400, 256, 640, 16), (300, 1111, 2000, 11)])
def test_a_row_has_the_same_bits_beside_any_rows(n, k, n_out, every):
    g = torch.Generator().manual_seed(n + k)
    x = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(torch.bfloat16).to(dev())
    w = torch.randint(-128, 128, (n_out, k), generator=g, dtype=torch.int8)
    s = scales(n_out, every, 3)
    say(f"odd scales n={n} k={k} n_out={n_out} every={every}")
    layer = Int8Linear(w.to(dev()), s.to(dev()))
    whole = layer(x)
    # up to 64 rows take another form of the kernel
    parts = torch.cat([layer(x[i : i + 64]) for i in range(0, n, 64)])
    assert torch.equal(whole, parts), int((whole != parts).sum())
    # an ordinary channel does not see the odd ones beside it
    plain = s.clone()
    plain[1::every] = 1e-4
    alone = Int8Linear(w.to(dev()), plain.to(dev()))(x)
    keep = torch.ones(n_out, dtype=torch.bool)
    keep[1::every] = False
    keep = keep.to(dev())
    assert torch.equal(whole[:, keep], alone[:, keep]), int((whole[:, keep] != alone[:, keep]).sum())


def test_bits_of_both_kinds_of_channels():
    """Sums below 2^24 are exact in fp32: ordinary channels are the sum times the product of the scales, each rounded to
    fp32, odd ones the product in 64 bits."""
    n, k, n_out = 2500, 600, 1536
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(torch.bfloat16)
    w = torch.randint(-128, 128, (n_out, k), generator=g, dtype=torch.int8)
    s = scales(n_out, 8, 5)
    v = x.float()
    sx = v.abs().amax(1, keepdim=True) / torch.full((n, 1), 127.0)
    total = torch.round(v / sx) @ w.float().t()
    odd = torch.zeros(n_out, dtype=torch.bool)
    odd[1::8] = True
    ordinary = (total * (sx * s)).to(torch.bfloat16)
    wide = (total.double() * (sx.double() * s.double())).float().to(torch.bfloat16)
    want = torch.where(odd, wide, ordinary)
    say("bits of odd and ordinary channels")
    y = Int8Linear(w.to(dev()), s.to(dev()))(x.to(dev())).cpu()
    assert (bits16(y) == bits16(want)).all(), int((bits16(y) != bits16(want)).sum())
