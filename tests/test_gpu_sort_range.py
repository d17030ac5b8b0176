"""GPU: sorted tokens at the ends of their range: ids and expert_lo, workgroups past 2^20, rows of any alignment."""

import pytest
import torch

from gpu_util import dev, say
from sgl_asap_amd.moe.sort import sort_tokens, unsort_tokens

pytestmark = pytest.mark.gpu

LEAST, LARGEST = -(2**31), 2**31 - 1


@pytest.mark.parametrize("n", [6, 3000])
@pytest.mark.parametrize("lo", [0, 5, LARGEST - 700, LARGEST - 3, LARGEST])
def test_ids_and_first_expert_of_any_size(n, lo):
    """A negative id is nowhere, also where the difference to expert_lo leaves 32 bits."""
    experts = 900
    g = torch.Generator().manual_seed(n)
    ids = torch.tensor([LEAST, LEAST + 1, LEAST + 800, -1, 0, 4, 5, 700, LARGEST - 701, LARGEST - 700, LARGEST - 1, LARGEST],
                       dtype=torch.int32)
    ids = ids[torch.randint(0, ids.numel(), (n, 3), generator=g)]
    e = ids.long() - lo
    here = (e >= 0) & (e < experts)
    key = torch.where(here, e, experts).reshape(-1)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel())
    place[~here.reshape(-1)] = -1
    say(f"ids n={n} lo={lo}")
    x = torch.randn(n, 8, generator=g)
    rows, got = sort_tokens(x.to(dev()), ids.to(dev()), experts, expert_lo=lo)
    assert torch.equal(got.positions.cpu().long(), place.view(n, 3))
    assert torch.equal(got.counts.cpu().long(), torch.bincount(key, minlength=experts + 1)[:experts])
    assert int(got.offsets[-1]) == int(here.sum())
    assert (rows[int(here.sum()) :] == 0).all()


def test_more_than_two_to_the_twenty_workgroups():
    """4.3 million tokens: the moves, the way back and its gradient are launched in two dimensions."""
    n, hidden, experts = 4_300_003, 16, 7
    say("4300003 tokens of 16")
    g = torch.Generator(device=dev()).manual_seed(0)
    x = torch.randn(n, hidden, generator=g, device=dev(), dtype=torch.bfloat16).requires_grad_()
    ids = torch.randint(-1, experts, (n, 1), generator=g, device=dev(), dtype=torch.int32)
    w = torch.rand(n, 1, generator=g, device=dev()).requires_grad_()
    rows, order = sort_tokens(x, ids, experts)
    here = ids[:, 0] >= 0
    used = int(here.sum())
    key = torch.where(here, ids[:, 0], experts).cpu()
    want = torch.empty(n, dtype=torch.int64)
    want[torch.sort(key, stable=True).indices] = torch.arange(n)
    place = order.positions[:, 0].cpu().long()
    assert torch.equal(place, torch.where(here.cpu(), want, -1)) and int(order.offsets[-1]) == used
    sent, at = here.nonzero()[:, 0], order.positions[here, 0].long()
    moved = torch.zeros_like(rows)
    moved[at] = x.detach()[sent]
    assert torch.equal(rows, moved)
    out = unsort_tokens(rows, order, w)
    # one product a value in fp32, rounded once
    assert torch.equal(out, torch.where(here[:, None], (x.float() * w).to(torch.bfloat16), torch.zeros_like(x)))
    grad = torch.randn(n, hidden, generator=g, device=dev(), dtype=torch.bfloat16)
    dr, dw = torch.autograd.grad(out, (rows, w), grad)
    moved.zero_()
    moved[at] = (grad.float() * w.detach()).to(torch.bfloat16)[sent]
    assert torch.equal(dr, moved)
    exact = torch.where(here, (grad.double() * x.detach().double()).sum(-1), 0.0)
    mass = (grad.double() * x.detach().double()).abs().sum(-1)
    # 16 products and additions, then the result in fp32
    assert ((dw[:, 0].double() - exact).abs() <= 17 * 2.0**-24 * mass).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,hidden,k", [(40, 64, 4), (2000, 72, 3), (1300, 1000, 8), (30, 2048, 2), (25, 513, 4), (1100, 35, 2)])
def test_rows_of_any_alignment_have_the_same_bits(dtype, n, hidden, k):
    """A lane holds the same values whatever the rows' alignment, so sums have one order."""
    g = torch.Generator().manual_seed(n + hidden)
    x, rows = torch.randn(n, hidden, generator=g).to(dtype), torch.randn(n * k, hidden, generator=g).to(dtype)
    w, ids = torch.rand(n, k, generator=g), torch.randint(-1, 9, (n, k), generator=g).int()
    grad = torch.randn(n, hidden, generator=g).to(dtype).to(dev())
    say(f"alignment {dtype} n={n} hidden={hidden} k={k}")
    results = []
    for left, right in ((0, 0), (0, 8 - hidden % 8), (1, 6), (3, 2), (8, 8)):
        def placed(t):
            wide = torch.full((t.shape[0], left + hidden + right), 3.0, dtype=dtype, device=dev())
            wide[:, left : left + hidden] = t.to(dev())
            return wide[:, left : left + hidden]

        got, order = sort_tokens(placed(x), ids.to(dev()), 9)
        rs, ws = placed(rows).requires_grad_(), w.to(dev()).requires_grad_()
        out = unsort_tokens(rs, order, ws)
        results.append([got, *order, out.detach(), *torch.autograd.grad(out, (rs, ws), grad)])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
