"""GPU: orders that a program made of sort_tokens' own (tokens dropped past a capacity, a part of the tokens) and their
gradients."""

import copy
import pickle

import pytest
import torch
from torch.utils import _pytree as pytree

from error_bounds import Bounded
from gpu_util import dev, say
from sgl_asap_amd.moe.sort import TokenOrder, sort_tokens, unsort_tokens

pytestmark = pytest.mark.gpu


def make(n, hidden, experts, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, hidden, generator=g).to(dtype), torch.randn(n * k, hidden, generator=g).to(dtype),
            torch.rand(n, k, generator=g), torch.randint(0, experts, (n, k), generator=g).int(),
            torch.randn(n, hidden, generator=g).to(dtype))


def old_memory(*shapes):
    """Freed blocks of these sizes that hold NaN: what a call's new tensors may be made of."""
    for shape, dtype in shapes:
        torch.full(shape, float("nan"), dtype=dtype, device=dev())


def check(rows, w, order, g, d_rows, d_w):
    """Both gradients against the formula over the positions as they are, the rows that no pair names 0."""
    place = order.positions.cpu()
    here, at = place >= 0, place.clamp_min(0).long()
    want = torch.zeros(rows.shape, dtype=torch.float64)
    want[at[here]] = (w.double()[..., None] * g.double()[:, None])[here]
    assert Bounded(want).rounded().held(rows.dtype).holds(d_rows)
    idle = torch.ones(rows.shape[0], dtype=torch.bool)
    idle[at[here]] = False
    assert idle.any() and (d_rows.cpu()[idle] == 0).all()
    assert ((Bounded(rows[at]) * Bounded(g[:, None])).sum(-1) * Bounded(here)).held(torch.float32).holds(d_w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,hidden,k", [(40, 24, 4), (1500, 136, 3), (30, 33, 2)])
@pytest.mark.parametrize("kind", ["dropped", "in place", "part", "one token"])
def test_gradients_of_edited_orders(dtype, n, hidden, k, kind):
    x, rows, w, ids, g = make(n, hidden, 8, k, dtype, n)
    say(f"order {kind} {dtype} n={n} hidden={hidden} k={k}")
    _, order = sort_tokens(x.to(dev()), ids.to(dev()), 8)
    drop = torch.rand(n, k, generator=torch.Generator().manual_seed(1)).to(dev()) < 0.3
    if kind == "dropped":
        order = TokenOrder(order.positions.masked_fill(drop, -1), order.counts, order.offsets)
    elif kind == "in place":
        order.positions.masked_fill_(drop, -1)
    elif kind == "part":
        a, b = n // 4, n // 2
        order, w, g = order._replace(positions=order.positions[a:b]), w[a:b], g[a:b]
    else:
        order, w, g = order._replace(positions=order.positions[3:4]), w[3:4], g[3:4]
    rd, wd = rows.to(dev()).requires_grad_(), w.to(dev()).requires_grad_()
    out = unsort_tokens(rd, order, wd)
    old_memory((rows.shape, dtype), (w.shape, torch.float32))
    check(rows, w, order, g, *torch.autograd.grad(out, (rd, wd), g.to(dev())))


def test_rows_that_an_edited_order_names_past_the_last():
    """Positions decide, not offsets: rows from offsets[-1] on have a gradient where a pair names them."""
    x, rows, w, ids, g = make(30, 40, 6, 2, torch.float32, 3)
    say("offsets of another order")
    _, order = sort_tokens(x.to(dev()), ids.to(dev()), 6)
    order = TokenOrder(order.positions.masked_fill(torch.arange(60, device=dev()).view(30, 2) % 3 == 0, -1), order.counts,
                       torch.zeros_like(order.offsets))
    rd, wd = rows.to(dev()).requires_grad_(), w.to(dev()).requires_grad_()
    out = unsort_tokens(rd, order, wd)
    old_memory((rows.shape, rows.dtype))
    check(rows, w, order, g, *torch.autograd.grad(out, (rd, wd), g.to(dev())))


def test_copies_of_orders():
    x, rows, w, ids, g = make(30, 40, 6, 2, torch.float32, 4)
    say("copies of orders")
    _, order = sort_tokens(x.to(dev()), ids.to(dev()), 6)
    order.positions[::2] = -1  # a copy does not look like new
    clones = [pytree.tree_map(torch.clone, order), type(order)(*(t.clone() for t in order)), order._make(t.clone() for t in order)]
    for other in [copy.copy(order), copy.deepcopy(order), pickle.loads(pickle.dumps(order)), TokenOrder(*order)] + clones:
        assert isinstance(other, TokenOrder) and all(torch.equal(a, b) for a, b in zip(other, order))
        rd, wd = rows.to(dev()).requires_grad_(), w.to(dev()).requires_grad_()
        out = unsort_tokens(rd, other, wd)
        old_memory((rows.shape, rows.dtype))
        check(rows, w, other, g, *torch.autograd.grad(out, (rd, wd), g.to(dev())))


def test_parts_of_an_order_by_its_own_type():
    """Slices share the whole's version: they are not taken for all of it."""
    x, rows, w, ids, g = make(30, 40, 6, 2, torch.float32, 6)
    say("parts of an order")
    _, order = sort_tokens(x.to(dev()), ids.to(dev()), 6)
    parts = [pytree.tree_map(lambda t: t[4:20] if t.dim() == 2 else t, order), type(order)(order.positions[4:20], *order[1:])]
    for part in parts:
        rd, wd = rows.to(dev()).requires_grad_(), w[4:20].to(dev()).requires_grad_()
        out = unsort_tokens(rd, part, wd)
        old_memory((rows.shape, rows.dtype))
        check(rows, w[4:20], part, g[4:20], *torch.autograd.grad(out, (rd, wd), g[4:20].to(dev())))


def test_an_order_of_sort_tokens_is_known_to_be_complete():
    """Its rows' gradient is written once, without being cleared first, with a gradient by x or not."""
    x, rows, w, ids, g = (t.to(dev()) for t in make(30, 40, 6, 2, torch.float32, 7))
    say("complete orders")
    for data in (x, x.clone().requires_grad_()):
        _, order = sort_tokens(data, ids, 6)
        assert order.complete()
        order.counts.add_(1)
        assert order.complete()
        assert not order._replace(positions=order.positions[:5]).__class__ is type(order)
        order.offsets.add_(0)
        assert not order.complete()
    with torch.inference_mode():
        assert not sort_tokens(x.clone(), ids.clone(), 6)[1].complete()


def test_edited_order_captured_and_replayed():
    n, hidden, k = 200, 64, 3
    x, rows, w, ids, g = (t.to(dev()) for t in make(n, hidden, 8, k, torch.bfloat16, 5))
    capacity = 40
    say("edited order captured")

    def step():
        rs, ws = rows.detach().requires_grad_(), w.detach().requires_grad_()
        _, order = sort_tokens(x, ids, 8)
        e = ids.long().clamp_min(0)
        late = order.positions - order.offsets[e] >= capacity
        out = unsort_tokens(rs, order._replace(positions=order.positions.masked_fill(late, -1)), ws)
        return (out,) + torch.autograd.grad(out, (rs, ws), g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        for t, new in zip((x, rows, w, ids, g), make(n, hidden, 8, k, torch.bfloat16, 20 + i)):
            t.copy_(new.to(dev()))
        graph.replay()
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i
        assert (outs[1] == 0).all(1).any() and outs[1].isfinite().all()
