"""GPU parity of tokens sorted by expert and back (afd_sort_tokens, afd_unsort_tokens, afd_unsort_grad) and their gradients.

Positions, counts and moved rows are exact. Sums over a token's pairs and over a row's columns against 64 bits, within what
their fp32 additions and the result's type may be off (``error_bounds``)."""

import pytest
import torch

from error_bounds import Bounded
from gpu_util import dev, say
from sgl_asap_amd.moe.sort import TokenOrder, sort_tokens, unsort_tokens

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def order_of(ids, experts, lo=0):
    """(positions, counts, offsets) on the CPU, by a stable sort."""
    key = ids.long().reshape(-1) - lo
    here = (key >= 0) & (key < experts)
    key = torch.where(here, key, experts)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel())
    place[~here] = -1
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])
    return place.view(ids.shape).int(), counts.int(), offsets.int()


def moved(x, place):
    out = torch.zeros(place.numel(), x.shape[1], dtype=x.dtype)
    here = place.reshape(-1) >= 0
    out[place.reshape(-1)[here].long()] = x.repeat_interleave(place.shape[1], 0)[here]
    return out


def make(n, hidden, experts, k, dtype, seed, kind="random"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, hidden, generator=g).to(dtype)
    rows = torch.randn(n * k, hidden, generator=g).to(dtype)
    w = torch.rand(n, k, generator=g)
    if kind == "one":
        ids = torch.full((n, k), experts // 2)
    elif kind == "none":
        ids = torch.full((n, k), -1)
    else:
        ids = torch.randint(0, experts, (n, k), generator=g)
    return x, rows, w, ids.int()


def check_order(order, want):
    for got, exp in zip(order, want):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), exp)


# few pairs (up to 4096) go in one launch, more in three; past 262144 a chunk has 2048
SIZES = [(1, 1, 1, 1), (1, 8, 4, 2), (3, 33, 1024, 32), (8, 4096, 256, 8), (127, 130, 60, 4), (512, 64, 64, 8), (4096, 8, 7, 1),
         (513, 72, 64, 8), (1531, 100, 60, 4), (2048, 16, 1000, 5), (700, 24, 1024, 32), (9000, 8, 33, 32), (40000, 9, 256, 8),
         (70001, 2, 3, 7)]


@pytest.mark.parametrize("n,hidden,experts,k", SIZES)
def test_order_and_rows(n, hidden, experts, k):
    x, _, _, ids = make(n, hidden, experts, k, torch.bfloat16, n + k)
    say(f"sort n={n} hidden={hidden} experts={experts} k={k}")
    for lo, here in ((0, experts), (experts // 3, max(1, experts // 2)), (experts - 1, 8)):
        want = order_of(ids, here, lo)
        rows, order = sort_tokens(x.to(dev()), ids.to(dev()), here, expert_lo=lo)
        check_order(order, want)
        assert rows.shape == (n * k, hidden) and torch.equal(rows.cpu(), moved(x, want[0]))


@pytest.mark.parametrize("kind", ["one", "none"])
@pytest.mark.parametrize("n", [5, 300, 3000])
def test_one_expert_has_all_or_none_any(kind, n):
    x, rows, w, ids = make(n, 40, 16, 4, torch.float32, n, kind)
    say(f"sort {kind} n={n}")
    want = order_of(ids, 16)
    got, order = sort_tokens(x.to(dev()), ids.to(dev()), 16)
    check_order(order, want)
    assert torch.equal(got.cpu(), moved(x, want[0]))
    out = unsort_tokens(rows.to(dev()), order, w.to(dev())).cpu()
    assert (out == 0).all() if kind == "none" else (out != 0).any(1).all()


@pytest.mark.parametrize("n", [60, 2000])
def test_ids_of_any_value_and_not_finite_rows(n):
    """Ids outside the rank's are nowhere, whatever they are; a token without pairs gets 0 whatever its weights and the rows
    past the last hold."""
    x, rows, w, ids = make(n, 24, 10, 4, torch.float32, 3)
    odd = torch.tensor([-1, 10, 2**31 - 1, -(2**31)], dtype=torch.int32)
    ids[::3] = odd
    ids[1::3, 1] = odd[2]
    w[::3] = float("nan")
    want = order_of(ids, 10)
    used = int(want[2][-1])
    rows[used:] = float("inf")
    say(f"odd ids n={n}")
    got, order = sort_tokens(x.to(dev()), ids.to(dev()), 10)
    check_order(order, want)
    assert torch.equal(got.cpu(), moved(x, want[0]))
    out = unsort_tokens(rows.to(dev()), order, w.to(dev())).cpu()
    assert (out[::3] == 0).all() and out.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,hidden,k", [(7, 1, 3), (30, 257, 5), (30, 256, 8), (900, 1000, 4), (1500, 2048, 8), (1200, 131, 17),
                                        (5, 9000, 2), (1100, 4104, 3)])
def test_back_and_gradients(dtype, n, hidden, k):
    experts = 12
    x, rows, w, ids = make(n, hidden, experts, k, dtype, n + hidden)
    ids[::4, 0] = -1
    if n > 5:
        ids[5] = -1
    g = torch.Generator().manual_seed(1)
    g_rows, g_out = torch.randn(n * k, hidden, generator=g).to(dtype), torch.randn(n, hidden, generator=g).to(dtype)
    place, counts, offsets = order_of(ids, experts)
    here, at = place >= 0, place.clamp_min(0).long()
    say(f"back {dtype} n={n} hidden={hidden} k={k}")
    xd, rd, wd = (t.to(dev()).requires_grad_() for t in (x, rows, w))
    got, order = sort_tokens(xd, ids.to(dev()), experts)
    out = unsort_tokens(rd, order, wd)
    assert out.dtype == dtype
    dx, dr, dw = torch.autograd.grad((got, out), (xd, rd, wd), (g_rows.to(dev()), g_out.to(dev())))
    check_order(order, (place, counts, offsets))
    mask = Bounded(here[..., None])
    assert (Bounded(rows[at]) * Bounded(w[..., None]) * mask).sum(1).held(dtype).holds(out.detach())
    assert (Bounded(g_rows[at]) * mask).sum(1).held(dtype).holds(dx)
    want = torch.zeros(n * k, hidden, dtype=torch.float64)
    want[at[here]] = (w.double()[..., None] * g_out.double()[:, None])[here]
    assert Bounded(want).rounded().held(dtype).holds(dr)
    assert (dr.cpu()[int(offsets[-1]) :] == 0).all()
    assert ((Bounded(rows[at]) * Bounded(g_out[:, None])).sum(-1) * Bounded(here)).held(torch.float32).holds(dw)
    assert (dw.cpu()[~here] == 0).all()
    # one gradient alone is the same
    only = torch.autograd.grad(unsort_tokens(rd, order, w.to(dev())), rd, g_out.to(dev()))[0]
    assert torch.equal(only, dr)
    only = torch.autograd.grad(unsort_tokens(rows.to(dev()), order, wd), wd, g_out.to(dev()))[0]
    assert torch.equal(only, dw)
    # without weights
    plain = unsort_tokens(rd, order)
    assert (Bounded(rows[at]) * mask).sum(1).held(dtype).holds(plain.detach())
    d_plain = torch.autograd.grad(plain, rd, g_out.to(dev()))[0].cpu()
    ones = torch.zeros(n * k, hidden, dtype=dtype)
    ones[at[here]] = g_out[:, None].expand(n, k, hidden)[here]
    assert torch.equal(d_plain, ones)


def test_gradient_against_differences():
    """Out is linear in the rows and in the weights: a difference is the derivative but for its roundings."""
    n, hidden, k = 20, 64, 3
    x, rows, w, ids = make(n, hidden, 6, k, torch.float32, 8)
    g = torch.randn(n, hidden, generator=torch.Generator().manual_seed(2))
    rd, wd = rows.to(dev()).requires_grad_(), w.to(dev()).requires_grad_()
    say("differences")
    _, order = sort_tokens(x.to(dev()), ids.to(dev()), 6)
    dr, dw = torch.autograd.grad(unsort_tokens(rd, order, wd), (rd, wd), g.to(dev()))
    base = unsort_tokens(rd, order, wd).detach().double().cpu()
    # out's entries are below 16: each is off by less than 4 x 16 x 2^-24, a sum of 64 of them times |g| < 5 by 2^-9
    for t, j in ((0, 0), (7, 2), (19, 1)):
        w2 = w.clone()
        w2[t, j] += 1.0
        d = ((unsort_tokens(rd, order, w2.to(dev())).detach().double().cpu() - base) * g).sum()
        assert abs(float(d) - float(dw[t, j])) <= 2.0**-9
    for r, c in ((0, 0), (30, 5), (59, 63)):
        r2 = rows.clone()
        r2[r, c] += 1.0
        d = ((unsort_tokens(r2.to(dev()), order, wd).detach().double().cpu() - base) * g).sum()
        assert abs(float(d) - float(dr[r, c])) <= 2.0**-9


@pytest.mark.parametrize("n", [40, 2000])
@pytest.mark.parametrize("dtype,hidden", [(torch.bfloat16, 64), (torch.bfloat16, 33), (torch.float32, 17), (torch.float16, 34)])
def test_strides_and_given_rows(n, dtype, hidden):
    """x and rows with strides and offsets, rows into a larger buffer: what lies beside and behind them stays."""
    k, experts = 4, 9
    x, rows, w, ids = make(n, hidden, experts, k, dtype, 4)
    ids[::2, 1] = 99
    want = order_of(ids, experts)
    used = int(want[2][-1])
    say(f"strides {dtype} hidden={hidden} n={n}")
    for left in (3, 8):
        xw = torch.full((n, hidden + 24), 5.0, dtype=dtype, device=dev())
        xw[:, left : left + hidden] = x.to(dev())
        buf = torch.full((n * k + 5, hidden + 16), 7.0, dtype=dtype, device=dev())
        out = buf[:, left : left + hidden]
        got, order = sort_tokens(xw[:, left : left + hidden], ids.to(dev()), experts, out=out)
        assert got is out
        check_order(order, want)
        assert torch.equal(got[:used].cpu(), moved(x, want[0])[:used])
        buf[:used, left : left + hidden] = 7.0
        assert (buf == 7.0).all()
        buf[: n * k, left : left + hidden] = rows.to(dev())
        a = unsort_tokens(out, order, w.to(dev()))
        b = unsort_tokens(rows.to(dev()), order, w.to(dev()))
        assert torch.equal(a, b)
        grads = [torch.autograd.grad(unsort_tokens(r, order, v), (r, v), a)
                 for r, v in (((buf[: n * k, left : left + hidden].detach().requires_grad_()), w.to(dev()).requires_grad_()),
                              (rows.to(dev()).requires_grad_(), w.to(dev()).requires_grad_()))]
        assert torch.equal(grads[0][0], grads[1][0])
        # rows of another alignment are added up in another order: each sum of `hidden` products is within its own bound
        at = want[0].clamp_min(0).long()
        d_w = ((Bounded(rows[at]) * Bounded(a.cpu()[:, None])).sum(-1) * Bounded(want[0] >= 0)).held(torch.float32)
        assert d_w.holds(grads[0][1]) and d_w.holds(grads[1][1])
    t = x.to(dev()).t().contiguous().t()
    assert torch.equal(sort_tokens(t, ids.to(dev()).t().contiguous().t(), experts)[0].cpu(), moved(x, want[0]))
    same = x[:1].to(dev()).expand(n, hidden)
    assert torch.equal(sort_tokens(same, ids.to(dev()), experts)[0].cpu(), moved(x[:1].expand(n, hidden), want[0]))


def test_weights_of_other_types_and_a_gradient_without_strides():
    n, hidden, k = 50, 40, 3
    x, rows, w, ids = make(n, hidden, 8, k, torch.bfloat16, 5)
    say("weights of other types")
    _, order = sort_tokens(x.to(dev()), ids.to(dev()), 8)
    half = w.to(torch.bfloat16).to(dev()).requires_grad_()
    rd = rows.to(dev()).requires_grad_()
    out = unsort_tokens(rd, order, half)
    assert torch.equal(out, unsort_tokens(rd, order, half.float()))
    out.sum().backward()  # the incoming gradient has strides 0
    assert half.grad.dtype == torch.bfloat16
    wide = w.to(torch.bfloat16).float().to(dev()).requires_grad_()
    r2 = rows.to(dev()).requires_grad_()
    unsort_tokens(r2, order, wide).backward(torch.ones(n, hidden, dtype=torch.bfloat16, device=dev()))
    assert torch.equal(rd.grad, r2.grad) and torch.equal(half.grad, wide.grad.to(torch.bfloat16))
    # weights of a row that was broadcast
    row = w[:1].to(dev()).requires_grad_()
    unsort_tokens(rows.to(dev()), order, row.expand(n, k)).sum().backward()
    full = w[:1].expand(n, k).contiguous().to(dev()).requires_grad_()
    unsort_tokens(rows.to(dev()), order, full).sum().backward()
    assert torch.allclose(row.grad, full.grad.sum(0, keepdim=True))
    x2 = x.to(dev()).requires_grad_()
    sort_tokens(x2, ids.to(dev()), 8)[0].sum().backward()
    assert torch.equal(x2.grad, torch.full_like(x2, float(k)))


def test_no_tokens():
    say("no tokens")
    x = torch.zeros(0, 16, dtype=torch.bfloat16, device=dev(), requires_grad=True)
    ids = torch.zeros(0, 4, dtype=torch.int32, device=dev())
    rows, order = sort_tokens(x, ids, 5)
    assert rows.shape == (0, 16) and order.positions.shape == (0, 4)
    assert (order.counts == 0).all() and (order.offsets == 0).all() and order.offsets.shape == (6,)
    w = torch.zeros(0, 4, device=dev(), requires_grad=True)
    more = torch.ones(3, 16, dtype=torch.bfloat16, device=dev(), requires_grad=True)
    out = unsort_tokens(more, order, w)
    assert out.shape == (0, 16)
    out.sum().backward()
    assert (more.grad == 0).all() and w.grad.shape == (0, 4)
    sort_tokens(x, ids, 5)[0].sum().backward()
    assert x.grad.shape == (0, 16)


def test_rows_that_are_fewer_or_more_than_the_pairs():
    n, hidden, k = 40, 24, 4
    x, rows, w, ids = make(n, hidden, 8, k, torch.float32, 5)
    ids[:, 2:] = -1
    say("fewer, more rows")
    _, order = sort_tokens(x.to(dev()), ids.to(dev()), 8)
    used = int(order.offsets[-1])
    want = unsort_tokens(rows.to(dev()), order, w.to(dev()))
    for size in (used, n * k + 300):
        r = torch.full((size, hidden), float("nan"), device=dev())
        r[:used] = rows[:used].to(dev())
        r.requires_grad_()
        out = unsort_tokens(r, order, w.to(dev()))
        assert torch.equal(out, want)
        out.sum().backward()
        assert r.grad.isfinite().all() and (r.grad[used:] == 0).all() and (r.grad[:used] != 0).all()
    # positions past the rows that there are, are skipped
    cut = unsort_tokens(rows[:10].to(dev()), order, w.to(dev()))
    kept = torch.where(order.positions < 10, order.positions, torch.full_like(order.positions, -1))
    assert torch.equal(cut, unsort_tokens(rows.to(dev()), TokenOrder(kept, order.counts, order.offsets), w.to(dev())))


def test_derivatives_that_are_refused():
    x, rows, w, ids = make(10, 16, 4, 2, torch.float32, 1)
    say("second derivatives")
    xd, rd, wd = (t.to(dev()).requires_grad_() for t in (x, rows, w))
    got, order = sort_tokens(xd, ids.to(dev()), 4)
    out = unsort_tokens(rd, order, wd)
    for y, leaf in ((got, xd), (out, rd), (out, wd)):
        (d,) = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="no second"):
            d.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.to(dev()), torch.ones_like(x).to(dev()))
        with pytest.raises(NotImplementedError):
            sort_tokens(dual, ids.to(dev()), 4)
        dual = torch.autograd.forward_ad.make_dual(rows.to(dev()), torch.ones_like(rows).to(dev()))
        with pytest.raises(NotImplementedError):
            unsort_tokens(dual, order)
    # counts that are added up over ranks before the backward leave it as it is; positions that changed do not pass
    order.counts.add_(5)
    out.sum().backward(retain_graph=True)
    order.positions.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_refusals_of_calls():
    x, rows, w, ids = (t.to(dev()) for t in make(10, 16, 4, 2, torch.float32, 1))
    say("refusals")
    buf = torch.zeros(40, 16, device=dev())
    for bad in (buf[:19], buf[:, :15], buf.to(torch.bfloat16), buf[None], torch.zeros(40, 16), buf.t().contiguous().t(),
                torch.zeros(1, 16, device=dev()).expand(40, 16)):
        with pytest.raises(ValueError):
            sort_tokens(x, ids, 4, out=bad)
    for src, out in ((buf[:10], buf), (buf[30:40], buf[:39]), (buf[5:15], buf[10:35])):
        with pytest.raises(ValueError, match="memory"):
            sort_tokens(src, ids, 4, out=out)
    assert sort_tokens(buf[:10], ids, 4, out=buf[10:])[0].shape == (30, 16)
    with pytest.raises(NotImplementedError):
        sort_tokens(x.clone().requires_grad_(), ids, 4, out=buf)
    with pytest.raises(ValueError):
        sort_tokens(x, ids.cpu(), 4)
    with pytest.raises(ValueError):
        sort_tokens(x, ids, 4, expert_lo=-1)
    _, order = sort_tokens(x, ids, 4)
    with pytest.raises(ValueError):
        unsort_tokens(rows, order, w.cpu())
    with pytest.raises(ValueError):
        unsort_tokens(rows, order, w[:, :1])
    with pytest.raises(ValueError):
        unsort_tokens(rows, TokenOrder(order.positions.cpu(), order.counts, order.offsets), w)
    with pytest.raises(ValueError):
        unsort_tokens(rows, TokenOrder(order.positions, order.counts, order.offsets[:0]), w)


@pytest.mark.parametrize("n", [30, 3000])
def test_captured_and_replayed(n):
    """Forward and backward in a graph, replayed with other tokens beside eager calls."""
    hidden, k, experts = 64, 4, 20
    x, rows, w, ids = (t.to(dev()) for t in make(n, hidden, experts, k, torch.bfloat16, 2))
    say(f"captured n={n}")

    def step():
        xs, rs, ws = (t.detach().requires_grad_() for t in (x, rows, w))
        got, order = sort_tokens(xs, ids, experts)
        out = unsort_tokens(rs, order, ws)
        return (got, *order, out) + torch.autograd.grad((got, out), (xs, rs, ws), (got, out))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(3):
        for t, new in zip((x, rows, w, ids), make(n, hidden, experts, k, torch.bfloat16, 10 + i)):
            t.copy_(new.to(dev()))
        ids[::5, 0] = -1
        for graph, _ in graphs:
            graph.replay()
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def test_streams():
    say("streams")
    data = [[t.to(dev()) for t in make(600 + 50 * i, 72, 30, 8, torch.bfloat16, i)] for i in range(3)]
    want = [sort_tokens(x, ids, 30) for x, _, _, ids in data]
    back = [unsort_tokens(rows, order, w) for (_, rows, w, _), (_, order) in zip(data, want)]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in data]
    got = []
    for _ in range(10):
        for st, (x, rows, w, ids) in zip(side, data):
            with torch.cuda.stream(st):
                r, order = sort_tokens(x, ids, 30)
                got.append((r, order, unsort_tokens(rows, order, w)))
    torch.cuda.synchronize()
    for i, (r, order, out) in enumerate(got):
        assert torch.equal(r, want[i % 3][0]) and torch.equal(out, back[i % 3])
        assert all(torch.equal(a, b) for a, b in zip(order, want[i % 3][1]))


def test_rows_past_32_bits():
    """Sorted rows past 2^32 bytes and 2^31 elements, both ways."""
    n, hidden, k, experts = 70000, 4096, 8, 5
    say("560000 rows of 4096")
    g = torch.Generator(device=dev()).manual_seed(0)
    x = torch.randn(n, hidden, generator=g, device=dev(), dtype=torch.bfloat16)
    ids = torch.randint(0, experts, (n, k), generator=g, device=dev(), dtype=torch.int32)
    x.requires_grad_()
    rows, order = sort_tokens(x, ids, experts)
    check_order(order, order_of(ids.cpu(), experts))
    flat = order.positions.reshape(-1).long()
    for t in (0, 1, 30000, n - 1):
        for j in (0, k - 1):
            assert torch.equal(rows[flat[t * k + j]], x[t])
    w = torch.full((n, k), 1.0 / k, device=dev(), requires_grad=True)
    out = unsort_tokens(rows, order, w)
    # eight equal rows an eighth each: every product and sum is exact
    assert torch.equal(out, x)
    d_w, d_x = torch.autograd.grad(out, (w, x), x.detach())
    assert torch.equal(d_x, x)  # 8 x / 8
    mass = (x.detach().float() ** 2).sum(-1, keepdim=True)
    assert ((d_w - mass).abs() <= hidden * 2.0**-23 * mass).all()
