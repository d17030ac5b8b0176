"""GPU parity of the router: the choice of experts (exact, ties and borders included), its weights,
counts, the balance loss, and the gradients, against 64-bit definitions and against differences.

Tolerances. A score's relative error in fp32: the exponent's argument |x| <= 32 is rounded to
|x| 2^-24, the exponential and the logarithm add 2 ulps each, a sum of up to 1024 terms as a tree of
depth 10 ten half ulps, the quotient one: below 64 * 2^-24 = 2^-18. The weights carry that. A gradient is a
difference of such terms, no larger than twice the largest incoming gradient times the scale:
2^-16 of that bound, absolute, plus half a step of bf16 (eps / 2 = 2^-8, relative) where the logits
are bf16. The loss sums shares with error 2^-18 in fp32 blocks: 2^-16."""

import math

import pytest
import torch

import router_ref as R
from gpu_util import dev, say
from sgl_asap_amd.moe import balance as B
from sgl_asap_amd.moe import topk as T

pytestmark = pytest.mark.gpu

REL = 2.0**-18


def make(n, experts, seed, dtype=torch.float32, bias=False):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(n, experts, generator=g) * 2).to(dtype)
    b = torch.randn(experts, generator=g) * 0.05 if bias else None
    return logits, b


def check_choice(logits, top_k, out, scoring, bias=None, renorm=True, scale=1.0, groups=0, keep=0, valid=None):
    z = R.canon(logits)
    ids = R.choose(z, top_k, scoring, bias, groups, keep)
    w = R.weights(z, ids, scoring, renorm, scale)
    if valid is not None:
        ids = ids.masked_fill(~valid[:, None], -1)
        w = w.masked_fill(~valid[:, None], 0.0)
    assert out.topk_ids.dtype == torch.int32 and out.topk_weights.dtype == torch.float32
    assert torch.equal(out.topk_ids.cpu().long(), ids)
    got = out.topk_weights.cpu().double()
    assert torch.isfinite(got).all()
    assert ((got - w).abs() <= REL * w.abs() + 1e-37).all(), ((got - w).abs() / w.abs().clamp_min(1e-37)).max()
    return ids


def select(logits, top_k, bias=None, valid=None, groups=0, keep=0, scale=1.0, **more):
    return T.select_experts(logits.to(dev()), top_k, correction_bias=None if bias is None else bias.to(dev()),
                            valid=None if valid is None else valid.to(dev()), num_expert_group=groups or None,
                            topk_group=keep or None, routed_scaling_factor=scale, **more)


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,experts,top_k,groups,keep", [
    (1, 1, 1, 0, 0), (5, 8, 2, 0, 0), (33, 60, 4, 0, 0), (17, 64, 16, 0, 0), (9, 64, 20, 0, 0), (130, 128, 6, 8, 3),
    (67, 129, 8, 3, 1), (257, 256, 8, 8, 4), (12, 256, 32, 1, 1), (19, 384, 8, 64, 5), (31, 512, 8, 0, 0),
    (7, 1000, 32, 40, 39), (3, 1024, 32, 16, 2), (6, 32, 32, 0, 0), (4, 48, 3, 48, 3), (5, 63, 9, 9, 2),
    (11, 160, 6, 8, 3), (9, 320, 8, 10, 4), (21, 96, 6, 2, 1), (6, 64, 8, 32, 7), (13, 768, 12, 6, 2), (8, 16, 4, 16, 5),
])
def test_choice(n, experts, top_k, groups, keep, bias, scoring):
    for dtype in (torch.float32, torch.bfloat16):
        logits, b = make(n, experts, n + experts, dtype, bias)
        for renorm, scale in ((True, 2.5), (False, 1.0)):
            say(f"choice n={n} E={experts} k={top_k} groups={groups}/{keep} {scoring} bias={bias} {dtype} renorm={renorm}")
            out = select(logits, top_k, b, scoring=scoring, renormalize=renorm, groups=groups, keep=keep, scale=scale)
            check_choice(logits, top_k, out, scoring, b, renorm, scale, groups, keep)


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("bias", [False, True])
def test_choice_ties_go_to_the_lower_index(bias, scoring):
    """Few distinct values, both zeros among them, and a bias of few steps."""
    g = torch.Generator().manual_seed(3)
    logits = torch.randint(-2, 2, (200, 72), generator=g).float() * torch.where(torch.rand(200, 72, generator=g) < 0.5, -1.0, 1.0)
    b = torch.randint(-1, 2, (72,), generator=g).float() * 0.25 if bias else None
    for groups, keep in ((0, 0), (8, 3)):
        say(f"ties {scoring} bias={bias} groups={groups}")
        check_choice(logits, 8, select(logits, 8, b, scoring=scoring, groups=groups, keep=keep), scoring, b, groups=groups, keep=keep)


@pytest.mark.parametrize("scoring", R.SCORINGS)
def test_choice_between_close_scores(scoring):
    """Biases that make pairs of choice values differ by 1e-12: beyond 32 bits, within 64."""
    g = torch.Generator().manual_seed(5)
    n, experts = 64, 128
    logits = torch.randn(n, experts, generator=g)
    logits[:, 64:] = logits[:, :64]
    bias = torch.zeros(experts)
    # fp32 steps near 2^-40 on top of 0: the sums' 52 bits hold them, 24 bits do not
    bias[:64] = torch.where(torch.rand(64, generator=g) < 0.5, 0.0, 2.0**-40)
    bias[64:] = torch.where(torch.rand(64, generator=g) < 0.5, 0.0, 2.0**-40)
    say(f"close scores {scoring}")
    check_choice(logits, 16, select(logits, 16, bias, scoring=scoring), scoring, bias)


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_choice_of_infinite_and_masked_logits(dtype, bias, scoring):
    logits, b = make(12, 40, 11, dtype, bias)
    low, inf = torch.finfo(dtype).min, math.inf
    logits[0] = -inf
    logits[1] = low
    logits[2, 3:] = -inf
    logits[3, 5:] = low
    logits[4, 7] = math.nan
    logits[5] = math.nan
    logits[6, 9] = inf
    logits[7, [4, 30]] = inf
    logits[8] = inf
    logits[9, ::2] = low
    logits[10] = 0.0
    if bias:
        b[6], b[7], b[8] = math.nan, inf, -inf
    for renorm in (True, False):
        for groups, keep in ((0, 0), (10, 2)):
            say(f"masked {dtype} {scoring} bias={bias} renorm={renorm} groups={groups}")
            out = select(logits, 6, b, scoring=scoring, renormalize=renorm, groups=groups, keep=keep)
            check_choice(logits, 6, out, scoring, b, renorm, groups=groups, keep=keep)


def test_choice_of_padded_rows_and_strided_logits():
    logits, b = make(50, 96, 21, torch.float32, True)
    valid = torch.rand(50, generator=torch.Generator().manual_seed(1)) < 0.6
    wide = torch.full((50, 131), 99.0)
    wide[:, 17:113] = logits
    on = wide.to(dev())
    say("padded rows, rows with a stride, rows off alignment")
    out = T.select_experts(on[:, 17:113], 6, correction_bias=b.to(dev()), valid=valid.to(dev()), scoring="sigmoid")
    check_choice(logits, 6, out, "sigmoid", b, valid=valid)
    say("columns with a stride, one row repeated")
    check_choice(logits, 6, T.select_experts(on.t().contiguous().t()[:, 17:113], 6), "softmax")
    row = logits[:1].expand(9, 96)
    check_choice(row, 6, T.select_experts(row[:1].to(dev()).expand(9, 96), 6), "softmax")
    say("no rows")
    none = T.select_experts(on[:0, :96], 6)
    assert none.topk_ids.shape == (0, 6) and none.topk_weights.shape == (0, 6)


CU = {"all": None, "one": [0, 41], "parts": [0, 7, 7, 30, 41], "inner": [3, 9, 10, 38], "none": [5, 5, 5]}


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("spans", sorted(CU))
@pytest.mark.parametrize("experts,top_k", [(8, 2), (60, 4), (100, 17), (256, 8), (500, 8), (1024, 32)])
def test_balance_loss_counts_and_gradient(experts, top_k, spans, scoring):
    n, cu, alpha = 41, CU[spans], 0.01
    for dtype in (torch.float32, torch.bfloat16):
        logits, _ = make(n, experts, experts + top_k, dtype)
        g = torch.Generator().manual_seed(experts)
        ids = torch.randint(-1, experts + 1, (n, top_k), generator=g, dtype=torch.int32)  # repeated and foreign ones
        valid = torch.rand(n, generator=g) < 0.8 if spans != "one" else None
        say(f"balance E={experts} k={top_k} {spans} {scoring} {dtype}")
        leaf = logits.to(dev()).requires_grad_()
        loss, cnt = B.balance_loss(leaf, ids.to(dev()), alpha=alpha, scoring=scoring,
                                   cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev()),
                                   valid=None if valid is None else valid.to(dev()))
        (3.0 * loss).backward()
        z = R.canon(logits)
        want_cnt = R.counts(ids, experts, cu, valid)
        assert torch.equal(cnt.cpu().long().view(-1, experts), want_cnt)
        only = B.expert_counts(ids.to(dev()), experts, None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev()),
                               None if valid is None else valid.to(dev()))
        assert torch.equal(only, cnt)
        want = float(R.balance(z, ids, scoring, alpha, cu, valid))
        assert abs(float(loss.detach()) - want) <= 2.0**-16 * abs(want)
        grad = R.grads(logits, ids, scoring, gl=3.0, alpha=alpha, cu=cu, valid=valid)
        # the largest c_e: 3 alpha E cnt / (S' k T^2)
        most = 0.0
        used = sum(hi > lo for lo, hi in R.sequences(n, cu))
        for i, (lo, hi) in enumerate(R.sequences(n, cu)):
            rows = hi - lo if valid is None else int(valid[lo:hi].sum())
            if rows:
                most = max(most, 3 * alpha * experts * float(want_cnt[i].max()) / (used * top_k * rows * rows) * 2)
        tol = 2.0**-16 * most + (2.0**-8 * grad.abs() if dtype == torch.bfloat16 else 0.0)
        assert leaf.grad.dtype == dtype
        assert ((leaf.grad.cpu().double() - grad).abs() <= tol).all()


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("experts,top_k,bias", [(6, 1, False), (60, 4, True), (128, 17, False), (256, 8, True), (900, 32, True)])
def test_gradients_of_weights_and_loss_together(experts, top_k, bias, renorm, scoring):
    n, scale, alpha, cu = 37, 1.5, 0.02, [2, 12, 12, 35]
    for dtype in (torch.float32, torch.bfloat16):
        logits, b = make(n, experts, experts + 7, dtype, bias)
        g = torch.Generator().manual_seed(experts + 1)
        gw = torch.randn(n, top_k, generator=g)
        valid = torch.rand(n, generator=g) < 0.8
        args = dict(scoring=scoring, renormalize=renorm, correction_bias=None if b is None else b.to(dev()),
                    routed_scaling_factor=scale, valid=valid.to(dev()))
        say(f"gradients E={experts} k={top_k} bias={bias} renorm={renorm} {scoring} {dtype}")
        leaf = logits.to(dev()).requires_grad_()
        out, loss, cnt = B.select_and_balance(leaf, top_k, alpha=alpha, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev()), **args)
        ids = check_choice(logits, top_k, out, scoring, b, renorm, scale, valid=valid)
        assert torch.equal(cnt.cpu().long(), R.counts(ids, experts, cu, valid))
        want = float(R.balance(R.canon(logits), ids, scoring, alpha, cu, valid))
        assert abs(float(loss.detach()) - want) <= 2.0**-16 * abs(want)
        picked = ids.clamp_min(0)
        bound = 2.0**-16 * scale * float(gw.abs().max())
        for parts in ("both", "weights", "loss"):
            lo, hi = parts != "loss", parts != "weights"
            outs, gs = [], []
            if lo:
                outs.append(out.topk_weights), gs.append(gw.to(dev()))
            if hi:
                outs.append(loss), gs.append(torch.tensor(2.0, device=dev()))
            (got,) = torch.autograd.grad(outs, (leaf,), gs, retain_graph=True)
            ref = R.grads(logits, picked, scoring, renorm, scale, gw if lo else None, 2.0 if hi else None, alpha, cu, valid)
            tol = (bound if lo else 0.0) + (2.0**-16 * 2 * alpha * experts if hi else 0.0)
            tol = tol + (2.0**-8 * ref.abs() if dtype == torch.bfloat16 else 0.0)
            assert ((got.cpu().double() - ref).abs() <= tol).all(), parts
            assert (got[~valid.to(dev())] == 0).all()
        # the selection alone has the same gradient
        alone = T.select_experts(leaf, top_k, **args)
        assert torch.equal(alone.topk_ids, out.topk_ids) and torch.equal(alone.topk_weights, out.topk_weights)
        (g1,) = torch.autograd.grad(alone.topk_weights, leaf, gw.to(dev()))
        (g2,) = torch.autograd.grad(out.topk_weights, leaf, gw.to(dev()))
        assert torch.equal(g1, g2)


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_against_differences(renorm, scoring):
    """The kernel's gradient against central differences of the 64-bit loss (step h = 1e-4: truncation
    below h^2 = 1e-8 of the derivatives' size, far below the gradient's own tolerance)."""
    n, experts, top_k, alpha = 5, 12, 3, 0.5
    logits, _ = make(n, experts, 40, torch.float32)
    g = torch.Generator().manual_seed(2)
    gw = torch.randn(n, top_k, generator=g)
    say(f"differences {scoring} renorm={renorm}")
    leaf = logits.to(dev()).requires_grad_()
    out, loss, _ = B.select_and_balance(leaf, top_k, alpha=alpha, scoring=scoring, renormalize=renorm)
    (got,) = torch.autograd.grad((out.topk_weights, loss), (leaf,), (gw.to(dev()), torch.ones((), device=dev())))
    z, ids, h = logits.double(), out.topk_ids.cpu().long(), 1e-4

    def value(at):
        w = R.weights(at, ids, scoring, renorm, 1.0)
        return float((w * gw.double()).sum() + R.balance(at, ids, scoring, alpha))

    for t in range(n):
        for e in range(experts):
            up, down = z.clone(), z.clone()
            up[t, e] += h
            down[t, e] -= h
            d = (value(up) - value(down)) / (2 * h)
            assert abs(float(got[t, e]) - d) <= 2.0**-16 * float(gw.abs().max()) + 1e-6, (t, e)


@pytest.mark.parametrize("scoring", R.SCORINGS)
def test_gradients_of_masked_logits_are_finite(scoring):
    logits, _ = make(8, 40, 9)
    low = torch.finfo(torch.float32).min
    logits[0] = -math.inf
    logits[1] = low
    logits[2, 6:] = -math.inf
    logits[3, 6:] = low
    logits[4, 5] = math.nan
    logits[5, 5] = math.inf
    logits[6] = -200.0
    for renorm in (True, False):
        say(f"masked gradients {scoring} renorm={renorm}")
        leaf = logits.to(dev()).requires_grad_()
        out, loss, _ = B.select_and_balance(leaf, 4, alpha=0.1, scoring=scoring, renormalize=renorm)
        (g,) = torch.autograd.grad((out.topk_weights, loss), (leaf,), (torch.ones(8, 4, device=dev()), torch.ones((), device=dev())))
        assert torch.isfinite(g).all() and math.isfinite(float(loss.detach()))
        assert (g[0] == 0).all() and (g[2, 6:] == 0).all() and float(g[4, 5]) == 0.0


def test_many_rows_sequences_and_repeated_calls():
    """Workgroups that hold several sequences and sequences over many workgroups; the same bits each time."""
    n, experts, top_k = 5000, 256, 8
    logits, _ = make(n, experts, 77, torch.bfloat16)
    g = torch.Generator().manual_seed(4)
    cu = torch.cat([torch.randint(0, n + 1, (59,), generator=g), torch.tensor([0, 3, 3, 3, n])]).sort().values.tolist()
    cu_dev = torch.tensor(cu, dtype=torch.int32, device=dev())
    say("5000 rows in 63 sequences")
    first = None
    for _ in range(3):
        leaf = logits.to(dev()).requires_grad_()
        out, loss, cnt = B.select_and_balance(leaf, top_k, alpha=1.0, scoring="sigmoid", cu_seqlens=cu_dev)
        (g1,) = torch.autograd.grad(loss, leaf)
        now = (out.topk_ids, out.topk_weights, loss.detach(), cnt, g1)
        if first is None:
            first = now
        assert all(torch.equal(a, b) for a, b in zip(first, now))
    ids = first[0].cpu().long()
    assert torch.equal(ids, R.choose(R.canon(logits), top_k, "sigmoid"))
    assert torch.equal(first[3].cpu().long(), R.counts(ids, experts, cu))
    want = float(R.balance(R.canon(logits), ids, "sigmoid", 1.0, cu))
    assert abs(float(first[2]) - want) <= 2.0**-16 * want
    ref = R.grads(logits, ids, "sigmoid", gl=1.0, alpha=1.0, cu=cu)
    assert ((g1.cpu().double() - ref).abs() <= 2.0**-8 * ref.abs() + 2.0**-16 * experts).all()


def test_captured_and_replayed_with_other_inputs():
    """Forward and backward in one graph, two graphs in turn, other inputs copied in, eager calls between."""
    n, experts, top_k = 300, 128, 6
    make_one = lambda seed: make(n, experts, seed)[0].to(dev())
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device=dev())
    gw = torch.randn(n, top_k, device=dev())
    one = torch.ones((), device=dev())

    def step(leaf):
        out, loss, cnt = B.select_and_balance(leaf, top_k, alpha=0.1, cu_seqlens=cu)
        (g,) = torch.autograd.grad((out.topk_weights, loss), (leaf,), (gw, one))
        return out.topk_ids, out.topk_weights, loss, cnt, B.expert_counts(out.topk_ids, experts), g

    say("capture")
    graphs = []
    for seed in (1, 2):
        leaf = make_one(seed).requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(leaf)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(leaf)
        graphs.append((graph, leaf, outs))
    for round_ in range(3):
        for i, (graph, leaf, outs) in enumerate(graphs):
            with torch.no_grad():
                leaf.copy_(make_one(10 * round_ + i))
            graph.replay()
            want = step(leaf.detach().clone().requires_grad_())
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), (round_, i)


def test_on_another_stream():
    logits, b = make(700, 256, 31, bias=True)
    on, bias = logits.to(dev()), b.to(dev())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    say("another stream")
    with torch.cuda.stream(side):
        out = T.select_experts(on, 8, scoring="sigmoid", correction_bias=bias)
        cnt = B.expert_counts(out.topk_ids, 256)
    side.synchronize()
    ids = check_choice(logits, 8, out, "sigmoid", b)
    assert torch.equal(cnt.cpu().long(), R.counts(ids, 256)[0])


def test_more_logits_than_32_bits_count():
    """2^31 + logits: offsets and the slots' sums past one workgroup's limit; sampled rows against the definition."""
    n, experts, top_k = 9_000_000, 256, 2
    say("2.3e9 logits")
    g = torch.Generator(device=dev()).manual_seed(0)
    logits = torch.randn(n, experts, generator=g, device=dev(), dtype=torch.bfloat16)
    out, loss, cnt = B.select_and_balance(logits, top_k, alpha=1.0)
    rows = torch.cat([torch.arange(0, 50), torch.arange(8_388_600, 8_388_650), torch.arange(n - 50, n)]).to(dev())
    part = T.StandardTopKOutput(out.topk_weights[rows], out.topk_ids[rows])
    check_choice(logits[rows].cpu(), top_k, part, "softmax")
    assert torch.equal(cnt.long(), torch.bincount(out.topk_ids.reshape(-1).long(), minlength=experts))
    share = sum(torch.softmax(p.double(), 1).sum(0) for p in logits.split(1_000_000))
    want = experts / (top_k * n * n) * float((share * cnt.double()).sum())
    assert abs(float(loss) - want) <= 2.0**-12 * want  # blocks of 1024 rows: 256 fp32 sums in a row each


@pytest.mark.parametrize("which", ["select", "balance", "both"])
def test_no_second_derivative(which):
    """create_graph gives the gradient and an error where it is differentiated again."""
    logits, _ = make(4, 16, 50)
    leaf = logits.to(dev()).requires_grad_()
    say(f"second derivative {which}")

    def value(x):
        if which == "select":
            return (T.select_experts(x, 3).topk_weights ** 2).sum()
        if which == "balance":
            return B.balance_loss(x, torch.zeros(4, 3, dtype=torch.int32, device=dev()), alpha=1.0)[0]
        out, loss, _ = B.select_and_balance(x, 3, alpha=1.0)
        return (out.topk_weights ** 2).sum() + loss

    (plain,) = torch.autograd.grad(value(leaf), leaf)
    (graph,) = torch.autograd.grad(value(leaf), leaf, create_graph=True)
    assert torch.equal(plain, graph.detach())
    with pytest.raises(RuntimeError):
        graph.sum().backward()


MANY = 6151  # above the rows from which 16 lanes hold a row


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("experts,top_k,groups,keep", [(64, 8, 8, 3), (100, 6, 0, 0), (128, 16, 16, 9), (129, 4, 3, 2),
                                                       (200, 1, 0, 0), (256, 8, 8, 4), (256, 16, 16, 3)])
def test_choice_of_many_rows(experts, top_k, groups, keep, bias, scoring):
    for dtype in (torch.float32, torch.bfloat16):
        logits, b = make(MANY, experts, experts + 3, dtype, bias)
        renorm = experts % 2 == 0
        say(f"many rows E={experts} k={top_k} groups={groups}/{keep} {scoring} bias={bias} {dtype}")
        out = select(logits, top_k, b, scoring=scoring, renormalize=renorm, groups=groups, keep=keep, scale=1.5)
        check_choice(logits, top_k, out, scoring, b, renorm, 1.5, groups, keep)


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("experts", [72, 160])
def test_ties_close_scores_and_masks_of_many_rows(experts, bias, scoring):
    g = torch.Generator().manual_seed(experts)
    n = MANY
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.randn(n, experts, generator=g)
        sign = torch.where(torch.rand(n, experts, generator=g) < 0.5, -1.0, 1.0)
        logits[::3] = (torch.randint(-2, 2, (n, experts), generator=g).float() * sign)[::3]  # ties, both zeros
        logits[1::3, experts // 2 :] = logits[1::3, : experts // 2] * (1 + 2.0**-22)  # next floats
        logits[torch.rand(n, experts, generator=g) < 0.02] = -math.inf
        logits[torch.rand(n, experts, generator=g) < 0.005] = math.inf
        logits[torch.rand(n, experts, generator=g) < 0.005] = math.nan
        logits[torch.rand(n, experts, generator=g) < 0.01] = torch.finfo(dtype).min
        logits[5, 4:], logits[6], logits[7] = -math.inf, -math.inf, math.nan
        logits = logits.to(dtype)
        b = torch.randint(-1, 2, (experts,), generator=g).float() * 2.0**-40 if bias else None
        for groups, keep in ((0, 0), (8, 3)):
            say(f"many rows, ties and masks E={experts} {scoring} bias={bias} {dtype} groups={groups}")
            out = select(logits, 7, b, scoring=scoring, groups=groups, keep=keep)
            check_choice(logits, 7, out, scoring, b, groups=groups, keep=keep)


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("experts,top_k,bias,renorm", [(60, 4, False, False), (128, 8, True, True), (160, 6, True, False), (256, 8, False, True)])
def test_gradients_of_many_rows(experts, top_k, bias, renorm, scoring):
    n, scale, alpha, cu = MANY, 1.5, 5.0, [2, 12, 1500, 1500, 4000]
    for dtype in (torch.float32, torch.bfloat16):
        logits, b = make(n, experts, experts + 9, dtype, bias)
        g = torch.Generator().manual_seed(experts)
        gw = torch.randn(n, top_k, generator=g)
        valid = torch.rand(n, generator=g) < 0.9
        say(f"many rows, gradients E={experts} bias={bias} renorm={renorm} {scoring} {dtype}")
        leaf = logits.to(dev()).requires_grad_()
        out, loss, cnt = B.select_and_balance(leaf, top_k, alpha=alpha, scoring=scoring, renormalize=renorm,
                                              correction_bias=None if b is None else b.to(dev()), routed_scaling_factor=scale,
                                              valid=valid.to(dev()), cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev()))
        ids = check_choice(logits, top_k, out, scoring, b, renorm, scale, valid=valid)
        assert torch.equal(cnt.cpu().long(), R.counts(ids, experts, cu, valid))
        want = float(R.balance(R.canon(logits), ids, scoring, alpha, cu, valid))
        assert abs(float(loss.detach()) - want) <= 2.0**-16 * abs(want)
        for lo, hi in ((True, True), (False, True)):
            outs = ([out.topk_weights] if lo else []) + [loss]
            gs = ([gw.to(dev())] if lo else []) + [torch.tensor(2.0, device=dev())]
            (got,) = torch.autograd.grad(outs, (leaf,), gs, retain_graph=True)
            ref = R.grads(logits, ids.clamp_min(0), scoring, renorm, scale, gw if lo else None, 2.0, alpha, cu, valid)
            tol = 2.0**-16 * (scale * float(gw.abs().max()) if lo else 0.0) + 2.0**-16 * 2 * alpha * experts / 10
            tol = tol + (2.0**-8 * ref.abs() if dtype == torch.bfloat16 else 0.0)
            assert ((got.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("experts", [48, 72, 160, 300, 1000])
def test_ties_at_zero_and_denormals(experts):
    """Equal and nearly equal logits around zero, where a float's last bits are all that it has."""
    g = torch.Generator().manual_seed(experts)
    for n in (40, MANY):
        logits = torch.randint(-3, 4, (n, experts), generator=g).float() * 2.0**-149
        logits[1::4] = torch.where(torch.rand(n, experts, generator=g) < 0.5, -0.0, 0.0)[1::4]
        logits[2::4] = (torch.randint(-9, 10, (n, experts), generator=g).float() * 2.0**-130)[2::4]
        logits[3::4] = torch.randint(-3, 1, (n, experts), generator=g).float()[3::4]  # zeros are the best
        for groups, keep in ((0, 0), (4, 2)):
            say(f"around zero n={n} E={experts} groups={groups}")
            check_choice(logits, 8, select(logits, 8, groups=groups, keep=keep), "softmax", groups=groups, keep=keep)


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("experts", [64, 72, 256, 1000])
def test_choice_by_scores_that_leave_the_floats(experts, scoring):
    """No bias to speak of and scores that fp32 does not hold: the 64-bit score decides."""
    g = torch.Generator().manual_seed(experts)
    n = 60
    logits = -70 - 130 * torch.rand(n, experts, generator=g)
    logits[0::3, 5] = 0.0  # a softmax's others are below 2^-100
    logits[1::3] = -math.inf
    for b in (torch.zeros(experts), torch.randint(-1, 2, (experts,), generator=g).float() * 2.0**-145):
        for groups, keep in ((0, 0), (4, 2)):
            say(f"small scores E={experts} {scoring} groups={groups}")
            out = select(logits, 8, b, scoring=scoring, groups=groups, keep=keep, renormalize=False)
            ids = R.choose(R.canon(logits), 8, scoring, b, groups, keep)
            assert torch.equal(out.topk_ids.cpu().long(), ids)
            want = R.weights(R.canon(logits), ids, scoring, False, 1.0)
            # a score below 2^-126 may be 0; else the bound of the other tests
            assert ((out.topk_weights.cpu().double() - want).abs() <= 2.0**-20 * want + 2.0**-125).all()


@pytest.mark.parametrize("renorm", [False, True])
def test_sqrtsoftplus_of_small_logits_keeps_its_weights(renorm):
    """e^l leaves the floats at -88, sqrt(e^l) at -175."""
    g = torch.Generator().manual_seed(5)
    logits = -60 - 100 * torch.rand(50, 64, generator=g)
    say(f"small sqrtsoftplus {renorm}")
    out = select(logits, 6, scoring="sqrtsoftplus", renormalize=renorm)
    z = R.canon(logits)
    ids = R.choose(z, 6, "sqrtsoftplus")
    want = R.weights(z, ids, "sqrtsoftplus", renorm, 1.0)
    assert torch.equal(out.topk_ids.cpu().long(), ids)
    assert ((out.topk_weights.cpu().double() - want).abs() <= 2.0**-20 * want + 2.0**-125).all()


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("experts,top_k,groups,keep", [(129, 4, 3, 2), (160, 6, 8, 3), (200, 17, 0, 0), (256, 8, 8, 4), (256, 32, 32, 9)])
def test_biased_choice_of_many_rows(experts, top_k, groups, keep, scoring):
    """Above the rows from which 32 lanes hold a row with a bias: ordinary rows, ties, masks, next floats."""
    g = torch.Generator().manual_seed(experts + top_k)
    n = 12301
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.randn(n, experts, generator=g) * 2
        logits[::5] = torch.randint(-2, 2, (n, experts), generator=g).float()[::5]
        half = experts // 2
        logits[1::5, half : 2 * half] = logits[1::5, :half] * (1 + 2.0**-22)
        logits[torch.rand(n, experts, generator=g) < 0.01] = -math.inf
        logits[torch.rand(n, experts, generator=g) < 0.003] = math.inf
        logits[torch.rand(n, experts, generator=g) < 0.003] = math.nan
        logits[7, 9:], logits[8], logits[9] = -math.inf, -math.inf, math.nan
        logits = logits.to(dtype)
        for b in (torch.randn(experts, generator=g) * 0.05, torch.zeros(experts)):
            say(f"many biased rows E={experts} k={top_k} groups={groups}/{keep} {scoring} {dtype}")
            out = select(logits, top_k, b, scoring=scoring, groups=groups, keep=keep, scale=1.5)
            check_choice(logits, top_k, out, scoring, b, True, 1.5, groups, keep)


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("experts", [64, 256, 1000])
def test_scores_at_the_floats_lower_end_give_finite_results(experts, scoring):
    """Scores around 2^-126, where a reciprocal of their sum can leave the floats."""
    g = torch.Generator().manual_seed(experts)
    n, top_k, scale = 96, 8, 1.5
    low = -2.0 if scoring == "sqrtsoftplus" else -1.0
    # a row's logits within a few of the border, the rows from well above it to well below
    logits = low * torch.linspace(84, 106, n)[:, None] + torch.rand(n, experts, generator=g) * 2
    for renorm in (True, False):
        for b in (None, torch.zeros(experts)):
            say(f"lower end E={experts} {scoring} renorm={renorm} bias={b is not None}")
            leaf = logits.to(dev()).requires_grad_()
            out, loss, _ = B.select_and_balance(leaf, top_k, alpha=1.0, scoring=scoring, renormalize=renorm,
                                                correction_bias=None if b is None else b.to(dev()), routed_scaling_factor=scale)
            (grad,) = torch.autograd.grad((out.topk_weights.sum(), loss), (leaf,))
            w = out.topk_weights.detach()
            loss = loss.detach()
            assert torch.isfinite(w).all() and torch.isfinite(loss) and torch.isfinite(grad).all()
            assert (w >= 0).all() and (w.sum(1) <= scale * (1 + 2.0**-20)).all()
            # s' adds up to at most one a row, so the loss is at most experts / k * n * k / n
            assert 0 <= float(loss) <= experts * (1 + 2.0**-12)
            alone = select(logits, top_k, b, scoring=scoring, renormalize=renorm, scale=scale)
            assert torch.equal(alone.topk_ids, out.topk_ids) and torch.equal(alone.topk_weights, w)


@pytest.mark.parametrize("scoring,lo,hi", [("softmax", -60, 60), ("sigmoid", -80, 60), ("sqrtsoftplus", -160, 60)])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradients_of_logits_far_from_zero(scoring, lo, hi, renorm):
    """Weights' gradient within 2^-16 of its largest factor. Balance gradient: the shares' exponentials are off by |x| 2^-24
    relative with |x| <= 160, their sum by the same, so r s' (c - sum c s') by less than 2^-14 of the largest c,
    alpha E / (k T)."""
    n, experts, top_k, alpha, scale = 60, 128, 6, 3.0, 2.0
    g = torch.Generator().manual_seed(7)
    logits = lo + (hi - lo) * torch.rand(n, experts, generator=g)
    logits[::3] = lo + 20 * torch.rand(n, experts, generator=g)[::3]  # rows of small scores alone
    gw = torch.randn(n, top_k, generator=g)
    say(f"far gradients {scoring} renorm={renorm}")
    leaf = logits.to(dev()).requires_grad_()
    out, loss, _ = B.select_and_balance(leaf, top_k, alpha=alpha, scoring=scoring, renormalize=renorm, routed_scaling_factor=scale)
    ids = check_choice(logits, top_k, out, scoring, None, renorm, scale)
    for with_w in (True, False):
        outs, gs = ([out.topk_weights, loss], [gw.to(dev()), torch.tensor(1.0, device=dev())]) if with_w else ([loss], [torch.tensor(1.0, device=dev())])
        (got,) = torch.autograd.grad(outs, (leaf,), gs, retain_graph=True)
        want = R.grads(logits, ids, scoring, renorm, scale, gw if with_w else None, 1.0, alpha)
        tol = 2.0**-14 * alpha * experts / (top_k * n) + (2.0**-16 * scale * float(gw.abs().max()) if with_w else 0.0)
        assert ((got.cpu().double() - want).abs() <= tol).all(), float((got.cpu().double() - want).abs().max()) / tol


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("experts,top_k,bias", [(48, 1, False), (200, 1, True), (64, 4, False), (256, 8, True), (700, 3, True)])
def test_gradient_of_a_weight_that_holds_nearly_all(experts, top_k, bias, scoring):
    """Renormalized weights of which one is close to one: its gradient is small and still right. With g counted from
    the largest share's, u_i = share_i ((g_i - g*) - sum_j share_j (g_j - g*)): a share is off by 2^-21 of itself (an
    exponential of two ulps, a sum, a reciprocal), the differences by 2^-24, the slope by 2^-21."""
    g = torch.Generator().manual_seed(experts)
    n, scale = 40, 1.5
    logits = torch.randn(n, experts, generator=g) - 9
    logits[torch.arange(n), torch.randint(0, experts, (n,), generator=g)] = 5.0
    b = torch.randn(experts, generator=g) * 1e-5 if bias else None
    gw = torch.randn(n, top_k, generator=g)
    say(f"one share E={experts} k={top_k} {scoring}")
    leaf = logits.to(dev()).requires_grad_()
    out = T.select_experts(leaf, top_k, scoring=scoring, correction_bias=None if b is None else b.to(dev()), routed_scaling_factor=scale)
    (got,) = torch.autograd.grad(out.topk_weights, leaf, gw.to(dev()))
    ids = check_choice(logits, top_k, out, scoring, b, True, scale)
    want = R.grads(logits, ids, scoring, True, scale, gw)
    if top_k == 1:
        assert (got == 0).all() and (want.abs() < 1e-12).all()
        return
    share = R.weights(R.canon(logits), ids, scoring, True, 1.0)
    d = (gw.double() - gw.double().gather(1, share.argmax(1, keepdim=True))).abs()
    bound = torch.zeros(n, experts, dtype=torch.float64).scatter_(1, ids, scale * share * (d + (share * d).sum(1, keepdim=True)))
    # the reference goes through the whole softmax: fewer than 8 steps, each 2^-53 of terms up to scale |gw|, also in
    # the experts that were not chosen, whose gradient is 0
    own = 2.0**-50 * scale * float(gw.abs().max())
    assert ((got.cpu().double() - want).abs() <= 2.0**-18 * bound + own).all()


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("n,experts,top_k,groups,keep", [(40, 64, 6, 0, 0), (40, 60, 6, 12, 4), (40, 256, 8, 8, 4), (33, 160, 6, 8, 3),
                                                         (20, 700, 8, 0, 0), (20, 768, 8, 48, 7), (12301, 256, 8, 8, 4)])
def test_bias_that_bars_or_forces_experts(n, experts, top_k, groups, keep, scoring):
    """-inf and NaN in the bias bar an expert, +inf forces it; a group of both has no value."""
    g = torch.Generator().manual_seed(n + experts)
    logits = torch.randn(n, experts, generator=g) * 2
    for kinds in ((-math.inf,), (-math.inf, math.nan), (math.inf,), (math.inf, -math.inf)):
        b = torch.randn(experts, generator=g) * 0.05
        for kind in kinds:
            b[torch.rand(experts, generator=g) < (0.6 if len(kinds) == 2 and kind == -math.inf else 0.1)] = kind
        say(f"bias of {kinds} n={n} E={experts} groups={groups}/{keep} {scoring}")
        out = select(logits, top_k, b, scoring=scoring, groups=groups, keep=keep)
        check_choice(logits, top_k, out, scoring, b, groups=groups, keep=keep)


@pytest.mark.parametrize("scoring", ["sigmoid", "sqrtsoftplus"])
def test_one_pick_at_the_floats_lower_end(scoring):
    """One score around 2^-126: its renormalized weight is the scale or, where fp32 does not hold the score, 0."""
    n, experts, scale = 400, 64, 1.5
    low = (-2.0 if scoring == "sqrtsoftplus" else -1.0) * torch.linspace(85, 90, n)
    logits = torch.full((n, experts), -math.inf)
    logits[:, 9] = low
    for b in (None, torch.zeros(experts)):
        say(f"one pick, lower end {scoring} bias={b is not None}")
        leaf = logits.to(dev()).requires_grad_()
        out, loss, _ = B.select_and_balance(leaf, 1, alpha=1.0, scoring=scoring, routed_scaling_factor=scale,
                                            correction_bias=None if b is None else b.to(dev()))
        (grad,) = torch.autograd.grad((out.topk_weights.sum(), loss), (leaf,))
        w = out.topk_weights.detach().cpu()[:, 0]
        assert (out.topk_ids == 9).all() and torch.isfinite(grad).all() and torch.isfinite(loss.detach())
        assert (((w - scale).abs() <= 2.0**-20) | (w == 0)).all()
        assert (w[low > -86.5 * (2 if scoring == "sqrtsoftplus" else 1)] > 0).all()


@pytest.mark.parametrize("experts,top_k,groups,keep", [(257, 8, 0, 0), (300, 32, 0, 0), (384, 8, 12, 5), (480, 6, 32, 9), (512, 8, 8, 4)])
def test_unbiased_choice_of_many_rows_and_experts(experts, top_k, groups, keep):
    """32 lanes of 16 experts: ordinary rows, ties, masks, next floats."""
    g = torch.Generator().manual_seed(experts)
    n = MANY
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.randn(n, experts, generator=g) * 2
        logits[::4] = torch.randint(-2, 2, (n, experts), generator=g).float()[::4]
        half = experts // 2
        logits[1::4, half : 2 * half] = logits[1::4, :half] * (1 + 2.0**-22)
        logits[torch.rand(n, experts, generator=g) < 0.01] = -math.inf
        logits[torch.rand(n, experts, generator=g) < 0.003] = math.inf
        logits[torch.rand(n, experts, generator=g) < 0.003] = math.nan
        logits[7, 9:], logits[8], logits[9] = -math.inf, -math.inf, math.nan
        logits = logits.to(dtype)
        for scoring, renorm in (("softmax", True), ("softmax", False), ("sqrtsoftplus", True)):
            say(f"many rows and experts E={experts} k={top_k} groups={groups}/{keep} {scoring} {dtype}")
            out = select(logits, top_k, scoring=scoring, groups=groups, keep=keep, renormalize=renorm)
            check_choice(logits, top_k, out, scoring, None, renorm, 1.0, groups, keep)
