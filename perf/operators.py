"""Performance cases of the operators around the routed experts: the router's choice of experts
(scores, correction bias, groups, top-k) with its gradient, the balance loss and the experts'
counts with their gradient, and the FP8 block product of the shared expert.

``listed`` are fixed calls, ``draw`` gives more of the same ranges, ``prepare`` makes what a
program holds before the call, ``run`` is one pass, with elementary torch operations or (``own``)
through the public entry points, ``exact`` the same result in 64 bits.

A case is a dict of plain values with ``op``:

* "linear": ``n`` tokens, ``k`` input and ``out`` output features: x bf16 quantized to e4m3 per
  1x128, weights e4m3 with one fp32 scale per 128x128;
* "topk": the selection alone (serving), ``n`` tokens, ``experts``, ``topk``, ``scoring``, ``bias``,
  ``groups`` / ``keep`` (groups kept), ``renorm``, ``scale``, ``fmt`` of the logits;
* "train": selection, balance loss and counts, and the gradient of the logits from the weights'
  gradient and the loss's; ``seqs`` sequences (0: the batch is one), ``padded`` rows at the end
  that hold no token;
* "balance": balance loss, counts and gradient for given ids; "counts": the counts alone.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sgl-afd-plugin_amd")
BLOCK = 128
ALPHA = 1e-3  # the balance loss's weight


def _product(n, k, out, name=None):
    case = dict(op="linear", n=n, k=k, out=out)
    if name:
        case["name"] = name
    return case


def _router(op, n, experts, topk, name=None, *, scoring="softmax", bias=False, groups=0, keep=0, renorm=True,
            scale=1.0, fmt="f32", seqs=0, padded=0):
    case = dict(op=op, n=n, experts=experts, topk=topk, scoring=scoring, bias=bias, groups=groups, keep=keep,
                renorm=renorm, scale=scale, fmt=fmt, seqs=seqs, padded=padded)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the shared expert's gate and up projection of one decoded token
        _product(1, 4096, 4096, "linear_token"),
        # its down projection in a decode step of a batch
        _product(48, 2048, 4096, "linear_decode_48"),
        # a projection whose sizes fit no block, over a short prompt
        _product(300, 2000, 1111, "linear_ragged_300"),
        # a chunk of prompts
        _product(2900, 4096, 4096, "linear_chunk_2900"),
        # the whole prefill dispatch
        _product(16384, 4096, 4096, "linear_prefill_16384"),
        # the router of a decode step: 256 experts, square roots of softplus, correction bias
        _router("topk", 8, 256, 8, "topk_decode_8", scoring="sqrtsoftplus", bias=True, scale=1.5),
        # a chunk with bf16 logits over 64 experts (ties are common), softmax
        _router("topk", 2900, 64, 8, "topk_chunk_2900", fmt="bf16"),
        # prefill with expert groups: sigmoid, correction bias, 4 of 8 groups
        _router("topk", 16384, 256, 8, "topk_prefill_16384", scoring="sigmoid", bias=True, groups=8, keep=4, scale=2.5),
        # training the router: a packed batch of short sequences with padding behind, odd sizes
        _router("train", 1531, 60, 4, "train_packed_1531", renorm=False, fmt="bf16", seqs=5, padded=31),
        # training the router: one large batch
        _router("train", 16384, 256, 8, "train_16384", scoring="sqrtsoftplus", bias=True, scale=1.5),
        # the loss for ids that came from elsewhere, per sequence
        _router("balance", 8192, 64, 8, "balance_8192", seqs=32),
        # the counts that a serving rank keeps of where its tokens went
        _router("counts", 16384, 256, 8, "counts_16384"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "topk", "topk", "train", "balance", "counts"])
    if op == "linear":
        k, out = (rng.choice([128 * rng.randint(1, 32), _log(rng, 64, 4096)]) for _ in range(2))
        return _product(_log(rng, 1, 16384), k, out)
    experts = rng.choice([32, 64, 128, 256, 256, rng.randint(8, 256)])
    n = _log(rng, 1, 16384)
    more = dict(fmt=rng.choice(["f32", "f32", "bf16"]), scoring=rng.choice(["softmax", "sigmoid", "sqrtsoftplus"]))
    if op in ("topk", "train"):
        more.update(bias=rng.random() < 0.5, renorm=rng.random() < 0.7, scale=rng.choice([1.0, 1.5, 2.5]))
        if experts % 8 == 0 and rng.random() < 0.3:
            more.update(groups=8, keep=4)
    if op in ("train", "balance") and n >= 64:
        more.update(seqs=rng.choice([0, 0, rng.randint(1, 48)]), padded=rng.choice([0, rng.randint(1, n // 8)]))
    return _router(op, n, experts, rng.randint(1, min(8, experts // 2)), **more)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _product_inputs(case, seed):
    """x ~ N(0, 1) in bf16; weights ~ N(0, 0.02) held as e4m3 codes with fp32 block scales."""
    gen, n, k, out = _gen(seed), case["n"], case["k"], case["out"]
    x = torch.randn(n, k, generator=gen, device="cuda").to(torch.bfloat16)
    kb, nb = -(-k // BLOCK), -(-out // BLOCK)
    w = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
    w[:out, :k] = torch.randn(out, k, generator=gen, device="cuda").mul_(0.02)
    w = w.view(nb, BLOCK, kb, BLOCK)
    amax = w.abs().amax((1, 3))
    scales = amax / torch.full_like(amax, 448.0)
    codes = (w / scales[:, None, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    codes = codes.view(torch.uint8).reshape(nb * BLOCK, kb * BLOCK)[:out, :k].contiguous()
    return x, codes.view(torch.float8_e4m3fn), scales


def _bounds(case):
    """cu_seqlens of uneven sequences over the rows that hold tokens (the lengths belong to the case)."""
    live = case["n"] - case["padded"]
    rng = random.Random(case["n"])
    cuts = sorted(rng.sample(range(1, live), case["seqs"] - 1))
    return [0] + cuts + [live]


def _router_inputs(case, seed):
    """Logits of a router with popular and unpopular experts, the correction bias that answers
    them, ids as a router would give, and what a training step hands the backward."""
    gen, n, experts, topk = _gen(seed), case["n"], case["experts"], case["topk"]
    popular = torch.randn(experts, generator=_gen(experts), device="cuda") * 0.5
    logits = torch.randn(n, experts, generator=gen, device="cuda") + popular
    logits = logits.to(torch.bfloat16 if case["fmt"] == "bf16" else torch.float32)
    state = dict(logits=logits, bias=None, cu=None, valid=None, ids=None, gw=None, gl=None)
    if case["bias"]:
        state["bias"] = 0.02 * torch.randn(experts, generator=gen, device="cuda") - 0.1 * popular
    if case["op"] in ("balance", "counts"):
        noise = torch.rand(n, experts, generator=gen, device="cuda") * 2.0 + logits.float()
        state["ids"] = torch.topk(noise, topk, dim=-1).indices.to(torch.int32)
    if case["op"] in ("train", "balance"):
        if case["seqs"]:
            state["cu"] = torch.tensor(_bounds(case), dtype=torch.int32, device="cuda")
        if case["padded"]:
            state["valid"] = torch.arange(n, device="cuda") < n - case["padded"]
        state["gw"] = torch.randn(n, topk, generator=gen, device="cuda")
        state["gl"] = torch.ones((), device="cuda")
    return state


def prepare(case, seed):
    if case["op"] == "linear":
        x, codes, scales = _product_inputs(case, seed)
        state = dict(case=case, x=x, codes=codes, scales=scales)
        if own:
            if PKG not in sys.path:
                sys.path.insert(0, PKG)
            from sgl_asap_amd.moe.linear import Fp8BlockLinear

            state["layer"] = Fp8BlockLinear(codes, scales)
        return state
    state = dict(case=case, **_router_inputs(case, seed))
    if own:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        from sgl_asap_amd.moe import balance, topk

        state["balance"], state["topk"] = balance, topk
        if case["op"] in ("train", "balance"):
            state["logits"].requires_grad_()
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "topk": _own_topk, "train": _own_train, "balance": _own_balance,
                "counts": _own_counts}[op](state)
    return {"linear": _plain_linear, "topk": _plain_topk, "train": _plain_train, "balance": _plain_balance,
            "counts": _plain_counts}[op](state)


def _choice_args(case):
    return dict(scoring=case["scoring"], renormalize=case["renorm"], num_expert_group=case["groups"] or None,
                topk_group=case["keep"] or None, routed_scaling_factor=case["scale"])


def _own_linear(state):
    return state["layer"](state["x"])


def _own_topk(state):
    case = state["case"]
    out = state["topk"].select_experts(state["logits"], case["topk"], correction_bias=state["bias"], **_choice_args(case))
    return out.topk_weights, out.topk_ids


def _own_train(state):
    case, logits = state["case"], state["logits"]
    out, loss, counts = state["balance"].select_and_balance(
        logits, case["topk"], alpha=ALPHA, correction_bias=state["bias"], cu_seqlens=state["cu"], valid=state["valid"],
        **_choice_args(case))
    (grad,) = torch.autograd.grad((out.topk_weights, loss), (logits,), (state["gw"], state["gl"]))
    return out.topk_weights, out.topk_ids, loss, counts, grad


def _own_balance(state):
    case, logits = state["case"], state["logits"]
    loss, counts = state["balance"].balance_loss(logits, state["ids"], alpha=ALPHA, scoring=case["scoring"],
                                                 cu_seqlens=state["cu"], valid=state["valid"])
    (grad,) = torch.autograd.grad((loss,), (logits,), (state["gl"],))
    return loss, counts, grad


def _own_counts(state):
    return state["balance"].expert_counts(state["ids"], state["case"]["experts"])


# ---------------------------------------------------------------- plain forms
def _plain_linear(state):
    """Quantize x per 1x128, hold both operands in fp32, multiply, round once."""
    x, codes, scales, case = state["x"], state["codes"], state["scales"], state["case"]
    n, k, kb = case["n"], case["k"], scales.shape[1]
    v = torch.zeros(n, kb * BLOCK, device=x.device)
    v[:, :k] = x
    v = v.view(n, kb, BLOCK)
    amax = v.abs().amax(-1, keepdim=True).clamp_min(1e-10)
    s = amax / torch.full_like(amax, 448.0)
    v = ((v / s).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float() * s).view(n, kb * BLOCK)[:, :k]
    w = codes.float()
    rows = torch.arange(w.shape[0], device=x.device) // BLOCK
    cols = torch.arange(k, device=x.device) // BLOCK
    w = w * scales[rows][:, cols]
    return torch.mm(v, w.t()).to(torch.bfloat16)


def _scores(v, scoring):
    if scoring == "softmax":
        e = torch.exp(v - v.amax(-1, keepdim=True))
        return e / e.sum(-1, keepdim=True)
    if scoring == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    return torch.sqrt(_softplus(v))


def _softplus(v):
    return torch.log1p(torch.exp(-v.abs())) + v.clamp_min(0.0)


def _pick(case, logits, bias):
    """ids of the chosen experts: order of the logits, or of the scores plus the bias in 64 bits."""
    v = logits.float() if bias is None else _scores(logits.double(), case["scoring"]) + bias.double()
    if case["groups"]:
        g = v.view(v.shape[0], case["groups"], -1)
        best = g.sort(-1, descending=True).values
        best = best[..., 0] if bias is None else best[..., :2].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, : case["keep"]]
        mask = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        v = torch.where(mask[..., None], g, torch.full_like(g, -math.inf)).view_as(v)
    return v.sort(dim=-1, descending=True, stable=True).indices[:, : case["topk"]]


def _weights(case, scores, ids):
    w = scores.gather(1, ids)
    if case["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return w * case["scale"]


def _plain_topk(state):
    case, logits = state["case"], state["logits"]
    ids = _pick(case, logits, state["bias"])
    return _weights(case, _scores(logits.float(), case["scoring"]), ids), ids.to(torch.int32)


def _sequences(state):
    """(sequence of each row, which rows count, the number of sequences)."""
    case = state["case"]
    n, dev = case["n"], state["logits"].device
    live = torch.ones(n, dtype=torch.bool, device=dev) if state["valid"] is None else state["valid"]
    if state["cu"] is None:
        return torch.zeros(n, dtype=torch.int64, device=dev), live, 1
    cu = state["cu"].long()
    rows = torch.arange(n, device=dev)
    seq = (rows[:, None] >= cu[None, 1:]).sum(1)
    live = live & (rows >= cu[0]) & (seq < case["seqs"])
    return seq.clamp_max(case["seqs"] - 1), live, case["seqs"]


def _count(state, ids):
    case = state["case"]
    seq, live, seqs = _sequences(state)
    slots = (seq[:, None] * case["experts"] + ids)[live].reshape(-1)
    return torch.bincount(slots, minlength=seqs * case["experts"]).view(seqs, case["experts"]).to(torch.int32)


def _plain_balance_parts(state, ids, scores):
    """(loss, counts, gradient of the loss by the logits)."""
    case, logits = state["case"], state["logits"].float()
    experts, topk = case["experts"], case["topk"]
    seq, live, seqs = _sequences(state)
    counts = _count(state, ids)
    rows = torch.zeros(seqs, device=logits.device).index_add_(0, seq, live.float())
    share = scores / scores.sum(-1, keepdim=True) * live[:, None]
    mean = torch.zeros(seqs, experts, device=logits.device).index_add_(0, seq, share)
    used = (rows > 0).sum()
    rows = rows.clamp_min(1.0)[:, None]
    factor = ALPHA * experts / (topk * rows * rows * used) * counts
    loss = (factor * mean).sum()
    c = factor[seq] * state["gl"]
    d = share * (c - (c * share).sum(-1, keepdim=True))
    if case["scoring"] == "sigmoid":
        d = d * (1.0 - scores)
    elif case["scoring"] == "sqrtsoftplus":
        d = d / (2.0 * (1.0 + torch.exp(-logits)) * _softplus(logits))
    return loss, counts, d


def _plain_weights_grad(state, scores, ids):
    """Gradient by the logits of the weights, from the weights' gradient."""
    case, logits, gw = state["case"], state["logits"].float(), state["gw"] * state["case"]["scale"]
    picked = scores.gather(1, ids)
    if case["renorm"]:
        # the differences cancel where one weight holds nearly all (always with one expert): 64 bits
        total = picked.double().sum(-1, keepdim=True)
        gs = ((gw - (gw * (picked / total)).sum(-1, keepdim=True)) / total).float()
    else:
        gs = gw
    _, live, _ = _sequences(dict(state, cu=None))
    d = torch.zeros_like(scores).scatter_(1, ids, gs * live[:, None])
    if case["scoring"] == "softmax":
        return scores * (d - (d * scores).sum(-1, keepdim=True))
    if case["scoring"] == "sigmoid":
        return d * scores * (1.0 - scores)
    return d / ((1.0 + torch.exp(-logits)) * 2.0 * scores)


def _plain_train(state):
    case, logits = state["case"], state["logits"]
    ids = _pick(case, logits, state["bias"])
    scores = _scores(logits.float(), case["scoring"])
    weights = _weights(case, scores, ids)
    loss, counts, grad = _plain_balance_parts(state, ids, scores)
    grad = grad + _plain_weights_grad(state, scores, ids)
    if state["valid"] is not None:
        ids = torch.where(state["valid"][:, None], ids, torch.full_like(ids, -1))
        weights = weights * state["valid"][:, None]
    if state["cu"] is None:
        counts = counts[0]
    return weights, ids.to(torch.int32), loss, counts, grad.to(logits.dtype)


def _plain_balance(state):
    case, logits = state["case"], state["logits"]
    loss, counts, grad = _plain_balance_parts(state, state["ids"].long(), _scores(logits.float(), case["scoring"]))
    return loss, counts if state["cu"] is not None else counts[0], grad.to(logits.dtype)


def _plain_counts(state):
    return _count(state, state["ids"].long())[0]


# ---------------------------------------------------------------- what a pass needs
def work(case):
    n = case["n"]
    if case["op"] == "linear":
        k, out = case["k"], case["out"]
        blocks = -(-k // BLOCK) * -(-out // BLOCK)
        return {"bytes": n * k * 2 + out * k + blocks * 4 + n * out * 2, "flops": 2 * n * out * k}
    experts, topk = case["experts"], case["topk"]
    logits = n * experts * (2 if case["fmt"] == "bf16" else 4)
    seqs = max(1, case["seqs"])
    if case["op"] == "counts":
        return {"bytes": n * topk * 4 + experts * 4, "flops": n * topk}
    if case["op"] == "topk":
        return {"bytes": logits + n * topk * 8 + (experts * 4 if case["bias"] else 0), "flops": 8 * n * experts}
    if case["op"] == "balance":
        return {"bytes": 2 * logits + n * topk * 4 + seqs * experts * 4 + 4, "flops": 16 * n * experts}
    return {"bytes": 2 * logits + n * topk * 12 + seqs * experts * 4 + 4, "flops": 24 * n * experts}


# ---------------------------------------------------------------- the results in 64 bits
def exact(case, seed):
    if case["op"] == "linear":
        return _exact_linear(case, seed)
    data = _router_inputs(case, seed)
    if case["op"] == "counts":
        return _exact_counts(case, data, data["ids"])
    z = data["logits"].double()
    if case["op"] == "topk":
        w, ids = _exact_choice(case, z, data["bias"])
        return w, ids.to(torch.int32)
    z.requires_grad_()
    if case["op"] == "balance":
        loss = _exact_loss(case, data, z, data["ids"])
        (grad,) = torch.autograd.grad(loss, z)
        return loss.detach(), _exact_counts(case, data, data["ids"]), grad
    w, ids = _exact_choice(case, z, data["bias"])
    if data["valid"] is not None:
        ids = ids.masked_fill(~data["valid"][:, None], -1)
        w = w.masked_fill(~data["valid"][:, None], 0.0)
    loss = _exact_loss(case, data, z, ids)
    (grad,) = torch.autograd.grad((w * data["gw"].double()).sum() + loss, z)
    return w.detach(), ids.to(torch.int32), loss.detach(), _exact_counts(case, data, ids), grad


def _exact_linear(case, seed):
    x, codes, scales = _product_inputs(case, seed)
    y = torch.zeros(case["n"], case["out"], dtype=torch.float64, device=x.device)
    for at in range(0, case["k"], BLOCK):
        end = min(at + BLOCK, case["k"])
        part = x[:, at:end].float()
        top = part.abs().max(dim=1, keepdim=True).values.clamp(min=1e-10)
        s = top / torch.full_like(top, 448.0)
        q = (part / s).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).double() * s.double()
        for to in range(0, case["out"], BLOCK):
            last = min(to + BLOCK, case["out"])
            w = codes[to:last, at:end].double() * scales[to // BLOCK, at // BLOCK].double()
            y[:, to:last] += q @ w.t().contiguous()
    return y


def _exact_scores(z, scoring):
    if scoring == "softmax":
        return torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
    if scoring == "sigmoid":
        return torch.sigmoid(z)
    return torch.nn.functional.softplus(z, threshold=1e9).sqrt()


def _first_best(v, count):
    """Indices of the ``count`` largest values of each row, one by one, the first of equals."""
    v, picked = v.clone(), []
    for _ in range(count):
        top = v.max(dim=1, keepdim=True).values
        at = (v == top).to(torch.uint8).argmax(dim=1, keepdim=True)
        picked.append(at)
        v.scatter_(1, at, -math.inf)
    return torch.cat(picked, dim=1)


def _exact_choice(case, z, bias):
    scores = _exact_scores(z, case["scoring"])
    choice = z.detach().clone() if bias is None else scores.detach() + bias.double()
    if case["groups"]:
        size = case["experts"] // case["groups"]
        parts = choice.split(size, dim=1)
        value = [p.topk(min(2, size) if bias is not None else 1, dim=1).values.sum(1) for p in parts]
        keep = _first_best(torch.stack(value, dim=1), case["keep"])
        for g in range(case["groups"]):
            gone = ~(keep == g).any(1)
            choice[gone, g * size : (g + 1) * size] = -math.inf
    ids = _first_best(choice, case["topk"])
    w = torch.take_along_dim(scores, ids, dim=1)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return w * case["scale"], ids


def _exact_spans(case, data):
    if data["cu"] is None:
        return [(0, case["n"])]
    cu = data["cu"].tolist()
    return list(zip(cu, cu[1:]))


def _exact_counts(case, data, ids):
    rows = []
    for lo, hi in _exact_spans(case, data):
        part = ids[lo:hi] if data["valid"] is None else ids[lo:hi][data["valid"][lo:hi]]
        hot = torch.zeros(case["experts"], dtype=torch.int64, device=ids.device)
        hot.scatter_add_(0, part.reshape(-1).long(), torch.ones_like(part.reshape(-1), dtype=torch.int64))
        rows.append(hot.to(torch.int32))
    return rows[0] if data["cu"] is None else torch.stack(rows)


def _exact_loss(case, data, z, ids):
    counts = _exact_counts(case, data, ids)
    counts = (counts[None] if data["cu"] is None else counts).double()
    scores = _exact_scores(z, case["scoring"])
    share = scores / scores.sum(1, keepdim=True)
    terms = []
    for s, (lo, hi) in enumerate(_exact_spans(case, data)):
        part = share[lo:hi] if data["valid"] is None else share[lo:hi][data["valid"][lo:hi]]
        if part.shape[0]:
            f = counts[s] * case["experts"] / (case["topk"] * part.shape[0])
            terms.append((f * part.mean(0)).sum())
    return ALPHA * torch.stack(terms).mean()
