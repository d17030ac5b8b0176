"""Performance cases of the operators that stand around a MoE block's experts: the int8 product of its shared
expert, its tokens sorted by expert and back (with their gradients), and the norms before and after the block
with its gate and residual scale (with their gradients).

``listed`` are fixed calls, ``draw`` gives more of the same ranges, ``prepare`` makes what a
program holds before the call, ``run`` is one pass, with elementary torch operations or (``own``)
through the public entry points, ``exact`` the same result in 64 bits.

A case is a dict of plain values with ``op``:

* "linear": ``n`` tokens, ``k`` input and ``out`` output features: x bf16 quantized to int8 per token,
  weights int8 with one fp32 scale per output channel;
* "mlp": the shared expert, a SwiGLU MLP of two such products, ``n`` tokens, ``hidden``, ``inter``;
* "sort": ``n`` tokens of ``hidden`` values (``dtype``), each sent to ``topk`` of ``experts`` experts, of which this
  rank holds the first ``local``; sorted by expert, and the experts' rows (given) added up with their weights.
  ``padded`` tokens at the end have no experts; ``train``: the gradients too;
* "norm": ``n`` tokens of ``hidden`` values (``dtype``): ``pre``: the norm before the block; then residual + scale * gate *
  norm(block's output), ``gate`` "none", "channel" [hidden], "token" [n, 1] or "element" [n, hidden]; ``post``: with
  that norm; ``next``: and the norm before the block behind it. ``wide``: weights in fp32; ``train``: the gradients too.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sgl-afd-plugin_amd")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _case(op, name, **more):
    case = dict(op=op, **more)
    if name:
        case["name"] = name
    return case


def _linear(n, k, out, name=None):
    return _case("linear", name, n=n, k=k, out=out)


def _mlp(n, hidden, inter, name=None):
    return _case("mlp", name, n=n, hidden=hidden, inter=inter)


def _sort(n, hidden, experts, topk, name=None, *, local=0, dtype="bf16", padded=0, train=False):
    return _case("sort", name, n=n, hidden=hidden, experts=experts, topk=topk, local=local or experts, dtype=dtype,
                 padded=padded, train=train)


def _norm(n, hidden, name=None, *, dtype="bf16", pre=False, post=True, gate="none", next=False, scale=1.0, wide=False,
          train=False):
    return _case("norm", name, n=n, hidden=hidden, dtype=dtype, pre=pre, post=post, gate=gate, next=next, scale=scale,
                 wide=wide, train=train)


def listed():
    return [
        # the shared expert's gate and up projection of one decoded token
        _linear(1, 4096, 4096, "linear_token"),
        # a projection whose sizes fit no block, over a short prompt
        _linear(300, 2000, 1111, "linear_ragged_300"),
        # the whole prefill dispatch
        _linear(16384, 4096, 4096, "linear_prefill_16384"),
        # a chunk of prompts through the whole shared expert
        _mlp(2900, 4096, 1536, "mlp_chunk_2900"),
        # a decode step on a rank that holds a quarter of the experts
        _sort(8, 4096, 256, 8, "sort_decode_8", local=64),
        # training on a packed batch with padding behind, odd sizes
        _sort(1531, 1000, 60, 4, "sort_packed_1531", dtype="fp16", padded=31, train=True),
        # a training step of a large batch, every expert here
        _sort(8192, 2048, 64, 8, "sort_train_8192", train=True),
        # the whole prefill dispatch on a rank that holds a quarter of the experts
        _sort(16384, 4096, 256, 8, "sort_prefill_16384", local=64),
        # a decode step: the norm before the block and the one behind it, gated by channel
        _norm(8, 4096, "norm_decode_8", pre=True, gate="channel"),
        # prefill: the block's output into the residual, and the next block's input from it
        _norm(16384, 4096, "norm_prefill_16384", next=True, scale=0.22),
        # training in fp32 on a packed batch of odd sizes, a gate per token
        _norm(1531, 1111, "norm_packed_1531", dtype="fp32", pre=True, gate="token", scale=0.5, wide=True, train=True),
        # a training step of a large batch, weights and gate in fp32
        _norm(8192, 4096, "norm_train_8192", gate="channel", next=True, wide=True, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step):
    """A size of [lo, hi] over its logarithm, a multiple of ``step`` half of the time."""
    size = _log(rng, lo, hi)
    return size if rng.random() < 0.5 else max(step, size // step * step)


def draw(rng):
    op = rng.choice(["linear", "linear", "mlp", "sort", "sort", "sort", "norm", "norm", "norm"])
    if op == "linear":
        return _linear(_log(rng, 1, 16384), _size(rng, 64, 4096, 128), _size(rng, 64, 4096, 128))
    if op == "mlp":
        return _mlp(_log(rng, 1, 8192), _size(rng, 256, 4096, 128), _size(rng, 128, 2048, 128))
    train = rng.random() < 0.5
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "sort":
        n, experts = _log(rng, 1, 8192), rng.choice([32, 64, 128, 256, rng.randint(8, 256)])
        return _sort(n, _size(rng, 128, 2048, 64), experts, rng.randint(1, min(8, experts // 2)), dtype=dtype, train=train,
                     local=rng.choice([experts, experts, max(1, experts // 4)]),
                     padded=rng.choice([0, 0, rng.randint(0, n // 8)]))
    return _norm(_log(rng, 1, 8192), _size(rng, 128, 4096, 64), dtype=dtype, pre=rng.random() < 0.4, post=rng.random() < 0.7,
                 gate=rng.choice(["none", "channel", "token", "element"]), next=rng.random() < 0.6,
                 scale=rng.choice([1.0, 0.5, 0.22]), wide=rng.random() < 0.5, train=train)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _int8_weights(gen, out, k):
    """Weights ~ N(0, 0.02), held as int8 codes with one scale per output channel."""
    w = _randn(gen, out, k).mul_(0.02)
    amax = w.abs().amax(1)
    scales = amax / torch.full_like(amax, 127.0)
    return torch.round(w / scales[:, None]).to(torch.int8), scales


def _tokens(gen, n, hidden):
    """Hidden states: a few channels are much larger than the others, as in trained models."""
    x = _randn(gen, n, hidden)
    x[:, :: max(1, hidden // 7)] *= 8.0
    return x


def _linear_inputs(case, seed):
    gen = _gen(seed)
    x = _tokens(gen, case["n"], case["k"]).to(torch.bfloat16)
    codes, scales = _int8_weights(gen, case["out"], case["k"])
    return dict(x=x, codes=codes, scales=scales)


def _mlp_inputs(case, seed):
    gen = _gen(seed)
    x = _tokens(gen, case["n"], case["hidden"]).to(torch.bfloat16)
    w13, s13 = _int8_weights(gen, 2 * case["inter"], case["hidden"])
    w2, s2 = _int8_weights(gen, case["hidden"], case["inter"])
    return dict(x=x, w13=w13, s13=s13, w2=w2, s2=s2)


def _sort_inputs(case, seed):
    """Tokens, ids as a router with popular experts gives them, weights that add up to 1, and the experts' rows."""
    gen, n, topk, hidden = _gen(seed), case["n"], case["topk"], case["hidden"]
    dtype = DTYPES[case["dtype"]]
    popular = _randn(_gen(case["experts"]), case["experts"]) * 0.5
    score = torch.rand(n, case["experts"], generator=gen, device="cuda") * 2.0 + popular
    weights, ids = torch.topk(score, topk, dim=-1)
    weights = torch.softmax(weights, -1)
    ids = ids.to(torch.int32)
    if case["padded"]:
        ids[n - case["padded"] :] = -1
        weights[n - case["padded"] :] = 0.0
    state = dict(x=_randn(gen, n, hidden).to(dtype), ids=ids, weights=weights, rows=_randn(gen, n * topk, hidden).to(dtype))
    if case["train"]:
        state["g_rows"] = _randn(gen, n * topk, hidden).to(dtype)
        state["g_out"] = _randn(gen, n, hidden).to(dtype)
    return state


def _norm_inputs(case, seed):
    """The residual stream, the block's output, weights near 1 and a gate of both signs."""
    gen, n, hidden, dtype = _gen(seed), case["n"], case["hidden"], DTYPES[case["dtype"]]
    held = torch.float32 if case["wide"] else dtype
    state = dict(x=_tokens(gen, n, hidden).to(dtype), y=(0.3 * _randn(gen, n, hidden)).to(dtype), gate=None)
    for name in ("w_pre", "w_post", "w_next"):
        wanted = case[name[2:]]
        state[name] = (1.0 + 0.2 * _randn(gen, hidden)).to(held) if wanted else None
    shape = {"channel": (hidden,), "token": (n, 1), "element": (n, hidden)}.get(case["gate"])
    if shape:
        state["gate"] = torch.tanh(_randn(gen, *shape)).to(held)
    if case["train"]:
        for name in ("g_pre", "g_h", "g_next"):
            state[name] = _randn(gen, n, hidden).to(dtype)
    return state


INPUTS = {"linear": _linear_inputs, "mlp": _mlp_inputs, "sort": _sort_inputs, "norm": _norm_inputs}
LEAVES = {"sort": ("x", "rows", "weights"), "norm": ("x", "y", "gate", "w_pre", "w_post", "w_next")}


def prepare(case, seed):
    state = dict(case=case, **INPUTS[case["op"]](case, seed))
    if own:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        if case["op"] == "linear":
            from sgl_asap_amd.moe.linear import Int8Linear

            state["layer"] = Int8Linear(state["codes"], state["scales"])
        elif case["op"] == "mlp":
            from sgl_asap_amd.moe.shared import Int8SharedExpertMLP

            state["layer"] = Int8SharedExpertMLP(state["w13"], state["s13"], state["w2"], state["s2"])
        elif case["op"] == "sort":
            from sgl_asap_amd.moe import sort

            state["sort"] = sort
            if not case["train"]:  # a serving rank's own buffer of rows
                state["sorted"] = torch.zeros_like(state["rows"])
        else:
            from sgl_asap_amd.moe import norm

            state["norm"] = norm
        if case.get("train"):
            for name in LEAVES[case["op"]]:
                if state[name] is not None:
                    state[name].requires_grad_()
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_layer, "mlp": _own_layer, "sort": _own_sort, "norm": _own_norm}[op](state)
    return {"linear": _plain_linear, "mlp": _plain_mlp, "sort": _plain_sort, "norm": _plain_norm}[op](state)


def _own_layer(state):
    return state["layer"](state["x"])


def _own_sort(state):
    case, sort = state["case"], state["sort"]
    if not case["train"]:
        rows, order = sort.sort_tokens(state["x"], state["ids"], case["local"], out=state["sorted"])
        out = sort.unsort_tokens(state["rows"], order, state["weights"])
        return rows, order.positions, order.counts, out
    rows, order = sort.sort_tokens(state["x"], state["ids"], case["local"])
    out = sort.unsort_tokens(state["rows"], order, state["weights"])
    grads = torch.autograd.grad((rows, out), (state["x"], state["rows"], state["weights"]), (state["g_rows"], state["g_out"]))
    return (rows, order.positions, order.counts, out) + grads


def _own_norm(state):
    case, norm = state["case"], state["norm"]
    outs, given = [], []
    if case["pre"]:
        outs.append(norm.rms_norm(state["x"], state["w_pre"], eps=EPS))
        given.append(state.get("g_pre"))
    hidden, normed = norm.residual_norm(state["y"], state["x"], post_weight=state["w_post"], gate=state["gate"],
                                        scale=case["scale"], next_weight=state["w_next"], eps=EPS)
    outs.append(hidden)
    given.append(state.get("g_h"))
    if case["next"]:
        outs.append(normed)
        given.append(state.get("g_next"))
    if not case["train"]:
        return tuple(outs)
    leaves = [state[name] for name in LEAVES["norm"] if state[name] is not None]
    return tuple(outs) + torch.autograd.grad(outs, leaves, given)


# ---------------------------------------------------------------- plain forms
def _quantized(x):
    """x fp32 as int8 codes (held in fp32) and one scale per token."""
    amax = x.abs().amax(-1, keepdim=True).clamp_min(1e-10)
    s = amax / torch.full_like(amax, 127.0)
    return torch.round(x / s), s


def _product(x, codes, scales):
    q, s = _quantized(x)
    return (torch.mm(q, codes.float().t()) * s * scales).to(torch.bfloat16)


def _plain_linear(state):
    return _product(state["x"].float(), state["codes"], state["scales"])


def _plain_mlp(state):
    inter = state["case"]["inter"]
    gate_up = _product(state["x"].float(), state["w13"], state["s13"]).float()
    gate, up = gate_up[:, :inter], gate_up[:, inter:]
    act = (gate / (1.0 + torch.exp(-gate)) * up).to(torch.bfloat16)
    return _product(act.float(), state["w2"], state["s2"])


def _plain_order(state):
    """(positions [n, topk], -1: not here; counts [local])."""
    case, ids = state["case"], state["ids"]
    here = (ids >= 0) & (ids < case["local"])
    key = torch.where(here, ids, torch.full_like(ids, case["local"])).reshape(-1).long()
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.shape[0], device=order.device)
    place = torch.where(here.reshape(-1), place, torch.full_like(place, -1)).view_as(ids)
    counts = torch.bincount(key, minlength=case["local"] + 1)[: case["local"]]
    return place.to(torch.int32), counts.to(torch.int32)


def _plain_sort(state):
    case, x, rows, weights = state["case"], state["x"], state["rows"], state["weights"]
    place, counts = _plain_order(state)
    here, at = place >= 0, place.clamp_min(0).long()
    token = torch.arange(case["n"], device=x.device)[:, None].expand_as(place)
    moved = torch.zeros_like(rows)
    moved[at[here]] = x[token[here]]
    w = weights * here
    picked = rows[at].float()
    out = (picked * w[..., None]).sum(1).to(rows.dtype)
    if not case["train"]:
        return moved, place, counts, out
    g_out = state["g_out"].float()
    d_x = (state["g_rows"][at].float() * here[..., None]).sum(1).to(x.dtype)
    d_rows = torch.zeros_like(rows)
    d_rows[at[here]] = (w[..., None] * g_out[:, None, :]).to(rows.dtype)[here]
    d_w = (picked * g_out[:, None, :]).sum(-1) * here
    return moved, place, counts, out, d_x, d_rows, d_w


def _unit(v):
    """(v over its root mean square, one over that)."""
    r = 1.0 / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)
    return v * r, r


def _unit_grad(g, unit, r):
    """The gradient by v from that by _unit(v)[0]."""
    return r * (g - unit * (g * unit).mean(-1, keepdim=True))


def _plain_norm(state):
    case = state["case"]
    x, y, scale = state["x"].float(), state["y"].float(), case["scale"]
    gate, w_pre, w_post, w_next = (None if state[k] is None else state[k].float() for k in ("gate", "w_pre", "w_post", "w_next"))
    dtype, outs = state["x"].dtype, []
    if case["pre"]:
        unit_x, r_x = _unit(x)
        outs.append((unit_x * w_pre).to(dtype))
    unit_y, r_y = _unit(y) if case["post"] else (y, None)
    post = unit_y * w_post if case["post"] else y
    gated = post * scale if gate is None else post * gate * scale
    h = x + gated
    outs.append(h.to(dtype))
    if case["next"]:
        unit_h, r_h = _unit(h)
        outs.append((unit_h * w_next).to(dtype))
    if not case["train"]:
        return tuple(outs)
    d = state["g_h"].float()
    grads = dict.fromkeys(LEAVES["norm"])
    if case["next"]:
        g = state["g_next"].float()
        grads["w_next"] = (g * unit_h).sum(0)
        d = d + _unit_grad(g * w_next, unit_h, r_h)
    d_post = d * scale if gate is None else d * gate * scale
    if gate is not None:
        g = d * post * scale
        grads["gate"] = {"channel": lambda: g.sum(0), "token": lambda: g.sum(-1, keepdim=True), "element": lambda: g}[case["gate"]]()
    if case["post"]:
        grads["w_post"] = (d_post * unit_y).sum(0)
        grads["y"] = _unit_grad(d_post * w_post, unit_y, r_y)
    else:
        grads["y"] = d_post
    if case["pre"]:
        g = state["g_pre"].float()
        grads["w_pre"] = (g * unit_x).sum(0)
        # the residual and the norm before the block each give a gradient of their own, which are added up
        d = d.to(dtype).float() + _unit_grad(g * w_pre, unit_x, r_x).to(dtype).float()
    grads["x"] = d
    return tuple(outs) + tuple(grads[k].to(state[k].dtype) for k in LEAVES["norm"] if grads[k] is not None)


# ---------------------------------------------------------------- what a pass needs
def work(case):
    n = case["n"]
    if case["op"] == "linear":
        k, out = case["k"], case["out"]
        return {"bytes": n * k * 2 + out * k + out * 4 + n * out * 2, "flops": 2 * n * out * k}
    if case["op"] == "mlp":
        h, i = case["hidden"], case["inter"]
        return {"bytes": n * h * 4 + 3 * h * i + (2 * i + h) * 4, "flops": 6 * n * h * i}
    h, size = case["hidden"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "sort":
        # the rows that are here (of a uniform choice), moved there and back
        pairs = n * case["topk"]
        here = (n - case["padded"]) * case["topk"] * case["local"] // case["experts"]
        row, small = h * size, pairs * 12 + case["local"] * 4
        if not case["train"]:
            return {"bytes": 2 * (n + here) * row + small, "flops": 2 * here * h}
        # x, sorted, rows, out; then g_rows, dx, g_out, rows again with its gradient, and the weights'
        return {"bytes": (4 * n + 3 * pairs + 2 * here) * row + small + pairs * 8, "flops": 7 * here * h}
    row, params = n * h * size, h * (4 if case["wide"] else size)
    gate = {"none": 0, "channel": params, "token": params * n // h, "element": params * n}[case["gate"]]
    weights = params * (case["pre"] + case["post"] + case["next"])
    passes = 3 + case["pre"] + case["next"]  # x, y, h and the norms
    if not case["train"]:
        return {"bytes": passes * row + weights + gate, "flops": 6 * passes * n * h}
    # the gradients of what came out, in; those of x and y, out
    return {"bytes": (passes + 3 + case["pre"] + case["next"]) * row + 2 * (weights + gate), "flops": 18 * passes * n * h}


# ---------------------------------------------------------------- the results in 64 bits
def exact(case, seed):
    return {"linear": _exact_linear, "mlp": _exact_mlp, "sort": _exact_sort, "norm": _exact_norm}[case["op"]](
        case, INPUTS[case["op"]](case, seed))


def _exact_product(x, codes, scales):
    """Codes by the definition, whose quotients are fp32's; the rest in 64 bits."""
    top = x.float().abs().max(dim=-1).values.clamp(min=1e-10)
    s = torch.div(top, torch.full_like(top, 127.0))
    q = torch.div(x.float(), s.unsqueeze(1)).round().double()
    return q @ codes.double().t().contiguous() * torch.outer(s.double(), scales.double())


def _exact_linear(case, data):
    return _exact_product(data["x"], data["codes"], data["scales"])


def _exact_mlp(case, data):
    gate, up = _exact_product(data["x"], data["w13"], data["s13"]).to(torch.bfloat16).double().chunk(2, dim=1)
    act = (gate * torch.sigmoid(gate) * up).to(torch.bfloat16)
    return _exact_product(act, data["w2"], data["s2"])


def _exact_sort(case, data):
    ids, n, topk = data["ids"].long().cpu(), case["n"], case["topk"]
    pairs = [torch.nonzero(ids.reshape(-1) == e)[:, 0] for e in range(case["local"])]
    counts = torch.tensor([p.numel() for p in pairs], dtype=torch.int32)
    pairs = torch.cat(pairs)
    place = torch.full((n * topk,), -1, dtype=torch.int32)
    place[pairs] = torch.arange(pairs.numel(), dtype=torch.int32)
    pairs, dev = pairs.cuda(), data["x"].device
    x, rows, w = (data[k].double().requires_grad_(case["train"]) for k in ("x", "rows", "weights"))
    sort = torch.zeros(n * topk, case["hidden"], dtype=torch.float64, device=dev)
    sort = sort.index_copy(0, torch.arange(pairs.numel(), device=dev), x.index_select(0, pairs // topk))
    back = rows[: pairs.numel()] * w.reshape(-1).index_select(0, pairs)[:, None]
    out = torch.zeros(n, case["hidden"], dtype=torch.float64, device=dev).index_add(0, pairs // topk, back)
    result = (sort.detach(), place.view(n, topk).cuda(), counts.cuda(), out.detach())
    if not case["train"]:
        return result
    return result + torch.autograd.grad((sort, out), (x, rows, w), (data["g_rows"].double(), data["g_out"].double()))


def _exact_rms(v, weight):
    return v * torch.rsqrt(v.pow(2).sum(-1, keepdim=True) / v.shape[-1] + EPS) * weight


def _exact_norm(case, data):
    leaf = {k: data[k].double().requires_grad_(case["train"]) for k in LEAVES["norm"] if data[k] is not None}
    outs, given = [], []
    if case["pre"]:
        outs.append(_exact_rms(leaf["x"], leaf["w_pre"]))
        given.append(data.get("g_pre"))
    block = _exact_rms(leaf["y"], leaf["w_post"]) if case["post"] else leaf["y"]
    if "gate" in leaf:
        block = leaf["gate"] * block
    outs.append(leaf["x"] + case["scale"] * block)
    given.append(data.get("g_h"))
    if case["next"]:
        outs.append(_exact_rms(outs[-1], leaf["w_next"]))
        given.append(data.get("g_next"))
    result = tuple(v.detach() for v in outs)
    if not case["train"]:
        return result
    return result + torch.autograd.grad(outs, list(leaf.values()), [g.double() for g in given])
