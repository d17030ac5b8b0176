"""The router's definitions in 64 bits with plain torch operations (CPU): what the tests compare against."""

import math

import torch

SCORINGS = ("softmax", "sigmoid", "sqrtsoftplus")


def canon(logits):
    """NaN counts as -inf, +inf as the largest fp32."""
    z = logits.detach().cpu().double()
    z = torch.where(z.isnan(), torch.full_like(z, -math.inf), z)
    return z.clamp(max=torch.finfo(torch.float32).max)


def scores(z, scoring):
    if scoring == "softmax":
        top = z.amax(1, keepdim=True)
        e = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = e.sum(1, keepdim=True)
        return e / torch.where(total == 0, torch.ones_like(total), total)
    if scoring == "sigmoid":
        return torch.sigmoid(z)
    return torch.sqrt(torch.log1p(torch.exp(-z.abs())) + z.clamp(min=0.0))


def choose(z, top_k, scoring, bias=None, groups=0, keep=0):
    """ids [n, top_k] row by row, best first, the lowest index of equals."""
    choice = z if bias is None else scores(z, scoring) + bias.cpu().double()
    choice = torch.where(choice.isnan(), torch.full_like(choice, -math.inf), choice)
    out = []
    for row in choice.tolist():
        allowed = list(range(len(row)))
        if groups > 1:
            size = len(row) // groups
            value = []
            for g in range(groups):
                best = sorted(row[g * size : (g + 1) * size], reverse=True)
                v = best[0] if bias is None or size == 1 else best[0] + best[1]
                value.append(-math.inf if v != v else v)
            kept = set(sorted(range(groups), key=lambda g: (-value[g], g))[:keep])
            allowed = [e for e in allowed if e // size in kept]
        out.append(sorted(allowed, key=lambda e: (-row[e], e))[:top_k])
    return torch.tensor(out, dtype=torch.int64).reshape(len(out), top_k)


def weights(z, ids, scoring, renorm, scale):
    s = scores(z, scoring).gather(1, ids)
    if renorm:
        total = s.sum(1, keepdim=True)
        s = s / torch.where(total == 0, torch.ones_like(total), total)
    return s * scale


def sequences(n, cu):
    return [(0, n)] if cu is None else list(zip(cu, cu[1:]))


def counts(ids, experts, cu=None, valid=None):
    rows = []
    for lo, hi in sequences(ids.shape[0], cu):
        part = ids[lo:hi] if valid is None else ids[lo:hi][valid[lo:hi]]
        part = part.reshape(-1)
        part = part[(part >= 0) & (part < experts)]
        rows.append(torch.bincount(part.long(), minlength=experts))
    return torch.stack(rows)


def balance(z, ids, scoring, alpha, cu=None, valid=None):
    n, experts = z.shape
    s = scores(z, scoring)
    total = s.sum(1, keepdim=True)
    share = s / torch.where(total == 0, torch.ones_like(total), total)
    cnt = counts(ids, experts, cu, valid).double()
    terms = []
    for i, (lo, hi) in enumerate(sequences(n, cu)):
        part = share[lo:hi] if valid is None else share[lo:hi][valid[lo:hi]]
        t = part.shape[0]
        if t:
            terms.append(experts / (ids.shape[1] * t * t) * (cnt[i] * part.sum(0)).sum())
    return alpha * torch.stack(terms).mean() if terms else z.sum() * 0.0


def grads(logits, ids, scoring, renorm=True, scale=1.0, gw=None, gl=None, alpha=0.0, cu=None, valid=None):
    """Gradient by the logits of sum(gw * weights) + gl * loss."""
    z = canon(logits).requires_grad_()
    total = z.sum() * 0.0 if torch.isfinite(z.detach()).all() else torch.zeros((), dtype=torch.float64)
    if gw is not None:
        w = weights(z, ids, scoring, renorm, scale)
        if valid is not None:
            w = w * valid[:, None]
        total = total + (w * gw.cpu().double()).sum()
    if gl is not None:
        total = total + gl * balance(z, ids, scoring, alpha, cu, valid)
    (g,) = torch.autograd.grad(total, z)
    return g
