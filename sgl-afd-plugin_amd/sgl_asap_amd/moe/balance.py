"""How a batch's tokens spread over the experts: counts, and the balance loss that a router is trained with.

No counterpart in the reference, which serves. Per sequence s with T counted rows, cnt_e the (token, k)
pairs that chose expert e and s' the row's scores divided by their sum (``select_experts``' scores):

    L = alpha * mean over the sequences with T > 0 of  E / (k T^2) * sum_e cnt_e * sum_t s'_te

``expert_counts`` counts alone (what a serving rank keeps to place its experts), ``balance_loss``
takes ids that were chosen elsewhere, ``select_and_balance`` chooses them in the same pass over the
logits; its backward writes the gradient of the weights and of the loss in one pass too. Sums run
in a fixed order: the same call gives the same bits. The counts are the caller's, to add up over ranks before
the backward too (it keeps its own); the loss and its gradient are those of this call's rows.

``cu_seqlens`` int32 [S + 1] (not decreasing) cuts the rows into sequences; rows outside them
belong to none. Without it all rows are one sequence. ``valid`` bool [n]: rows of False are not counted.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch

from .. import _lib
from .topk import (StandardTopKOutput, choice_cfg, fit_ints, last, launch, logit_rows, need_gpu, no_tangent, on_device,
                   router_cfg, router_grad)


@lru_cache(maxsize=1024)
def _workspace_bytes(n: int, experts: int, seqs: int) -> int:
    fit_ints(n, experts, seqs)
    out = ctypes.c_uint64()
    _lib.call("afd_balance_workspace", n, experts, seqs, ctypes.byref(out))
    return out.value


def _workspace(n: int, experts: int, seqs: int, device) -> torch.Tensor:
    # one call's own: calls on other streams and captured graphs each have theirs
    return torch.empty(_workspace_bytes(n, experts, seqs), dtype=torch.uint8, device=device)


def _sequences(cu: Optional[torch.Tensor], device) -> Tuple[int, int]:
    if cu is None:
        return 0, 1
    if cu.dim() != 1 or cu.shape[0] < 2:
        raise ValueError(f"cu_seqlens must be [S + 1] with S >= 1, got {tuple(cu.shape)}")
    return on_device("cu_seqlens", cu, torch.int32, tuple(cu.shape), device), cu.shape[0] - 1


def _check_ids(ids: torch.Tensor) -> torch.Tensor:
    if ids.dtype != torch.int32 or ids.dim() != 2:
        raise TypeError(f"topk_ids must be int32 [n, k], got {ids.dtype} {tuple(ids.shape)}")
    if ids.shape[1] > 0x7FFFFFFF:
        fit_ints(ids.shape[1])
    return ids.contiguous()


def expert_counts(topk_ids: torch.Tensor, num_experts: int, cu_seqlens: Optional[torch.Tensor] = None,
                  valid: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int32 [num_experts] (with ``cu_seqlens``: [S, num_experts]): how many entries of ``topk_ids`` int32
    [n, k] name each expert. Other ids (-1: no expert) are skipped."""
    need_gpu("topk_ids", topk_ids)
    ids = _check_ids(topk_ids)
    n, k = ids.shape
    dev = ids.device
    cu_ptr, seqs = _sequences(cu_seqlens, dev)
    valid_ptr = on_device("valid", valid, torch.bool, (n,), dev)
    ws = _workspace(n, num_experts, seqs, dev)
    counts = torch.empty((num_experts,) if cu_seqlens is None else (seqs, num_experts), dtype=torch.int32, device=dev)
    launch("afd_expert_counts", dev, ids.data_ptr(), n, k, num_experts, valid_ptr, cu_ptr, seqs, counts.data_ptr(),
           ws.data_ptr(), ws.numel())
    return counts


class _Balance(torch.autograd.Function):
    """(weights, ids, loss, counts) with ids chosen here, (loss, counts) for given ones; logits as ``logit_rows`` gives them:
    what the backward reads is then the input itself."""

    @staticmethod
    def forward(ctx, logits, cfg, top_k, alpha, bias, ids, cu, valid):
        logits, ld = logit_rows(logits)
        n, experts = logits.shape
        dev = logits.device
        cu_ptr, seqs = _sequences(cu, dev)
        valid_ptr = on_device("valid", valid, torch.bool, (n,), dev)
        ws = _workspace(n, experts, seqs, dev)
        counts = torch.empty((experts,) if cu is None else (seqs, experts), dtype=torch.int32, device=dev)
        coef = torch.empty(seqs, dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        chosen = ids is None
        if chosen:
            bias_ptr = on_device("correction_bias", bias, torch.float32, (experts,), dev)
            ids = torch.empty(n, top_k, dtype=torch.int32, device=dev)
            weights = torch.empty(n, top_k, dtype=torch.float32, device=dev)
            launch("afd_topk_balance", dev, cfg, logits.data_ptr(), ld, bias_ptr, valid_ptr, cu_ptr, seqs, n, alpha,
                   ids.data_ptr(), weights.data_ptr(), counts.data_ptr(), coef.data_ptr(), loss.data_ptr(),
                   ws.data_ptr(), ws.numel())
        else:
            launch("afd_balance", dev, cfg, logits.data_ptr(), ld, ids.data_ptr(), valid_ptr, cu_ptr, seqs, n, alpha,
                   counts.data_ptr(), coef.data_ptr(), loss.data_ptr(), ws.data_ptr(), ws.numel())
        # counts of the backward's own: the caller's may be added up over ranks before it, by collectives that
        # autograd does not see
        own = counts.clone() if ctx.needs_input_grad[0] else None
        ctx.save_for_backward(logits, ids if chosen else None, cu, valid, own, coef)
        ctx.cfg = cfg
        ctx.set_materialize_grads(False)
        if chosen:
            ctx.mark_non_differentiable(ids, counts)
            return weights, ids, loss, counts
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    def backward(ctx, *grads):
        logits, ids, cu, valid, counts, coef = ctx.saved_tensors
        gw, gloss = (grads[0], grads[2]) if ids is not None else (None, grads[0])
        grad = None
        if gw is not None or gloss is not None:
            with_loss = (None,) * 4 if gloss is None else (cu, counts, coef, gloss)
            grad = last(router_grad(ctx.cfg, logits, ids, valid, gw, *with_loss), logits, gw, gloss)
        return (grad,) + (None,) * 7


def balance_loss(router_logits: torch.Tensor, topk_ids: torch.Tensor, *, alpha: float, scoring: str = "softmax",
                 cu_seqlens: Optional[torch.Tensor] = None,
                 valid: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, fp32 scalar; counts, int32 [num_experts] or [S, num_experts]) of ``router_logits`` [n,
    num_experts] (fp32 or bf16) and the ids that were chosen. The loss has a gradient by the logits (the counts do not)."""
    ids = _check_ids(topk_ids)
    if router_logits.dim() != 2 or ids.shape[0] != router_logits.shape[0]:
        raise ValueError(f"{ids.shape[0]} rows of ids for logits {tuple(router_logits.shape)}")
    if ids.device != router_logits.device:
        raise ValueError(f"topk_ids is on {ids.device}, router_logits on {router_logits.device}")
    cfg = router_cfg(router_logits.shape[1], ids.shape[1], scoring, False, 0, 0, 1.0, router_logits.dtype)
    need_gpu("router_logits", router_logits)
    no_tangent("balance_loss", router_logits)
    return _Balance.apply(logit_rows(router_logits)[0], cfg, ids.shape[1], float(alpha), None, ids, cu_seqlens, valid)


def select_and_balance(
    router_logits: torch.Tensor,
    top_k: int,
    *,
    alpha: float,
    scoring: str = "softmax",
    renormalize: bool = True,
    correction_bias: Optional[torch.Tensor] = None,
    num_expert_group: Optional[int] = None,
    topk_group: Optional[int] = None,
    routed_scaling_factor: Optional[float] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
    valid: Optional[torch.Tensor] = None,
) -> Tuple[StandardTopKOutput, torch.Tensor, torch.Tensor]:
    """``select_experts`` and ``balance_loss`` of what it chose, as one pass over the logits each way:
    (top-k output, loss, counts)."""
    cfg = choice_cfg(router_logits, top_k, scoring, renormalize, num_expert_group, topk_group, routed_scaling_factor)
    need_gpu("router_logits", router_logits)
    no_tangent("select_and_balance", router_logits)
    weights, ids, loss, counts = _Balance.apply(logit_rows(router_logits)[0], cfg, top_k, float(alpha), correction_bias, None,
                                                cu_seqlens, valid)
    return StandardTopKOutput(weights, ids, router_logits), loss, counts
