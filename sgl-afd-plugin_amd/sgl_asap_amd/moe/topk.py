"""The top-k output the expert call takes, with the reference's field names.

The reference passes SGLang's ``StandardTopKOutput(topk_weights, topk_ids, router_logits)``
(``python/sgl_asap_plugin/srt/managers/scheduler.py:410-412``;
``srt/model_executor/runner/ffn_cuda_graph_runner.py:57``). SGLang is not a dependency here,
so the same three-field tuple is defined locally; any object with ``topk_weights`` and
``topk_ids`` attributes is accepted where it is consumed.

``select_experts`` makes that output from a router's logits (``afd_topk``; the reference
leaves it to the serving engine), with its gradient; ``TopK`` is the module form, with the argument
names that the engine's models use:

    s   = softmax(l), sigmoid(l) or sqrt(softplus(l))
    c   = l, or s + correction_bias (in 64 bits)        the choice value
    ids = the top_k largest c (equal values: lowest index first), with expert groups only those
          of the topk_group best groups; a group's value is its largest c, with a bias the sum of its two largest
    w   = routed_scaling_factor * s[ids] (/ the sum of s[ids] if renormalize)
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from .. import _lib


class StandardTopKOutput(NamedTuple):
    topk_weights: torch.Tensor  # f32 [n, k], routed scaling already applied
    topk_ids: torch.Tensor  # i32 [n, k], global expert ids
    router_logits: Optional[torch.Tensor] = None


def format_is_standard(topk_output) -> bool:
    """``TopKOutputChecker.format_is_standard`` as the dispatcher uses it
    (``srt/layers/moe/token_dispatcher/asap.py:60``): explicit ids and weights."""
    return hasattr(topk_output, "topk_ids") and hasattr(topk_output, "topk_weights")


SCORINGS = {"softmax": _lib.AFD_SCORE_SOFTMAX, "sigmoid": _lib.AFD_SCORE_SIGMOID,
            "sqrtsoftplus": _lib.AFD_SCORE_SQRTSOFTPLUS}
LOGITS_FORMATS = {torch.float32: _lib.AFD_LOGITS_F32, torch.bfloat16: _lib.AFD_LOGITS_BF16}


def launch(name: str, device: torch.device, *args) -> None:
    """``_lib.call`` on ``device``'s current stream, with ``device`` current."""
    if torch.jit.is_tracing() or get_proxy_mode() is not None:
        raise NotImplementedError(f"{name} cannot be traced: the graph would hold the results' memory, not what writes it")
    # (the plain bindings: torch.cuda's wrappers of these two cost a microsecond each)
    index = device.index
    if index == torch._C._cuda_getDevice():
        return _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def fit_ints(*sizes: int) -> None:
    """Refuses sizes that a C int of the entry points would cut to its 32 bits."""
    if max(sizes) > 0x7FFFFFFF or min(sizes) < -0x80000000:
        raise ValueError(f"sizes must fit 32 bits, got {sizes}")


@lru_cache(maxsize=256)
def router_cfg(num_experts: int, top_k: int, scoring: str, renormalize: bool, groups: int, keep: int, scale: float,
               dtype: torch.dtype):
    """A pointer to the router's C config."""
    if scoring not in SCORINGS:
        raise NotImplementedError(f"scoring {scoring!r} (supported: {sorted(SCORINGS)})")
    if dtype not in LOGITS_FORMATS:
        raise TypeError(f"router logits must be float32 or bfloat16, got {dtype}")
    fit_ints(num_experts, top_k, groups, keep)
    cfg = _lib.AfdRouterCfg(num_experts, top_k, SCORINGS[scoring], groups, keep, int(renormalize), scale,
                            LOGITS_FORMATS[dtype])
    return ctypes.pointer(cfg)


def matrix_rows(t: torch.Tensor):
    """(t [n, columns] with contiguous rows, their stride in elements)."""
    n, columns = t.shape
    if n > 0x7FFFFFFF:
        fit_ints(n)
    if t.is_contiguous():
        return t, columns
    if n == 1 or t.stride(1) != 1 or t.stride(0) < columns:
        return t.contiguous(), columns
    return t, t.stride(0)


def logit_rows(logits: torch.Tensor):
    if logits.dim() != 2:
        raise ValueError(f"router logits must be [n, num_experts], got {tuple(logits.shape)}")
    return matrix_rows(logits)


def on_device(name: str, t: Optional[torch.Tensor], dtype: torch.dtype, shape: tuple, device) -> int:
    """The address of an optional argument, checked (0: not given)."""
    if t is None:
        return 0
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {shape}, got {tuple(t.shape)} strides {t.stride()}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other arguments on {device}")
    return t.data_ptr()


def need_gpu(name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU, got {t.device}: there is no CPU path")


def no_tangent(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses tensors that carry a tangent, which a launch would drop (one needs no gradient, nor gradients enabled)."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # no level is open: spares the calls
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no forward-mode derivative")


def _groups(num_expert_group: Optional[int], topk_group: Optional[int]):
    if num_expert_group is None and topk_group is None:
        return 0, 0
    if num_expert_group is None or topk_group is None:
        raise ValueError("num_expert_group and topk_group come together")
    if num_expert_group < 1:
        raise ValueError(f"num_expert_group must be positive, got {num_expert_group}")
    return num_expert_group, topk_group


def choice_cfg(logits, top_k, scoring, renormalize, num_expert_group, topk_group, routed_scaling_factor):
    if logits.dim() != 2:
        raise ValueError(f"router logits must be [n, num_experts], got {tuple(logits.shape)}")
    groups, keep = _groups(num_expert_group, topk_group)
    scale = 1.0 if routed_scaling_factor is None else float(routed_scaling_factor)
    return router_cfg(logits.shape[1], top_k, scoring, bool(renormalize), groups, keep, scale, logits.dtype)


def choose(cfg, top_k, logits, bias, valid):
    """(ids, weights) of ``afd_topk``."""
    need_gpu("router_logits", logits)
    logits, ld = logit_rows(logits)
    n, experts = logits.shape
    dev = logits.device
    bias_ptr = on_device("correction_bias", bias, torch.float32, (experts,), dev)
    valid_ptr = on_device("valid", valid, torch.bool, (n,), dev)
    ids = torch.empty(n, top_k, dtype=torch.int32, device=dev)
    weights = torch.empty(n, top_k, dtype=torch.float32, device=dev)
    launch("afd_topk", dev, cfg, logits.data_ptr(), ld, bias_ptr, valid_ptr, n, ids.data_ptr(), weights.data_ptr())
    return logits, ids, weights


def router_grad(cfg, logits, ids, valid, gw, cu=None, counts=None, coef=None, gloss=None) -> torch.Tensor:
    """The gradient by the logits (``afd_router_grad``); logits as ``logit_rows`` gives them."""
    n, experts = logits.shape
    dev = logits.device
    out = torch.empty(n, experts, dtype=logits.dtype, device=dev)
    if gw is not None:
        gw = gw.to(torch.float32).contiguous()
    if coef is not None:
        gloss = gloss.to(torch.float32)

    def ptr(t):
        return t.data_ptr() if t is not None else None

    launch("afd_router_grad", dev, cfg, logits.data_ptr(), logits.stride(0) if n > 1 else experts, ptr(ids), ptr(valid),
           n, ptr(gw), ptr(cu), 1 if cu is None else cu.shape[0] - 1, ptr(counts), ptr(coef), ptr(gloss), out.data_ptr())
    return out


class _NoDerivative(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad, *made_from):
        ctx.mark_dirty(grad)
        return grad

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("the router's gradient has no derivative of its own (no second derivatives)")


def last(grad: torch.Tensor, *made_from: Optional[torch.Tensor]) -> torch.Tensor:
    """``grad``, which a backward made from ``made_from``. Where a second derivative can be asked for (the backward runs with
    gradients enabled) it is tied to them, whether or not the incoming gradients need one, by a node that raises."""
    return _NoDerivative.apply(grad, *made_from) if torch.is_grad_enabled() else grad


class _Select(torch.autograd.Function):
    """logits as ``logit_rows`` gives them: what the backward reads is then the input itself."""

    @staticmethod
    def forward(ctx, logits, cfg, top_k, bias, valid):
        rows, ids, weights = choose(cfg, top_k, logits, bias, valid)
        ctx.save_for_backward(rows, ids, valid)
        ctx.cfg = cfg
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return weights, ids

    @staticmethod
    def backward(ctx, gw, _):
        if gw is None:
            return None, None, None, None, None
        logits, ids, valid = ctx.saved_tensors
        return last(router_grad(ctx.cfg, logits, ids, valid, gw), logits, gw), None, None, None, None


def select_experts(
    router_logits: torch.Tensor,
    top_k: int,
    *,
    scoring: str = "softmax",
    renormalize: bool = True,
    correction_bias: Optional[torch.Tensor] = None,
    num_expert_group: Optional[int] = None,
    topk_group: Optional[int] = None,
    routed_scaling_factor: Optional[float] = None,
    valid: Optional[torch.Tensor] = None,
) -> StandardTopKOutput:
    """The experts of each row of ``router_logits`` [n, num_experts] (fp32 or bf16) and their weights,
    best first, on the device's current stream.

    ``correction_bias`` f32 [num_experts] takes part in the choice, not in the weights, and has no
    gradient. ``valid`` bool [n]: rows of False (a padded batch) get ids -1, which the expert call
    skips, and weights 0. A NaN logit counts as -inf, +inf as the largest float; a row of
    -inf alone gets weights 0, and so does one whose chosen scores are all below 2^-126 (not with ``renormalize`` and
    softmax, whose weights are ratios to the largest chosen score). The weights have a gradient by the logits (zero in
    invalid rows), once: second, forward-mode and traced derivatives are refused."""
    cfg = choice_cfg(router_logits, top_k, scoring, renormalize, num_expert_group, topk_group, routed_scaling_factor)
    no_tangent("select_experts", router_logits)
    if torch.is_grad_enabled() and router_logits.requires_grad:
        need_gpu("router_logits", router_logits)
        weights, ids = _Select.apply(logit_rows(router_logits)[0], cfg, top_k, correction_bias, valid)
    else:
        _, ids, weights = choose(cfg, top_k, router_logits, correction_bias, valid)
    return StandardTopKOutput(weights, ids, router_logits)


class TopK(torch.nn.Module):
    """``select_experts`` with a layer's settings. ``correction_bias`` is a buffer that moves with the module and stays in its
    fp32 when the module is cast."""

    def __init__(
        self,
        top_k: int,
        *,
        use_grouped_topk: bool = False,
        num_expert_group: Optional[int] = None,
        topk_group: Optional[int] = None,
        renormalize: bool = True,
        scoring_func: str = "softmax",
        correction_bias: Optional[torch.Tensor] = None,
        routed_scaling_factor: Optional[float] = None,
    ):
        super().__init__()
        if use_grouped_topk and (num_expert_group is None or topk_group is None):
            raise ValueError("use_grouped_topk needs num_expert_group and topk_group")
        if scoring_func not in SCORINGS:
            raise NotImplementedError(f"scoring {scoring_func!r} (supported: {sorted(SCORINGS)})")
        self.top_k = top_k
        self.register_buffer("correction_bias", correction_bias)
        self.settings = dict(scoring=scoring_func, renormalize=renormalize,
                             num_expert_group=num_expert_group if use_grouped_topk else None,
                             topk_group=topk_group if use_grouped_topk else None,
                             routed_scaling_factor=routed_scaling_factor)

    def _apply(self, fn, recurse=True):
        bias = self.correction_bias
        super()._apply(fn, recurse)
        if bias is not None and bias.dtype == torch.float32 != self.correction_bias.dtype:
            self.correction_bias = bias.to(self.correction_bias.device)
        return self

    def forward(self, router_logits: torch.Tensor, valid: Optional[torch.Tensor] = None) -> StandardTopKOutput:
        return select_experts(router_logits, self.top_k, correction_bias=self.correction_bias, valid=valid,
                              **self.settings)
