"""Expert ids and scores from the router's logits: host side of ``dm_select_experts`` / ``_bwd`` (csrc/select_experts.cu)."""

from __future__ import annotations

from typing import Literal

import torch

from . import _native as nat
from ._bf16 import _plain_execution
from ._call import differentiable_once, on_device, refuse_tangents

MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 32, 32
_FLOATS = (torch.float32, torch.bfloat16)
_LARGEST = torch.finfo(torch.float32).max  # what the kernel takes the scale as


def _forward(logits, o):
    T, E = logits.shape
    top_k, sigmoid, bias, groups, kept, group_top, renormalize, scale, mask, ids_dtype, scores_dtype = o
    ids = torch.empty((T, top_k), dtype=ids_dtype, device=logits.device)
    scores = torch.empty((T, top_k), dtype=scores_dtype, device=logits.device)
    nat.check(nat.lib.dm_select_experts(
        logits.data_ptr(), logits.dtype is torch.bfloat16, logits.stride(0), T, E, top_k, sigmoid, nat.ptr(bias), groups, kept,
        group_top, renormalize, scale, nat.ptr(mask), ids.data_ptr(), ids_dtype is torch.int64, scores.data_ptr(),
        scores_dtype is torch.bfloat16, nat.stream_ptr()), "dm_select_experts", int(T > 0))
    return ids, scores


def _forward_seen(logits, o):
    """``_forward``, through the registered operator where something acts on operators."""
    top_k, sigmoid, bias, groups, kept, group_top, renormalize, scale, mask, ids_dtype, scores_dtype = o
    if _plain_execution(logits, logits if bias is None else bias, logits if mask is None else mask):
        with on_device(logits.device):
            return _forward(logits, o)
    return torch.ops.dist_moe.select_experts(logits, bias, mask, top_k, _name(sigmoid), groups, kept, group_top, renormalize, scale,
                                             ids_dtype, scores_dtype)


def _name(sigmoid: bool) -> str:
    return "sigmoid" if sigmoid else "softmax"


class _SelectExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, options):
        ids, scores = _forward_seen(logits, options)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, ids)
        ctx.options = options
        return ids, scores

    @staticmethod
    def backward(ctx, _, grad_scores):
        if grad_scores is None:
            return None, None
        logits, ids = ctx.saved_tensors
        if not torch.is_grad_enabled():
            return _backward_seen(ctx.options, logits, ids, grad_scores), None
        with torch.no_grad():
            grad = _backward_seen(ctx.options, logits, ids, grad_scores)
        return *differentiable_once("select_experts", (grad,), (grad_scores, logits)), None


def _backward_seen(options, logits, ids, grad_scores):
    _, sigmoid, _, _, _, _, renormalize, scale, _, _, _ = options
    if _plain_execution(logits, ids, grad_scores):
        return _backward(logits, ids, grad_scores, sigmoid, renormalize, scale)
    return torch.ops.dist_moe.select_experts_backward(logits, ids, grad_scores, _name(sigmoid), renormalize, scale)


def _backward(logits, ids, grad_scores, sigmoid, renormalize, scale):
    (T, E), top_k = logits.shape, ids.shape[1]
    with on_device(logits.device):
        grad_scores = grad_scores.contiguous()
        out = torch.empty_like(logits) if logits.is_contiguous() else torch.empty((T, E), dtype=logits.dtype, device=logits.device)
        nat.check(nat.lib.dm_select_experts_bwd(
            logits.data_ptr(), logits.dtype is torch.bfloat16, logits.stride(0), T, E, top_k, sigmoid, renormalize, scale,
            ids.data_ptr(), ids.dtype is torch.int64, grad_scores.data_ptr(), grad_scores.dtype is torch.bfloat16,
            out.data_ptr(), nat.stream_ptr()), "dm_select_experts_bwd", int(T > 0))
    return out


def _check(logits_TE, top_k, score, bias_E, num_groups, num_kept_groups, group_top, renormalize, scale, token_mask_T, ids_dtype,
           scores_dtype) -> None:
    if not isinstance(logits_TE, torch.Tensor) or logits_TE.dtype not in _FLOATS:
        raise TypeError("logits_TE must be a torch.float32 or torch.bfloat16 tensor")
    if logits_TE.ndim != 2:
        raise ValueError("logits_TE must have shape [T, E]")
    T, E = logits_TE.shape
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"logits_TE must name 1..{MAX_EXPERTS} experts")
    if not type(top_k) is type(num_groups) is type(num_kept_groups) is type(group_top) is int:
        for name, value in (("top_k", top_k), ("num_groups", num_groups), ("num_kept_groups", num_kept_groups), ("group_top", group_top)):
            if isinstance(value, bool) or not isinstance(value, int):
                raise TypeError(f"{name} must be an integer")
    if not 1 <= top_k <= min(E, MAX_TOP_K):
        raise ValueError(f"top_k must be in [1, {min(E, MAX_TOP_K)}]")
    if not 1 <= num_groups <= MAX_GROUPS or E % num_groups:
        raise ValueError(f"num_groups must be in [1, {MAX_GROUPS}] and divide the number of experts")
    if not 1 <= num_kept_groups <= num_groups or group_top not in (1, 2):
        raise ValueError("num_kept_groups must be in [1, num_groups] and group_top 1 or 2")
    if top_k > num_kept_groups * (E // num_groups):
        raise ValueError("top_k exceeds the experts of the kept groups")
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    if not isinstance(renormalize, bool):
        raise TypeError("renormalize must be a bool")
    if not isinstance(scale, (int, float)) or not abs(scale) <= _LARGEST:
        raise ValueError("scale must be finite, in float32 too")
    if ids_dtype not in (torch.int32, torch.int64):
        raise TypeError("ids_dtype must be torch.int32 or torch.int64")
    if scores_dtype not in _FLOATS:
        raise TypeError("scores_dtype must be torch.float32 or torch.bfloat16")
    device = logits_TE.device
    if bias_E is not None:
        if not isinstance(bias_E, torch.Tensor) or bias_E.dtype != torch.float32:
            raise TypeError("bias_E must be a torch.float32 tensor")
        if bias_E.shape != (E,):
            raise ValueError(f"bias_E must have shape [{E}]")
        if bias_E.requires_grad and torch.is_grad_enabled():
            raise ValueError("bias_E takes part in the choice alone and has no gradient")
    if token_mask_T is not None:
        if not isinstance(token_mask_T, torch.Tensor) or token_mask_T.dtype != torch.bool:
            raise TypeError("token_mask_T must be a torch.bool tensor")
        if token_mask_T.shape != (T,):
            raise ValueError(f"token_mask_T must have shape [{T}]")
    if (device.type != "cuda" or (bias_E is not None and bias_E.device != device)
            or (token_mask_T is not None and token_mask_T.device != device)):
        raise ValueError("all operation tensors must reside on the same CUDA device")


def _laid_out(logits_TE, bias_E, token_mask_T):
    """Other layouts are copied; rows of logits may lie apart."""
    if logits_TE.stride(1) != 1 and logits_TE.shape[1] > 1:
        logits_TE = logits_TE.contiguous()
    if bias_E is not None and not bias_E.is_contiguous():
        bias_E = bias_E.contiguous()
    if token_mask_T is not None and not token_mask_T.is_contiguous():
        token_mask_T = token_mask_T.contiguous()
    return logits_TE, bias_E, token_mask_T


def select_experts(logits_TE: torch.Tensor, top_k: int, *, score: Literal["softmax", "sigmoid"] = "softmax",
                   bias_E: torch.Tensor | None = None, num_groups: int = 1, num_kept_groups: int = 1, group_top: int = 2,
                   renormalize: bool = False, scale: float = 1.0, token_mask_T: torch.Tensor | None = None,
                   ids_dtype: torch.dtype = torch.int32, scores_dtype: torch.dtype = torch.float32):
    """Choose the experts of every token; returns ``(topk_expert_ids_TK, topk_scores_TK)`` as :func:`routed_experts` takes them.

    ``p`` is the softmax of a row of logits (float32 or bf16) or their sigmoid, and ``c = p + bias_E`` (float32, for the choice
    alone: it takes no gradient).  With ``num_groups`` > 1 the experts are consecutive groups of equal size, of which the
    ``num_kept_groups`` with the largest sums of their ``group_top`` (1 or 2) largest ``c`` remain.  The ids are the ``top_k`` largest
    ``c`` in falling order, equal ones by index, as in 64-bit arithmetic (without a bias by their logits); the scores ``scale * p``,
    with ``renormalize`` divided by the sum of the chosen ``p``.  The scores are differentiable in the logits.

    An expert whose logit or bias is -inf or NaN is not chosen.  Where fewer than ``top_k`` are left, and for tokens whose
    ``token_mask_T`` (bool) is false, ids are -1 and scores 0: the routed experts drop such routes.
    """
    _check(logits_TE, top_k, score, bias_E, num_groups, num_kept_groups, group_top, renormalize, scale, token_mask_T, ids_dtype,
           scores_dtype)
    refuse_tangents("select_experts", logits_TE, bias_E)
    logits_TE, bias_E, token_mask_T = _laid_out(logits_TE, bias_E, token_mask_T)
    options = (top_k, score == "sigmoid", bias_E, num_groups, num_kept_groups, group_top, renormalize, float(scale), token_mask_T,
               ids_dtype, scores_dtype)
    if logits_TE.requires_grad and torch.is_grad_enabled():
        return _SelectExperts.apply(logits_TE, options)
    return _forward_seen(logits_TE, options)
