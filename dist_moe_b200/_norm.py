"""The residual's addition and the RMS norm in front of a layer, with MXFP8 rows for block-scaled experts.

Host side of ``dm_add_rmsnorm_fwd`` / ``_bwd`` (csrc/add_rmsnorm.cu).  The quantised rows are the packed rows that an MXFP8
inference call publishes, so that ``routed_experts`` takes them in place of bf16 tokens and copies instead of quantising.
"""

from __future__ import annotations

import dataclasses

import torch

from . import _native as nat
from ._bf16 import _plain_execution
from ._call import address, differentiable_once, on_device, refuse_tangents

_TYPES = (torch.bfloat16, torch.float32)
_TINY, _LARGEST = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max  # what the kernels take eps and the centre as


@dataclasses.dataclass(frozen=True, eq=False)
class QuantizedRows:
    """Tokens in MXFP8: ``packed`` uint8 ``[T, stride]``, a row being ``hidden_dim`` bytes E4M3, ``hidden_dim / 32`` scales
    E8M0 and padding to 16 bytes."""

    packed: torch.Tensor
    hidden_dim: int

    def __post_init__(self) -> None:
        t, D = self.packed, self.hidden_dim
        if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.device.type != "cuda":
            raise TypeError("packed must be a CUDA uint8 tensor")
        if isinstance(D, bool) or not isinstance(D, int) or D <= 0 or D % 32:
            raise ValueError("hidden_dim must be a positive multiple of 32")
        if t.ndim != 2 or t.shape[1] != _row_bytes(D) or not t.is_contiguous() or address(t) % 16:
            raise ValueError(f"packed must be a contiguous, 16-byte aligned tensor of shape [T, {_row_bytes(D)}]")

    @property
    def data(self) -> torch.Tensor:
        """The E4M3 values ``[T, hidden_dim]``, a view."""
        return self.packed[:, :self.hidden_dim].view(torch.float8_e4m3fn)

    @property
    def scales(self) -> torch.Tensor:
        """The scales' exponent bytes ``[T, hidden_dim / 32]``, a view: a block's values times ``2 ** (byte - 127)``."""
        return self.packed[:, self.hidden_dim:self.hidden_dim + self.hidden_dim // 32]

    def dequantize(self) -> torch.Tensor:
        """The rows' values as bf16 ``[T, hidden_dim]``: exact, but for values below 2 ** -133, which bf16 does not have."""
        if _plain_execution(self.packed):
            return _dequantize(self.packed, self.hidden_dim)
        return torch.ops.dist_moe.dequantize_mxfp8_rows(self.packed, self.hidden_dim)


def _dequantize(packed, D):
    T, stride = packed.shape
    with on_device(packed.device):
        out = torch.empty(T, D, dtype=torch.bfloat16, device=packed.device)
        nat.check(nat.lib.dm_dequant_mxfp8_rows(packed.data_ptr(), stride, T, D, out.data_ptr(), nat.stream_ptr()),
                  "dm_dequant_mxfp8_rows", int(T > 0))
    return out


def _row_bytes(dim: int) -> int:
    return (dim + dim // 32 + 15) // 16 * 16


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with its rows' elements next to one another; rows may lie apart."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _rows_and_result(t: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``_rows`` of ``t``, and a contiguous tensor for a result of its shape."""
    if t.is_contiguous():
        return t, torch.empty_like(t)
    return _rows(t), torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _forward(x, residual, weight, eps, center, want_rstd, quantize):
    T, D = x.shape
    device = x.device
    if quantize:  # the quantiser's 16-byte pieces
        x, weight = _aligned(x), _aligned(weight)
        residual = None if residual is None else _aligned(residual)
    x, y = _rows_and_result(x)
    total = residual_ptr = total_ptr = None
    residual_stride = residual_f32 = 0
    if residual is not None:
        residual, total = _rows_and_result(residual)
        residual_ptr, total_ptr, residual_stride = residual.data_ptr(), total.data_ptr(), residual.stride(0)
        residual_f32 = residual.dtype is torch.float32
    rstd = torch.empty(T, dtype=torch.float32, device=device) if want_rstd else None
    rows, stride = None, 0
    if quantize:
        stride = _row_bytes(D)
        rows = torch.empty((T, stride), dtype=torch.uint8, device=device)
    nat.check(nat.lib.dm_add_rmsnorm_fwd(
        x.data_ptr(), x.stride(0), residual_ptr, residual_f32, residual_stride, weight.data_ptr(), weight.dtype is torch.float32,
        center, eps, T, D, total_ptr, y.data_ptr(), None if rstd is None else rstd.data_ptr(),
        None if rows is None else rows.data_ptr(), stride, nat.stream_ptr()),
        "dm_add_rmsnorm_fwd", int(T > 0))
    return y, total, rstd, rows


def _forward_seen(x, residual, weight, eps, center, want_rstd, quantize):
    """``_forward``, through the registered operator where something acts on operators."""
    if _plain_execution(x, weight, x if residual is None else residual):
        with on_device(x.device):
            return _forward(x, residual, weight, eps, center, want_rstd, quantize)
    y, total, rstd, rows = torch.ops.dist_moe.add_rms_norm(x, residual, weight, float(eps), float(center), want_rstd, quantize)
    return y, None if residual is None else total, rstd if want_rstd else None, rows if quantize else None


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, center):
        y, total, rstd, _ = _forward_seen(x, residual, weight, eps, center, True, False)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if residual is None else total, weight, rstd)
        ctx.center = center
        return y if residual is None else (y, total)

    @staticmethod
    def backward(ctx, grad_y, grad_sum=None):
        want_x, want_residual, want_weight = ctx.needs_input_grad[:3]
        total, weight, rstd = ctx.saved_tensors
        if grad_y is None:  # the stream alone is differentiated
            if grad_sum is None:
                return None, None, None, None, None
            return (grad_sum.to(torch.bfloat16) if want_x else None, grad_sum if want_residual else None,
                    torch.zeros_like(weight) if want_weight else None, None, None)
        if not torch.is_grad_enabled():
            return *_backward_seen(ctx, grad_y, grad_sum, total, weight, rstd), None, None
        with torch.no_grad():
            gx, gr, gw = _backward_seen(ctx, grad_y, grad_sum, total, weight, rstd)
        gx, gr = differentiable_once("add_rms_norm", (gx, gr), (grad_y, grad_sum, total, weight))
        gw, = differentiable_once("add_rms_norm", (gw,), (grad_y, total if want_x or want_residual else None))
        return gx, gr, gw, None, None


def _backward_seen(ctx, grad_y, grad_sum, total, weight, rstd):
    want_x, want_residual, want_weight = ctx.needs_input_grad[:3]
    apart = total.dtype is torch.float32
    wanted = want_x or (want_residual and not apart), want_residual and apart, want_weight
    if _plain_execution(grad_y, total, weight):
        gx, gr, gw = _backward(grad_y, grad_sum, total, weight, rstd, ctx.center, *wanted)
    else:
        grads = torch.ops.dist_moe.add_rms_norm_backward(grad_y, grad_sum, total, weight, rstd, ctx.center, *wanted)
        gx, gr, gw = (g if want else None for g, want in zip(grads, wanted))
    return gx if want_x else None, (gr if apart else gx) if want_residual else None, gw


def _backward(grad_y, grad_sum, total, weight, rstd, center, want_bf16, want_float32, want_weight):
    T, D = grad_y.shape
    with on_device(grad_y.device):
        grad_y = grad_y.contiguous()
        if grad_sum is not None:
            grad_sum = grad_sum.contiguous()
        gx = torch.empty_like(grad_y) if want_bf16 else None
        gr = torch.empty_like(total) if want_float32 else None
        gw = partial = None
        if want_weight:
            gw = torch.empty_like(weight)
            partial = rstd.new_empty((nat.lib.dm_add_rmsnorm_shares(T, D), D))
        if T == 0:
            gw = gw.zero_() if want_weight else None
        else:
            nat.check(nat.lib.dm_add_rmsnorm_bwd(
                grad_y.data_ptr(), nat.ptr(grad_sum), total.data_ptr(), total.dtype is torch.float32, total.stride(0), weight.data_ptr(),
                weight.dtype is torch.float32, center, rstd.data_ptr(), T, D, nat.ptr(gx), nat.ptr(gr), nat.ptr(partial),
                nat.ptr(gw), nat.stream_ptr()), "dm_add_rmsnorm_bwd", 2 if want_weight else 1)
    return gx, gr, gw


def _check(x_TD, weight_D, residual_TD, eps, gain_center, quantize) -> None:
    if not isinstance(x_TD, torch.Tensor) or x_TD.dtype != torch.bfloat16:
        raise TypeError("x_TD must be a torch.bfloat16 tensor")
    if not isinstance(weight_D, torch.Tensor) or weight_D.dtype not in _TYPES:
        raise TypeError("weight_D must be a torch.bfloat16 or torch.float32 tensor")
    if residual_TD is not None and (not isinstance(residual_TD, torch.Tensor) or residual_TD.dtype not in _TYPES):
        raise TypeError("residual_TD must be a torch.bfloat16 or torch.float32 tensor")
    if x_TD.ndim != 2 or x_TD.shape[1] == 0:
        raise ValueError("x_TD must have shape [T, D] with D > 0")
    D = x_TD.shape[1]
    if weight_D.shape != (D,):
        raise ValueError(f"weight_D must have shape [{D}]")
    if residual_TD is not None and residual_TD.shape != x_TD.shape:
        raise ValueError(f"residual_TD must have the shape of x_TD, {tuple(x_TD.shape)}")
    device = x_TD.device
    if device.type != "cuda" or weight_D.device != device or (residual_TD is not None and residual_TD.device != device):
        raise ValueError("all operation tensors must reside on the same CUDA device")
    if not isinstance(eps, (int, float)) or not _TINY <= eps <= _LARGEST:
        raise ValueError("eps must be finite and positive, in float32 too")
    if not isinstance(gain_center, (int, float)) or not abs(gain_center) <= _LARGEST:
        raise ValueError("gain_center must be finite, in float32 too")
    if not isinstance(quantize, bool):
        raise TypeError("quantize must be a bool")
    if quantize and (D % 32 or D > 16384):
        raise ValueError("quantised rows need D to be a multiple of 32 and at most 16384")


def add_rms_norm(x_TD: torch.Tensor, weight_D: torch.Tensor, *, residual_TD: torch.Tensor | None = None, eps: float = 1e-6,
                 gain_center: float = 0.0, quantize: bool = False):
    """Add ``x_TD`` to the residual stream and normalise the sum for the next layer.

    ``sum = x + residual`` rounded to the residual's type (bf16 or float32; without a residual ``sum`` is ``x_TD`` itself) and
    ``y = bf16(sum / sqrt(mean(sum ** 2) + eps) * (weight + gain_center))``: the stored sum is what is normalised.  Returns
    ``(y_TD, sum_TD)``, differentiable in ``x_TD``, ``residual_TD`` and ``weight_D`` (bf16 or float32).  Rows may lie apart (a slice
    of a wider tensor); other layouts are copied.

    With ``quantize=True`` returns ``(y_TD, sum_TD, rows)``: ``rows`` are the MXFP8 :class:`QuantizedRows` of ``y_TD``, which
    :func:`routed_experts` takes on MXFP8 contexts in forward-only calls, with the result that ``y_TD`` gives.  They have no
    gradient: where one would be recorded the call raises.  ``hidden_dim`` must be a multiple of 32, at most 16384.
    """
    _check(x_TD, weight_D, residual_TD, eps, gain_center, quantize)
    grads = torch.is_grad_enabled() and (x_TD.requires_grad or weight_D.requires_grad
                                         or (residual_TD is not None and residual_TD.requires_grad))
    if quantize and grads:
        raise RuntimeError("quantised rows have no gradient: call add_rms_norm(quantize=True) under torch.no_grad()")
    refuse_tangents("add_rms_norm", x_TD, residual_TD, weight_D)
    if not weight_D.is_contiguous():
        weight_D = weight_D.contiguous()
    if grads:
        if residual_TD is None:
            kept = _rows(x_TD)  # what is saved is what the gradients depend on
            return _AddRmsNorm.apply(kept, None, weight_D, float(eps), float(gain_center)), x_TD
        return _AddRmsNorm.apply(x_TD, residual_TD, weight_D, float(eps), float(gain_center))
    y, total, _, rows = _forward_seen(x_TD, residual_TD, weight_D, eps, gain_center, False, quantize)
    if residual_TD is None:
        total = x_TD
    return (y, total, QuantizedRows(rows, int(x_TD.shape[1]))) if quantize else (y, total)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    if t.data_ptr() % 16 or (t.ndim == 2 and t.stride(0) * t.element_size() % 16):
        return t.clone(memory_format=torch.contiguous_format)
    return t
