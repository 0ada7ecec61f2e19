"""Layer norm and its gradients by the library's kernels (csrc/abh_norm.hip).

Elsewhere than on plain GPU tensors of float32 or bfloat16, and where an operation is traced, transformed or
differentiated twice, the same values come from torch operations.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _hip
from .losses import _observed, _plain_backward

__all__ = ["layer_norm"]

_TYPES = (torch.bfloat16, torch.float32)
_MOST = 1 << 30   # rows and columns, adambridge_layer_norm's


def plain(*tensors: torch.Tensor | None) -> bool:
    """Whether the tensors' memory is what the kernels take: ordinary strided tensors of their types on one GPU."""
    device = tensors[0].device
    return device.type == "cuda" and all(
        t is None or type(t) in (torch.Tensor, torch.nn.Parameter) and t.dtype in _TYPES and t.device == device
        and t.layout == torch.strided and not t.is_neg() for t in tensors)


def _torch_layer_norm(x, weight, bias, eps):
    """The definition in torch operations, FP32 inside."""
    wide = torch.promote_types(x.dtype, torch.float32)
    cast = [t if t is None else t.to(wide) for t in (weight, bias)]
    return F.layer_norm(x.to(wide), x.shape[-1:], *cast, eps).to(x.dtype)


class _LayerNorm(torch.autograd.Function):
    """Keeps x and the rows' mean and rstd."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _hip.load().layer_norm(x, weight, bias, eps, with_stats=True)
        ctx.save_for_backward(x, weight, stats)
        ctx.eps, ctx.w_dtype = eps, (x if weight is None and bias is None else bias if weight is None else weight).dtype
        return y

    @staticmethod
    def backward(ctx, gout):
        x, weight, stats = ctx.saved_tensors
        wanted = ctx.needs_input_grad[:3]
        if _plain_backward(gout):
            return (*_hip.load().layer_norm_backward(gout.contiguous(), x, weight, stats, ctx.w_dtype, wanted), None)
        with torch.autocast(x.device.type, enabled=False):
            xf, g = x.float(), gout.float()
            var, mean = torch.var_mean(xf, 1, correction=0, keepdim=True)
            rstd = (var + ctx.eps).rsqrt()
            xh = (xf - mean) * rstd
            gw = g if weight is None else g * weight.float()
            dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
            return (dx.to(x.dtype), (g * xh).sum(0).to(ctx.w_dtype) if wanted[1] else None,
                    g.sum(0).to(ctx.w_dtype) if wanted[2] else None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of ``x`` over its last axis, times ``weight`` plus ``bias`` (each ``[x.shape[-1]]`` or None),
    in ``x``'s type; mean, variance and everything between them are FP32.

    ``weight`` and ``bias`` are of one type, ``x``'s or another.  Differentiable in all three; the backward pass
    reads ``x`` and the gradient once and sums the weight's and the bias's gradients over all rows in FP32.
    """
    cols = x.shape[-1] if x.dim() else 0
    if cols < 1 or not x.is_floating_point():
        raise ValueError(f"x must hold floating-point rows of one value or more, got {x.dtype} {tuple(x.shape)}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (tuple(t.shape) != (cols,) or not t.is_floating_point()):
            raise ValueError(f"{name} must be [{cols}] floating-point values, got {t.dtype} {tuple(t.shape)}")
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must be of one type, got {weight.dtype} and {bias.dtype}")
    rows = x.numel() // cols
    if not plain(x, weight, bias) or not 0 < rows <= _MOST or cols > _MOST or _observed():
        return _torch_layer_norm(x, weight, bias, eps)
    flat = x.reshape(rows, cols).contiguous()
    weight, bias = (t if t is None else t.contiguous() for t in (weight, bias))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(flat, weight, bias, eps).view(x.shape)
    return _hip.load().layer_norm(flat, weight, bias, eps, with_stats=False)[0].view(x.shape)
