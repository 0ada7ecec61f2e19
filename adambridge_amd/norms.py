"""Layer norm and its gradients by the library's kernels (csrc/abh_norm.hip, called by csrc/abh_ops.cpp).

Elsewhere than on plain GPU tensors of float32 or bfloat16, and where an operation is traced, transformed or
differentiated twice, the same values come from torch operations.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _hip
from .losses import _observed

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


def _backward(gout, x, weight, eps, want_x, want_w, want_b, w_dtype):
    """The gradients in torch operations, differentiable in turn."""
    with torch.autocast(x.device.type, enabled=False):
        xf, g = x.float(), gout.float()
        var, mean = torch.var_mean(xf, -1, correction=0, keepdim=True)
        rstd = (var + eps).rsqrt()
        xh = (xf - mean) * rstd
        gw = g if weight is None else g * weight.float()
        rows = tuple(range(x.dim() - 1))   # of none, a single row's sum is itself
        dx = dw = db = None
        if want_x:
            dx = (rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))).to(x.dtype)
        if want_w:
            dw = ((g * xh).sum(rows) if rows else g * xh).to(w_dtype)
        if want_b:
            db = (g.sum(rows) if rows else g).to(w_dtype)
        return dx, dw, db


BACKWARD = {"layer_norm": _backward}   # for the backward passes that the kernels do not take


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of ``x`` over its last axis, times ``weight`` plus ``bias`` (each ``[x.shape[-1]]`` or None),
    in ``x``'s type; mean, variance and everything between them are FP32.

    ``weight`` and ``bias`` are of one type, ``x``'s or another.  Differentiable in all three; the backward pass
    reads ``x`` and the gradient once and sums the weight's and the bias's gradients over all rows in FP32.
    """
    if x.is_cuda and not torch.compiler.is_compiling():
        y = _hip.ops().layer_norm(x, weight, bias, float(eps))
        if y is not None:
            return y
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
    y = _hip.ops().layer_norm(*(t if t is None else t.contiguous() for t in (x, weight, bias)), float(eps))
    return _torch_layer_norm(x, weight, bias, eps) if y is None else y
