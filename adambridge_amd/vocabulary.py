"""A language model's ends: token ids to rows of an embedding.

On plain GPU tensors of float32 or bfloat16 the library's kernels compute it (csrc/abh_embed.hip, called by
csrc/abh_ops.cpp); elsewhere, and where an operation is traced, transformed or differentiated twice, torch operations do.
"""

from __future__ import annotations

import torch

from . import _hip
from .experts import _uncompiled
from .losses import _observed
from .norms import plain

__all__ = ["embed"]

_MOST_TOKENS, _MOST_WORDS, _MOST_HIDDEN = 1 << 30, 1 << 30, 1 << 22   # adambridge_embed's


# ----------------------------------------------------------------------- embed

def _torch_embed(ids, weight, scale, padding_idx):
    """The definition in torch operations."""
    vocab, hidden = weight.shape
    flat = ids.reshape(-1)
    inside = (flat >= 0) & (flat < vocab)
    wide = weight.to(torch.promote_types(weight.dtype, torch.float32))   # before the rows are taken: their gradients are summed so
    rows = wide.index_select(0, torch.where(inside, flat, 0))
    if padding_idx is not None:
        rows = torch.where((flat == padding_idx)[:, None], rows.detach(), rows)
    y = torch.where(inside[:, None], rows * scale, torch.nan)
    return y.to(weight.dtype).reshape(*ids.shape, hidden)


def _embed_backward(gout, ids, vocab, scale, padding_idx):
    """The embedding's gradient in torch operations, differentiable in turn."""
    flat = ids.reshape(-1)
    inside = (flat >= 0) & (flat < vocab)
    if padding_idx is not None:
        inside = inside & (flat != padding_idx)
    rows = gout.reshape(flat.numel(), gout.shape[-1]).float() * scale
    rows = torch.where(inside[:, None], rows, 0.0)
    total = rows.new_zeros(vocab, rows.shape[-1]).index_add(0, torch.where(inside, flat, 0), rows)
    return None, total.to(gout.dtype)


def embed(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """The rows of ``weight`` (``[vocab, hidden]``) that ``ids`` (int64 or int32, of any shape) name, times ``scale``:
    ``[*ids.shape, hidden]`` in ``weight``'s type, the product in FP32 and rounded once.

    The weight's gradient sums each word's rows in FP32, in an order of their own, times ``scale``; it is zero for words
    without tokens and for ``padding_idx``, whose rows themselves are as any other's.  An id outside the vocabulary gives a row
    of NaN, as a target outside it gives a loss of NaN, and has no gradient."""
    if torch.compiler.is_compiling():
        return _uncompiled(embed, ids, weight, scale, padding_idx)
    if weight.is_cuda:
        y = _hip.ops().embed(ids, weight, scale, padding_idx)
        if y is not None:
            return y
    if weight.dim() != 2 or not weight.is_floating_point() or not weight.shape[0] or not weight.shape[1]:
        raise ValueError(f"weight must be floating-point [vocab, hidden], not empty, got {weight.dtype} {tuple(weight.shape)}")
    if ids.dtype not in (torch.int64, torch.int32) or ids.device != weight.device:
        raise ValueError(f"ids must be int64 or int32 on {weight.device}, got {ids.dtype} on {ids.device}")
    if isinstance(scale, bool) or not isinstance(scale, (int, float)):
        raise ValueError(f"scale must be a number, got {scale!r}")
    if padding_idx is not None and (isinstance(padding_idx, bool) or not isinstance(padding_idx, int)
                                    or not 0 <= padding_idx < weight.shape[0]):
        raise ValueError(f"padding_idx must be None or an int from 0 to {weight.shape[0] - 1}, got {padding_idx!r}")
    if (not plain(weight) or type(ids) is not torch.Tensor or not 0 < ids.numel() <= _MOST_TOKENS or weight.shape[0] > _MOST_WORDS
            or weight.shape[1] > _MOST_HIDDEN or _observed()):
        return _torch_embed(ids, weight, float(scale), padding_idx)
    y = _hip.ops().embed(ids.contiguous(), weight.contiguous(), float(scale), padding_idx)
    return _torch_embed(ids, weight, float(scale), padding_idx) if y is None else y


# for the backward passes that the kernels do not take
BACKWARD = {"embed": _embed_backward}
