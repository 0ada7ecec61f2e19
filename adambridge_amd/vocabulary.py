"""A language model's ends: token ids to rows of an embedding, and rows to their losses over the vocabulary.

On plain GPU tensors of float32 or bfloat16 the library's kernels compute it (csrc/abh_embed.hip, csrc/abh_head.hip, called by
csrc/abh_ops.cpp); elsewhere, and where an operation is traced, transformed or differentiated twice, torch operations do.
"""

from __future__ import annotations

import torch

from . import _hip
from .experts import _uncompiled
from .losses import _observed
from .norms import plain

__all__ = ["embed", "token_losses"]

_MOST_TOKENS, _MOST_WORDS, _MOST_HIDDEN = 1 << 30, 1 << 30, 1 << 22   # adambridge_embed's
_MOST_ROWS, _MOST_CLASSES, _MOST_SIZE = 1 << 23, 1 << 22, 1 << 20       # adambridge_token_losses's
_LEAST_SIZE = {torch.bfloat16: 8, torch.float32: 4}


# ----------------------------------------------------------------------- embed

def _torch_embed(ids, weight, scale, padding_idx):
    """The definition in torch operations."""
    vocab, hidden = weight.shape
    flat = ids.reshape(-1).long()   # a vocabulary past 32 bits is compared as it is
    inside = (flat >= 0) & (flat < vocab)
    wide, at = torch.promote_types(weight.dtype, torch.float32), torch.where(inside, flat, 0)
    if _observed() or torch.is_grad_enabled() and weight.requires_grad:
        rows = weight.to(wide).index_select(0, at)   # widened before the rows are taken: their gradients are summed so
    else:
        rows = weight.index_select(0, at).to(wide)
    if padding_idx is not None:
        rows = torch.where((flat == padding_idx)[:, None], rows.detach(), rows)
    y = torch.where(inside[:, None], rows, torch.nan) * scale   # (in this order zeros go back to the rows of ids outside, whatever the scale)
    return y.to(weight.dtype).reshape(*ids.shape, hidden)


def _embed_backward(gout, ids, vocab, scale, padding_idx):
    """The embedding's gradient in torch operations, differentiable in turn."""
    flat = ids.reshape(-1).long()
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


# ---------------------------------------------------------------- token_losses

def _scored(hidden, targets, vocab, ignore_index):
    """The rows, zeros where they are not scored; which are; their targets, 0 for none."""
    rows, flat = hidden.reshape(-1, hidden.shape[-1]), targets.reshape(-1)
    scored = flat != ignore_index
    rows = torch.where(scored[:, None], rows.to(torch.promote_types(rows.dtype, torch.float32)), 0.0)
    inside = (flat >= 0) & (flat < vocab)
    return rows, scored, inside, torch.where(inside, flat, 0)


def _torch_token_losses(hidden, weight, targets, ignore_index):
    """The definition in torch operations, which hold all logits."""
    rows, scored, inside, at = _scored(hidden, targets, weight.shape[0], ignore_index)
    logits = torch.where(scored[:, None], rows @ weight.to(rows.dtype).t(), 0.0)   # (zeros times an infinite weight are NaN)
    loss = -torch.gather(logits.log_softmax(1), 1, at[:, None])[:, 0]   # NaN where a logit is inf, as the kernels'
    # a factor, so that a target outside the vocabulary makes its row's gradients NaN too
    loss = loss * torch.where(inside | ~scored, 1.0, torch.nan).to(loss.dtype)
    return torch.where(scored, loss, 0.0).reshape(targets.shape)


def _token_losses_backward(gout, hidden, weight, targets, ignore_index, want_hidden, want_weight):
    """Both gradients in torch operations, differentiable in turn."""
    with torch.autocast(gout.device.type, enabled=False):
        vocab = weight.shape[0]
        rows, scored, inside, at = _scored(hidden, targets, vocab, ignore_index)
        wide = weight.to(rows.dtype)
        seed = torch.where(scored, torch.where(inside, gout.reshape(-1), torch.nan), 0.0)[:, None]
        hot = torch.arange(vocab, device=at.device) == at[:, None]
        logits = torch.where(scored[:, None], rows @ wide.t(), 0.0)   # (zeros times an infinite weight are NaN)
        grad = (logits.softmax(1) - hot.to(rows.dtype)) * seed
        dhidden = dweight = None
        if want_hidden:
            dhidden = torch.where(scored[:, None], grad @ wide, 0.0).to(hidden.dtype).reshape(hidden.shape)
        if want_weight:
            dweight = (grad.t() @ rows).to(weight.dtype)
        return dhidden, dweight, None, None


def token_losses(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """Each row's cross-entropy of ``hidden @ weight.T`` against its target, without the logits: ``hidden`` ``[..., size]``,
    ``weight`` ``[vocab, size]`` (a Linear head's), ``targets`` (int64 or int32) ``[...]``; float32 ``[...]`` (float64 from float64).

    ``-token_losses(...)`` is the log-probability of each target.  Differentiable in ``hidden`` and ``weight``: the backward pass
    goes through the vocabulary in pieces and computes each piece's logits again, from ``weight`` as it is then: as any saved
    operand, it must not be written between the two passes.  Its scratch: a copy of ``hidden``, FP32 sums of ``hidden``'s size, a
    piece's gradient of at most 2^28 values (half a GiB in BF16), or 4096 words for every row.  The forward pass's: a copy of
    ``hidden`` and 8 bytes for each row and 256 words.

    Where a target is ``ignore_index`` the loss is 0 and its row reaches nothing, whatever it holds (and of more than 16 rows,
    it is left out of the products); a target outside the vocabulary gives a loss and gradients of NaN, as a logit of inf does.
    ``hidden`` and ``weight`` are of one type (under autocast, taken in its type, as a Linear's are).  Rows shorter than 16 bytes
    take torch operations."""
    if torch.compiler.is_compiling():
        return _uncompiled(token_losses, hidden, weight, targets, ignore_index)
    if weight.is_cuda:
        losses = _hip.ops().token_losses(hidden, weight, targets, ignore_index)
        if losses is not None:
            return losses
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or not weight.shape[0] or not weight.shape[1]:
        raise ValueError(f"token_losses takes hidden [..., size] and weight [vocab, size], not empty, got {tuple(hidden.shape)} and "
                         f"{tuple(weight.shape)}")
    if targets.dtype not in (torch.int64, torch.int32) or targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets must be int64 or int32 {tuple(hidden.shape[:-1])}, got {targets.dtype} {tuple(targets.shape)}")
    if hidden.device != weight.device or targets.device != weight.device:
        raise ValueError(f"hidden, weight and targets must be on one device, got {hidden.device}, {weight.device} and {targets.device}")
    if isinstance(ignore_index, bool) or not isinstance(ignore_index, int):
        raise ValueError(f"ignore_index must be an int, got {ignore_index!r}")
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"ignore_index must be an int of 64 bits, got {ignore_index}")
    targets = targets.long()   # an ignore_index past 32 bits is compared as it is
    if torch.is_autocast_enabled(hidden.device.type):
        cast = torch.get_autocast_dtype(hidden.device.type)
        hidden, weight = (t.to(cast) if t.is_floating_point() and t.dtype != torch.float64 else t for t in (hidden, weight))
    if hidden.dtype != weight.dtype or not hidden.is_floating_point():
        raise ValueError(f"hidden and weight must be of one floating-point type, got {hidden.dtype} and {weight.dtype}")
    with torch.autocast(hidden.device.type, enabled=False):
        if (plain(hidden, weight) and type(targets) is torch.Tensor and 0 < targets.numel() <= _MOST_ROWS and weight.shape[0] <= _MOST_CLASSES
                and _LEAST_SIZE[weight.dtype] <= weight.shape[1] <= _MOST_SIZE and not _observed()):
            losses = _hip.ops().token_losses(hidden.contiguous(), weight.contiguous(), targets.contiguous(), ignore_index)
            if losses is not None:
                return losses
        return _torch_token_losses(hidden, weight, targets, ignore_index)


# for the backward passes that the kernels do not take
BACKWARD = {"embed": _embed_backward, "token_losses": _token_losses_backward}
