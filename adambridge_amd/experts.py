"""Expert layers: the router's choice, the rows' way to the experts and back, and the experts' products.

An expert MLP of ``top_k`` experts a token is::

    r = route(x @ router.T, top_k)                  # which experts, with what weights, in what order
    rows = dispatch(x, r)                           # [tokens * top_k, hidden], sorted by expert
    rows = expert_mm(F.gelu(expert_mm(rows, up, r.ends)), down, r.ends)
    y = combine(rows, r)                            # each token's weighted sum

Nothing of it waits for the device: how many rows an expert has is read there (``r.ends``).  On plain GPU
tensors of float32 or bfloat16 the library's kernels compute it (csrc/abh_route.hip, csrc/abh_experts.hip, called by
csrc/abh_ops.cpp); elsewhere, and where an operation is traced, transformed or differentiated twice, torch operations do.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _hip
from .losses import _observed
from .norms import plain

__all__ = ["Routing", "route", "dispatch", "expert_mm", "combine"]

_MOST_EXPERTS, _MOST_CHOSEN, _MOST_ASSIGNED = 1024, 64, (1 << 31) - 1   # adambridge_route's
_MOST_ROWS, _MOST_SIZE, _MOST_MM_EXPERTS = 1 << 30, 1 << 22, 4096       # adambridge_expert_mm's


class Routing(NamedTuple):
    """Where tokens go.  The assignments ``(t, j)``, numbered ``t * top_k + j``, are sorted by expert, stably.

    ``weights``: ``[tokens, top_k]`` float32 (float64 from float64 logits), differentiable; ``experts``: ``[tokens, top_k]``, largest weight first;
    ``ends``: ``[experts]``, one past each expert's last row; ``order``: ``[tokens * top_k]``, the assignment
    that is each row; ``position``: ``[tokens, top_k]``, each assignment's row.  The last four are int32."""

    weights: torch.Tensor
    experts: torch.Tensor
    ends: torch.Tensor
    order: torch.Tensor
    position: torch.Tensor


@torch.compiler.disable
def _uncompiled(fn, *args):
    """``fn`` outside a compiled graph, which breaks there."""
    return fn(*args)


# ----------------------------------------------------------------------- route

def _torch_route(logits, top_k, normalize):
    """The definition in torch operations."""
    wide = logits.to(torch.promote_types(logits.dtype, torch.float32))
    tokens, experts = wide.shape
    chosen = torch.sort(wide.detach() + 0.0, dim=1, descending=True, stable=True).indices[:, :top_k]
    values = torch.gather(wide, 1, chosen)
    top = values[:, :1].detach()
    shift = torch.where(top == -torch.inf, 0.0, top)   # a row without any finite logit: weights 0
    e = torch.exp(values - shift)
    total = (e if normalize else torch.exp(wide - shift)).sum(1, keepdim=True)
    weights = e / torch.where(total == 0.0, 1.0, total)
    flat = chosen.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    at = torch.arange(tokens * top_k, device=logits.device)   # nothing in place below: ``logits`` may be a batch
    position = torch.zeros_like(order).scatter(0, order, at).view(tokens, top_k)
    ends = torch.zeros(experts, dtype=torch.int64, device=logits.device).scatter_add(0, flat, torch.ones_like(flat)).cumsum(0)
    return Routing(weights, chosen.int(), ends.int(), order.int(), position.int())


def _route_backward(gout, weights, chosen, logits, experts, normalize, dtype):
    """The logits' gradient in torch operations, differentiable in turn."""
    seed = weights * gout
    total = seed.sum(1, keepdim=True)
    spread = weights.new_zeros(weights.shape[0], experts)
    if normalize:
        return spread.scatter(1, chosen.long(), seed - weights * total).to(dtype), None, None
    wide = logits.float()
    top = wide.detach().amax(1, keepdim=True)
    e = torch.exp(wide - torch.where(top == -torch.inf, 0.0, top))
    norm = e.sum(1, keepdim=True)
    p = e / torch.where(norm == 0.0, 1.0, norm)
    return (spread.scatter(1, chosen.long(), seed) - p * total).to(dtype), None, None


def route(logits: torch.Tensor, top_k: int, normalize: bool = True) -> Routing:
    """The ``top_k`` largest of each token's ``logits`` (``[tokens, experts]``; the lower index of equal ones, a NaN
    counting as the largest), their softmax weights -- over the chosen if ``normalize``, else over all experts --
    and the order of the assignments by expert.

    An expert masked by ``-inf`` has weight 0 and is chosen only where nothing else is left; a token all of
    whose logits are ``-inf`` has weights 0 and no gradient."""
    if torch.compiler.is_compiling():
        return _uncompiled(route, logits, top_k, normalize)
    if logits.is_cuda:
        out = _hip.ops().route(logits, top_k, bool(normalize))
        if out is not None:
            return Routing(*out)
    if logits.dim() != 2 or not logits.is_floating_point() or logits.shape[1] < 1:
        raise ValueError(f"logits must be floating-point [tokens, experts], got {logits.dtype} {tuple(logits.shape)}")
    tokens, experts = logits.shape
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 1 <= top_k <= experts:
        raise ValueError(f"top_k must be an int from 1 to the number of experts, {experts}, got {top_k!r}")
    if tokens * top_k > _MOST_ASSIGNED:
        raise ValueError(f"tokens * top_k must be below 2^31, got {tokens * top_k}")
    if not plain(logits) or not tokens or experts > _MOST_EXPERTS or top_k > _MOST_CHOSEN or _observed():
        return _torch_route(logits, top_k, normalize)
    out = _hip.ops().route(logits.contiguous(), top_k, bool(normalize))
    return _torch_route(logits, top_k, normalize) if out is None else Routing(*out)


# -------------------------------------------------------- dispatch and combine

def _checked_position(name: str, routing: Routing, device: torch.device) -> tuple[int, int]:
    position = routing.position
    if position.dim() != 2 or position.dtype != torch.int32 or position.device != device:
        raise ValueError(f"the routing's position must be int32 [tokens, top_k] on {name}'s device, {device}, got "
                         f"{position.dtype} {tuple(position.shape)} on {position.device}")
    if not 1 <= position.shape[1]:
        raise ValueError("the routing assigns no rows")
    return position.shape


def _fits(tokens: int, top_k: int, cols: int) -> bool:
    return tokens > 0 and top_k <= _MOST_CHOSEN and 0 < cols <= _MOST_SIZE and tokens * top_k <= _MOST_ASSIGNED


def _assignments(position):
    """The assignment that each row is, 0 where no position names it.  (Positions outside the rows go to one row more.)"""
    flat, n = position.reshape(-1).long(), position.numel()
    flat = torch.where((flat >= 0) & (flat < n), flat, n)
    return flat.new_zeros(n + 1).scatter(0, flat, torch.arange(n, device=flat.device))[:n]


def _picked(rows, position, j):
    """Each token's row of its choice ``j``, zeros for a position outside the rows.  (No views: ``rows`` may be a batch.)"""
    at, n = position[:, j].long(), position.numel()
    inside = ((at >= 0) & (at < n))[:, None]
    return torch.where(inside, rows.index_select(0, at.clamp(0, max(n - 1, 0))), 0.0)


def _torch_dispatch(x, position):
    return x.index_select(0, _assignments(position) // position.shape[1])


def _torch_gather_sum(rows, weights, position):
    wide = torch.promote_types(rows.dtype, torch.float32)
    total = None
    for j in range(position.shape[1]):   # in order
        picked = _picked(rows, position, j).to(wide)
        if weights is not None:
            picked = picked * weights[:, j:j + 1]   # never narrower than FP32
        total = picked if total is None else total + picked
    return total.to(rows.dtype)


def _dispatch_backward(gout, position):
    return _torch_gather_sum(gout, None, position), None


def _combine_backward(gout, rows, weights, position, want_rows, want_weights):
    """Both gradients in torch operations, differentiable in turn."""
    g = gout.float()
    drows = dweights = None
    if want_rows:
        assignment = _assignments(position)
        w = weights.reshape(-1).index_select(0, assignment)[:, None]
        drows = (g.index_select(0, assignment // position.shape[1]) * w).to(gout.dtype)
    if want_weights:
        dweights = torch.stack([(_picked(rows, position, j).float() * g).sum(1) for j in range(position.shape[1])], 1)
    return drows, dweights, None


def dispatch(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Each token's row of ``x`` (``[tokens, hidden]``) at its ``top_k`` rows of the experts' order:
    ``[tokens * top_k, hidden]``."""
    if torch.compiler.is_compiling():
        return _uncompiled(dispatch, x, routing)
    if x.is_cuda:
        rows = _hip.ops().dispatch(x, routing.position)
        if rows is not None:
            return rows
    if x.dim() != 2 or not x.is_floating_point():
        raise ValueError(f"x must be floating-point [tokens, hidden], got {x.dtype} {tuple(x.shape)}")
    tokens, top_k = _checked_position("x", routing, x.device)
    if x.shape[0] != tokens:
        raise ValueError(f"x has {x.shape[0]} tokens, the routing {tokens}")
    if not plain(x) or not _fits(tokens, top_k, x.shape[1]) or _observed():
        return _torch_dispatch(x, routing.position)
    out = _hip.ops().dispatch(x.contiguous(), routing.position.contiguous())
    return _torch_dispatch(x, routing.position) if out is None else out


def combine(rows: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Each token's sum of its ``rows`` (``[tokens * top_k, hidden]``, in the experts' order), weighted by the routing's
    weights, summed in FP32 in the order of its choices and rounded once: ``[tokens, hidden]``.

    A position outside the rows, which :func:`route` never gives, counts as a row of zeros.  A row that no position names
    is unspecified in :func:`dispatch`'s result and in the gradient."""
    if torch.compiler.is_compiling():
        return _uncompiled(combine, rows, routing)
    if rows.is_cuda:
        out = _hip.ops().combine(rows, routing.weights, routing.position)
        if out is not None:
            return out
    if rows.dim() != 2 or not rows.is_floating_point():
        raise ValueError(f"rows must be floating-point [tokens * top_k, hidden], got {rows.dtype} {tuple(rows.shape)}")
    tokens, top_k = _checked_position("rows", routing, rows.device)
    if rows.shape[0] != tokens * top_k:
        raise ValueError(f"rows must be the routing's {tokens * top_k}, got {rows.shape[0]}")
    weights = routing.weights
    if (tuple(weights.shape) != (tokens, top_k) or weights.device != rows.device
            or weights.dtype not in (torch.float32, torch.promote_types(rows.dtype, torch.float32))):
        raise ValueError(f"the routing's weights must be float32 [{tokens}, {top_k}] on {rows.device}, got {weights.dtype} "
                         f"{tuple(weights.shape)} on {weights.device}")
    if not plain(rows, weights) or not _fits(tokens, top_k, rows.shape[1]) or _observed():
        return _torch_gather_sum(rows, weights, routing.position)
    out = _hip.ops().combine(rows.contiguous(), weights.contiguous(), routing.position.contiguous())
    return _torch_gather_sum(rows, weights, routing.position) if out is None else out


# ------------------------------------------------------------------- expert_mm

def _bounds(rows: int, ends: torch.Tensor) -> list[tuple[int, int]]:
    """Each expert's rows; an end out of range, or below one before it, is the nearest that is not, as the kernels take it."""
    out, lo = [], 0
    # under a function transform a copy to the host is a wrapped tensor, whose values come one by one
    for end in [e.item() for e in ends.cpu()] if torch._C._are_functorch_transforms_active() else ends.tolist():
        out.append((lo, min(max(end, lo), rows)))
        lo = out[-1][1]
    return out


def _torch_rows(x, weight, ends):
    """``x`` times each expert's ``weight[e]`` (rows x k by k x n); zeros for the rows that are no expert's."""
    parts = [x[lo:hi] @ weight[e] for e, (lo, hi) in enumerate(_bounds(x.shape[0], ends))]
    out = torch.cat(parts)
    return torch.cat((out, out.new_zeros(x.shape[0] - out.shape[0], out.shape[1]))) if out.shape[0] < x.shape[0] else out


def _torch_weights(gout, x, ends):
    return torch.stack([gout[lo:hi].t() @ x[lo:hi] for lo, hi in _bounds(x.shape[0], ends)])


def _expert_mm_backward(gout, x, weight, ends, want_x, want_w):
    """Both gradients in torch operations, differentiable in turn."""
    with torch.autocast(gout.device.type, enabled=False):
        return (_torch_rows(gout, weight, ends) if want_x else None,
                _torch_weights(gout, x, ends) if want_w else None, None)


# for the backward passes that the kernels do not take
BACKWARD = {"route": _route_backward, "dispatch": _dispatch_backward, "combine": _combine_backward,
            "expert_mm": _expert_mm_backward}


def expert_mm(x: torch.Tensor, weight: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """``x[r] @ weight[e].T`` for each row ``r`` of each expert ``e``: ``x`` ``[rows, in]`` sorted by expert, ``weight``
    ``[experts, out, in]`` (stacked Linear weights), expert ``e``'s rows ``ends[e - 1]`` to ``ends[e] - 1`` (``ends``: int32
    ``[experts]``, not decreasing, on the device; one that is below another before it counts as that, one beyond the rows as
    their number).  Rows from the last end on give zeros.

    Sums are FP32, rounded once.  Differentiable in ``x`` and ``weight``; an expert without rows has zero gradients.  (Under
    ``vmap`` the ends, which decide sizes, are one for all.)
    Under autocast both operands are taken in autocast's type, as a Linear's are (not float64)."""
    if torch.compiler.is_compiling():
        return _uncompiled(expert_mm, x, weight, ends)
    if x.is_cuda:
        out = _hip.ops().expert_mm(x, weight, ends)
        if out is not None:
            return out
    if x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[2]:
        raise ValueError(f"expert_mm takes x [rows, in] and weight [experts, out, in], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if ends.dim() != 1 or ends.shape[0] != weight.shape[0] or ends.dtype != torch.int32:
        raise ValueError(f"ends must be int32 [{weight.shape[0]}], got {ends.dtype} {tuple(ends.shape)}")
    if not weight.shape[0] or not weight.shape[1] or not weight.shape[2]:
        raise ValueError(f"weight must not be empty, got {tuple(weight.shape)}")
    if weight.device != x.device or ends.device != x.device:
        raise ValueError(f"x, weight and ends must be on one device, got {x.device}, {weight.device} and {ends.device}")
    if torch.is_autocast_enabled(x.device.type):
        cast = torch.get_autocast_dtype(x.device.type)
        x, weight = (t.to(cast) if t.is_floating_point() and t.dtype != torch.float64 else t for t in (x, weight))
    if x.dtype != weight.dtype or not x.is_floating_point():
        raise ValueError(f"x and weight must be of one floating-point type, got {x.dtype} and {weight.dtype}")
    experts, n, k = weight.shape
    if (not plain(x, weight) or x.shape[0] > _MOST_ROWS or experts > _MOST_MM_EXPERTS or n > _MOST_SIZE or k > _MOST_SIZE
            or _observed()):
        return _torch_rows(x, weight.transpose(1, 2), ends)
    with torch.autocast("cuda", enabled=False):
        out = _hip.ops().expert_mm(x.contiguous(), weight.contiguous(), ends.contiguous())
    return _torch_rows(x, weight.transpose(1, 2), ends) if out is None else out
