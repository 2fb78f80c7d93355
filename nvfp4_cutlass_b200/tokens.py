"""Routing, token rows sorted by expert, and back: what stands before and behind the grouped GEMM of a mixture-of-experts layer, with
gradients.

    ids, weights = route_tokens(logits, k)
    rows, order = sort_tokens(x, ids, num_experts)                 # the GEMM's contiguous layout, m_indices included
    m_grouped_bf16_dual_nvfp4_gemm_contiguous(rows, *w, d, order.m_indices)
    y = unsort_tokens(d, order, weights)

Nothing comes back to the host: the sorted buffer has as many rows as any routing of so many pairs can need, so the calls can be
captured in a CUDA graph whose replays see other routings.  All of it is CUDA kernels of the library; CPU tensors are refused.  Gradients are
computed once (no second derivatives) and backwards: tensors with tangents of forward mode are refused.  The reference project begins
at rows that are grouped already.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _C


def _differentiable(*tensors) -> bool:
    """Whether a call has to be recorded: outside of training the autograd layer costs a launch-bound call as much as its kernel."""
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors)


def _refuse_tangents(*tensors) -> None:
    """The operators have no forward-mode derivatives: an output without a tangent would pass for a constant."""
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("this operator has no derivative in forward mode: its inputs must not carry tangents")


def _own_signs(t):
    """A tensor whose memory holds its values: torch may keep a negated view as the memory of what it negates."""
    return t.resolve_neg() if isinstance(t, torch.Tensor) else t


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, scores, renormalize):
        ids, weights = _C.route_tokens(logits, k, scores, renormalize)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, ids)
        ctx.form = (scores, renormalize)
        ctx.mark_non_differentiable(ids)
        return ids, weights

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, dweights):
        if dweights is None:
            return None, None, None, None
        logits, ids = ctx.saved_tensors
        return _C.route_tokens_backward(logits, ids, _own_signs(dweights), *ctx.form), None, None, None


def route_tokens(logits: torch.Tensor, k: int, *, scores: str = "softmax", renormalize: bool = True):
    """The k experts of every token: (ids int64 (tokens, k), weights float32 (tokens, k)).

    ``logits`` (tokens, experts) BF16, FP16 or FP32.  Experts come in the order of their logits, equal ones by their index.  Weights are the
    softmax (over all experts) or sigmoid scores, with ``renormalize`` divided by the sum of the chosen ones.  A logit of -inf is an
    expert that is not to be had: it is never chosen, and where fewer than k others are left the remaining ids are -1 and their weights 0
    (``sort_tokens`` gives such a pair no row).  experts <= 1024, k <= 32.  Differentiable in ``logits``."""
    if _C._binding is not None and scores in _C.SCORE_CODES:
        result = _C._binding.route(logits, k, _C.SCORE_CODES[scores], 1 if renormalize else 0)
        if result is not None:
            return result
    _refuse_tangents(logits)
    logits = _own_signs(logits)
    if not _differentiable(logits):
        return _C.route_tokens(logits, int(k), scores, bool(renormalize))
    return _Route.apply(logits, int(k), scores, bool(renormalize))


class TokenOrder(NamedTuple):
    """Where sort_tokens put what."""
    place: torch.Tensor          # int64 (tokens, k): row of every (token, choice) pair, -1 = none
    source: torch.Tensor         # int32 (M,): pair token * k + choice of every row, -1 = padding
    m_indices: torch.Tensor      # int32 (M,): expert whose group holds the row, -1 behind the last group


class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, num_experts, alignment):
        rows, place, source, m_indices = _C.sort_tokens(x, ids, num_experts, alignment)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(place)
        ctx.mark_non_differentiable(place, source, m_indices)
        return rows, place, source, m_indices

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, drows, *_):
        if drows is None:
            return None, None, None, None
        return _C.unsort_tokens(_own_signs(drows).contiguous(), ctx.saved_tensors[0], None), None, None, None


def sort_tokens(x: torch.Tensor, ids: torch.Tensor, num_experts: int, *, alignment: int = 128):
    """Token rows ``x`` (tokens, hidden) in the order of their experts: (rows (M, hidden), TokenOrder).

    ``ids`` int64 (tokens, k), as route_tokens gives them; an id outside [0, num_experts) gives its pair no row.  Every expert's rows
    start on a multiple of ``alignment`` (the GEMM's m_alignment: 128, or 16 / 32 / 64 for its decode orientation) and keep the order of
    their pairs; rows without a pair are zero.  M depends on the sizes alone:
    (pairs + min(num_experts, pairs) * (alignment - 1)) rounded down to a multiple of alignment.  BF16 rows go into the GEMM as they
    are; FP16 and FP32 rows are moved too.  num_experts <= 1024.  Differentiable in ``x``."""
    if _C._binding is not None:
        result = _C._binding.sort(x, ids, num_experts, alignment)
        if result is not None:
            return result[0], TokenOrder(*result[1:])
    _refuse_tangents(x)
    x = _own_signs(x)
    call = _Sort.apply if _differentiable(x) else _C.sort_tokens
    rows, place, source, m_indices = call(x, ids, int(num_experts), int(alignment))
    return rows, TokenOrder(place, source, m_indices)


class _Unsort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, place, source):
        want_weights = weights is not None and ctx.needs_input_grad[1]
        ctx.save_for_backward(rows if want_weights else None, weights, place, source)
        return _C.unsort_tokens(rows, place, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        rows, weights, place, source = ctx.saved_tensors
        want_rows, want_weights = ctx.needs_input_grad[:2]
        drows, dweights = _C.unsort_tokens_backward(_own_signs(dy).contiguous(), rows, place, source, weights, want_rows, want_weights)
        return drows, dweights, None, None


def unsort_tokens(rows: torch.Tensor, order: TokenOrder, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = sum over the choices j of weights[t, j] * rows[order.place[t, j]], (tokens, hidden) of the rows' type.

    ``rows`` (M, hidden) in the order that sort_tokens gave, ``weights`` float32 (tokens, k), or None for a plain sum.  Sums are FP32 in
    ascending j, rounded once.  A pair without a row (a place outside [0, M)) contributes nothing, and its weight's gradient is 0.
    Differentiable in ``rows`` and ``weights``; the gradient of rows that no pair names is zero.  ``order.place`` may also be a part of the
    sort's, have pairs masked out, or name a row more than once (whose gradient is then the sum over its pairs): forward and backward follow
    it alone."""
    place, source = order.place, order.source
    if _C._binding is not None:
        result = _C._binding.unsort(rows, place, source, weights)
        if result is not None:
            return result
    _refuse_tangents(rows, weights)
    rows, weights = _own_signs(rows), _own_signs(weights)
    _C._require(isinstance(rows, torch.Tensor) and source.dtype == torch.int32 and source.dim() == 1 and source.is_contiguous() and
                rows.dim() == 2 and rows.shape[0] == source.shape[0], "rows has the rows of the order")
    _C._one_device(rows, weights, place, source)
    if weights is not None:
        _C._require(isinstance(weights, torch.Tensor) and weights.dtype == torch.float32 and weights.shape == place.shape,
                    "weights are float32, one for every place of the order")
        weights = weights.contiguous()
    if not _differentiable(rows, weights):
        return _C.unsort_tokens(rows, place, weights)
    return _Unsort.apply(rows, weights, place, source)
