"""Tokens sorted by expert and back on one GPU, with gradients.

Where a GPU holds the experts that its tokens go to (training on one GPU, data-parallel experts, the
experts of an expert-parallel rank after its own exchange), the tokens need no all-to-all object:

    rows = sort_by_expert(indices, num_experts)          # where the rows of the experts are
    x_rows = permute_tokens(x, rows)                     # every token to the rows of its experts
    ...                                                  # the experts, on their rows
    out = unpermute_tokens(y_rows, rows, weights)        # the weighted sum of each token's rows

``permute_tokens`` and ``unpermute_tokens`` are differentiable in the tokens, the rows and the
weights, in reverse mode; tensors that carry a forward-mode tangent are refused here and by the
quantisation and the product of 8-bit integers.  ``permute_tokens_int8`` quantises on the way, for ``grouped_gemm_int8``.  The reference
library has no such operators: its tokens always pass through dispatch and combine.

Two layouts of the rows.  ``capacity=0``: one expert's rows after the other's, as many as there are
entries of the routing (``[tokens * topk, hidden]``, rows beyond ``offsets[-1]`` without a token).
``capacity=c``: ``[num_experts, c, hidden]``, the layout that ``grouped_gemm`` and
``grouped_gemm_fp8`` take together with ``counts``; what an expert gets beyond ``c`` is dropped.

Nothing here synchronises with the host: all of it can be captured in a CUDA graph.
"""

from __future__ import annotations

import torch

from . import _ops


class ExpertRows:
    """Where the rows of the experts are.

    ``counts`` [num_experts] and ``offsets`` [num_experts + 1], int32: the number of rows of every
    expert and its first row.  ``row_of`` [tokens, topk], int32: the row of every entry of the
    routing, -1 for an entry without one.  ``bound_m``: the device-side number of valid tokens that
    the routing was sorted with, if any.
    """

    __slots__ = ("counts", "offsets", "row_of", "capacity", "bound_m")

    def __init__(self, counts: torch.Tensor, offsets: torch.Tensor, row_of: torch.Tensor,
                 capacity: int = 0, bound_m: torch.Tensor | None = None) -> None:
        self.counts, self.offsets, self.row_of = counts, offsets, row_of
        self.capacity, self.bound_m = capacity, bound_m

    def shape(self) -> tuple[int, ...]:
        """The dimensions of a tensor of rows in front of its last."""
        if self.capacity:
            return self.counts.size(0), self.capacity
        return (self.row_of.numel(),)


def sort_by_expert(indices: torch.Tensor, num_experts: int, capacity: int = 0,
                   bound_m: torch.Tensor | None = None) -> ExpertRows:
    """Sorts the routing by expert.  The entries of one expert keep the order of (token, k).

    ``indices`` [tokens, topk] (uint32, int32 or int64) names the experts of each token, up to 1024
    of them; a number outside ``[0, num_experts)`` is an entry without a row (an expert of another
    GPU).  A token may name an expert twice: it then has two of its rows.  ``bound_m`` (32-bit, on
    the device): tokens at or beyond it get no rows.
    """
    counts, offsets, row_of = _ops.sort_by_expert(indices, num_experts, capacity, bound_m)
    return ExpertRows(counts, offsets, row_of, capacity, bound_m)


def permute_tokens(x: torch.Tensor, rows: ExpertRows, zero_rest: bool | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Copies every token of ``x`` [tokens, hidden] to its rows: ``out[rows.row_of[t, k]] = x[t]``.

    ``x`` may have any type of 1, 2, 4 or 8 bytes.  Rows without a token are left as they are, or
    set to zero with ``zero_rest``; where a gradient is recorded (``x`` requires one) they are zero,
    and the gradient of ``x[t]`` is the sum of its rows' (in fp32, rounded once; bf16, fp16 and fp32).
    """
    if x.requires_grad and torch.is_grad_enabled():
        if zero_rest is False:
            raise ValueError("permute_tokens: rows without a token are zero where a gradient is recorded")
        if out is not None:
            raise _no_gradient("permute_tokens")
    if out is None:
        return _ops.permute_tokens(x, rows.counts, rows.offsets, rows.row_of, rows.capacity,
                                   bool(zero_rest))
    _ops.permute_tokens_out(x, rows.counts, rows.offsets, rows.row_of, rows.capacity, out,
                            bool(zero_rest))
    return out


def permute_tokens_backward(grad: torch.Tensor, rows: ExpertRows) -> torch.Tensor:
    """The gradient of ``permute_tokens`` with respect to the tokens, for that of its result."""
    return _ops.unpermute_tokens(grad, rows.counts, rows.offsets, rows.row_of, rows.capacity, None)


def permute_tokens_int8(x: torch.Tensor, rows: ExpertRows, zero_rest: bool = False,
                        out: torch.Tensor | None = None, out_scale: torch.Tensor | None = None,
                        ) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantises every token of ``x`` (bf16, fp16 or fp32) as ``quantize_rows_int8`` does and copies
    it to its rows.  Returns the rows and their fp32 scales.  Not differentiable."""
    if x.requires_grad and torch.is_grad_enabled():
        raise _no_gradient("permute_tokens_int8")
    if out is None and out_scale is None:
        return _ops.permute_tokens_int8(x, rows.counts, rows.offsets, rows.row_of, rows.capacity,
                                        zero_rest)
    if out is None:
        out = torch.empty(*rows.shape(), x.size(1), dtype=torch.int8, device=x.device)
    if out_scale is None:
        out_scale = torch.empty(rows.shape(), dtype=torch.float32, device=x.device)
    _ops.permute_tokens_int8_out(x, rows.counts, rows.offsets, rows.row_of, rows.capacity, out,
                                 out_scale, zero_rest)
    return out, out_scale


def unpermute_tokens(y: torch.Tensor, rows: ExpertRows, weights: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Sums each token's rows: ``out[t] = sum over k of weights[t, k] * y[rows.row_of[t, k]]``.

    ``y``: rows in bf16, fp16 or fp32; ``weights`` [tokens, topk] fp32, None for ones.  The sum is
    taken in fp32, in the order of k, and rounded once.  Entries without a row add nothing; a token
    without rows is zero.  Where the routing was sorted with ``bound_m``, an ``out`` that is given
    keeps its rows at or beyond it; they are zero in one that is allocated here.

    Differentiable, once, in ``y`` and ``weights``; the gradient of rows without a token is zero.
    """
    if out is None:
        return _ops.unpermute_tokens(y, rows.counts, rows.offsets, rows.row_of, rows.capacity, weights)
    if (y.requires_grad or (weights is not None and weights.requires_grad)) and torch.is_grad_enabled():
        raise _no_gradient("unpermute_tokens")
    _ops.unpermute_tokens_out(y, rows.counts, rows.offsets, rows.row_of, rows.capacity, weights, out,
                              rows.bound_m)
    return out


def unpermute_tokens_backward(
        grad: torch.Tensor, y: torch.Tensor, rows: ExpertRows, weights: torch.Tensor,
        need_y: bool = True, need_weights: bool = True,
        ) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """The gradients of ``unpermute_tokens`` with respect to the rows and the weights, for that of
    its result.  Rows without a token get zero, and so do the weights of entries without a row."""
    grad_y = torch.empty_like(y) if need_y else None
    grad_weights = torch.empty_like(weights) if need_weights else None
    _ops.unpermute_tokens_backward(grad, y, rows.counts, rows.offsets, rows.row_of, rows.capacity,
                                   weights, grad_y, grad_weights)
    return grad_y, grad_weights


def _no_gradient(name: str) -> ValueError:
    """The refusal of a call whose result could not carry the gradient that was asked for."""
    return ValueError(f"{name}: no gradient is recorded here; use torch.no_grad() or detach()")


def sort_by_expert_reference(indices: torch.Tensor, num_experts: int, capacity: int = 0,
                             bound_m: int | None = None) -> ExpertRows:
    """Plain statement of ``sort_by_expert``, entry by entry on the host."""
    m, topk = indices.shape
    taken: list[list[int]] = [[] for _ in range(num_experts)]
    for i, e in enumerate(indices.to(torch.int64).flatten().tolist()):
        if 0 <= e < num_experts and (bound_m is None or i < bound_m * topk) \
                and (not capacity or len(taken[e]) < capacity):
            taken[e].append(i)
    offsets = [0]
    row_of = torch.full((m * topk,), -1, dtype=torch.int32)
    for e, entries in enumerate(taken):
        row_of[entries] = torch.arange(offsets[e], offsets[e] + len(entries), dtype=torch.int32)
        offsets.append(offsets[e] + (capacity or len(entries)))
    counts = torch.tensor([len(entries) for entries in taken], dtype=torch.int32)
    return ExpertRows(counts, torch.tensor(offsets, dtype=torch.int32), row_of.view(m, topk), capacity)
