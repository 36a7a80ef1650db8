"""Tables of rows that do not fit the tensors: entries out of range are left out, and all others are
written, by every operator that follows the table."""

import pytest
import torch

from pplx_kernels_b200.ops.expert_rows import (
    permute_tokens,
    permute_tokens_int8,
    sort_by_expert,
    unpermute_tokens,
    unpermute_tokens_backward,
)
from pplx_kernels_b200.ops.quant import quantize_rows_int8_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
FILL = 9


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hidden", [32, 129, 1001, 2048])
@pytest.mark.parametrize("capacity", [0, 7])
def test_entries_out_of_range(dtype, hidden, capacity):
    m, topk, experts = 20, 3, 5
    gen = torch.Generator(device=DEV).manual_seed(hidden)
    rows = sort_by_expert(torch.randint(0, experts, (m, topk), generator=gen, device=DEV), experts, capacity)
    total = experts * capacity if capacity else m * topk
    for at, value in ((0, total), (4, 2 ** 31 - 1), (8, -(2 ** 31)), (17, -2), (18, total + 1), (19, total)):
        rows.row_of[at, at % topk] = value
    rows.row_of[11] = total + 5  # a token without any
    row = rows.row_of.long()
    there = (row >= 0) & (row < total)
    at = row[there]
    token = torch.arange(m, device=DEV)[:, None].expand(m, topk)[there]
    written = torch.zeros(total, dtype=torch.bool, device=DEV)
    written[at] = True

    def filled(*tail, dtype=dtype):
        return torch.full((*rows.shape(), *tail), FILL, dtype=dtype, device=DEV)

    def check(got, want):
        got = got.view(total, -1)
        assert torch.equal(got[at], want[token].view(at.numel(), -1))
        assert (got[~written] == FILL).all()

    x = torch.randn(m, hidden, generator=gen, device=DEV).to(dtype)
    y = permute_tokens(x, rows, out=filled(hidden))
    check(y, x)
    want_q, want_s = quantize_rows_int8_reference(x)
    q, s = permute_tokens_int8(x, rows, out=filled(hidden, dtype=torch.int8),
                               out_scale=filled(dtype=torch.float32))
    check(q, want_q)
    check(s, want_s)
    # Sums: whole numbers, so that they are exact.
    whole = torch.randint(-8, 9, (m, hidden), generator=gen, device=DEV).to(dtype)
    rows_of_whole = permute_tokens(whole, rows, out=filled(hidden))
    assert torch.equal(unpermute_tokens(rows_of_whole, rows), there.sum(1, keepdim=True).to(dtype) * whole)
    # Gradients: of the rows w[t, k] g[t], one rounding; of the weights the products of whole numbers.
    w = torch.rand(m, topk, generator=gen, device=DEV)
    grad_y, grad_w = filled(hidden), torch.full((m, topk), float(FILL), device=DEV)
    torch.ops.pplx_kernels_b200.unpermute_tokens_backward(
        whole, rows_of_whole, rows.counts, rows.offsets, rows.row_of, capacity, w, grad_y, grad_w)
    flat = grad_y.view(total, hidden)
    assert torch.equal(flat[at], (w[there][:, None] * whole[token].float()).to(dtype))
    rest = ~written
    live = torch.arange(total, device=DEV) < (total if capacity else int(rows.offsets[-1]))
    if capacity:
        place = torch.arange(total, device=DEV)
        live = place % capacity < rows.counts[place // capacity]
    assert (flat[rest & live] == FILL).all() and (flat[rest & ~live] == 0).all()
    assert torch.equal(grad_w, torch.where(there, (whole.float() ** 2).sum(1, keepdim=True), 0.0))
    again, none = unpermute_tokens_backward(whole, rows_of_whole, rows, w, need_weights=False)
    assert none is None and torch.equal(again.view(total, hidden)[at], flat[at])
