"""Gradients of the sum of rows where not all of its inputs need one."""

import pytest
import torch

from pplx_kernels_b200.ops.expert_rows import (
    sort_by_expert,
    unpermute_tokens,
    unpermute_tokens_backward,
)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hidden,capacity", [(129, 0), (1000, 9), (2048, 0)])
def test_frozen_weights_and_frozen_rows(dtype, hidden, capacity):
    m, topk, experts = 40, 3, 8
    gen = torch.Generator(device=DEV).manual_seed(hidden)
    rows = sort_by_expert(torch.randint(-1, experts, (m, topk), generator=gen, device=DEV), experts, capacity)
    y = torch.randn(*rows.shape(), hidden, generator=gen, device=DEV).to(dtype)
    w = torch.rand(m, topk, generator=gen, device=DEV)
    g = torch.randn(m, hidden, generator=gen, device=DEV).to(dtype)
    want_y, want_w = unpermute_tokens_backward(g, y, rows, w)
    for of_rows, of_weights in ((True, False), (False, True), (True, True)):
        yl, wl = y.clone().requires_grad_(of_rows), w.clone().requires_grad_(of_weights)
        unpermute_tokens(yl, rows, wl).backward(g)
        assert torch.equal(yl.grad, want_y) if of_rows else yl.grad is None
        assert torch.equal(wl.grad, want_w) if of_weights else wl.grad is None


def test_rows_are_freed_where_the_weights_are_frozen():
    """What is on the device after the forward pass: the result, and no rows that only it has read."""
    m, topk, hidden = 2048, 8, 1024
    rows = sort_by_expert(torch.arange(m * topk, device=DEV).view(m, topk) % 16, 16)
    y = torch.ones(m * topk, hidden, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w = torch.rand(m, topk, device=DEV)
    before = torch.cuda.memory_allocated()
    out = unpermute_tokens(y * 2, rows, w)
    assert torch.cuda.memory_allocated() - before < 1.5 * out.numel() * 2
    out.sum().backward()
    assert torch.equal(y.grad[rows.row_of.flatten().long(), 0],
                       (2 * w.flatten().bfloat16().float()).bfloat16())
