"""What autograd meets in the operators of the experts of one GPU, on Meta tensors."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from pplx_kernels_b200.ops.expert_rows import (
    permute_tokens,
    permute_tokens_backward,
    permute_tokens_int8,
    sort_by_expert,
    unpermute_tokens,
    unpermute_tokens_backward,
)
from pplx_kernels_b200.ops.grouped_gemm import grouped_gemm_int8
from pplx_kernels_b200.ops.quant import quantize_rows_int8

M, K, E, H = 6, 3, 5, 64


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def rows():
    return sort_by_expert(meta(M, K, dtype=torch.int32), E)


def product(x_scale, w_scale, **kwargs):
    return grouped_gemm_int8(meta(E, 4, H, dtype=torch.int8), x_scale, meta(E, 16, H, dtype=torch.int8),
                             w_scale, **kwargs)


# A call in one floating tensor, and its shape.
FLOATING = {
    "copy": (lambda t: permute_tokens(t, rows()), (M, H)),
    "copy, out": (lambda t: permute_tokens(t, rows(), out=meta(M * K, H)), (M, H)),
    "copy, into": (lambda t: permute_tokens(meta(M, H), rows(), out=t), (M * K, H)),
    "copy, gradient": (lambda t: permute_tokens_backward(t, rows()), (M * K, H)),
    "quantising copy": (lambda t: permute_tokens_int8(t, rows()), (M, H)),
    "quantising copy, out": (lambda t: permute_tokens_int8(t, rows(), out=meta(M * K, H, dtype=torch.int8)),
                             (M, H)),
    "quantising copy, scale": (lambda t: permute_tokens_int8(meta(M, H), rows(), out_scale=t), (M * K,)),
    "sum": (lambda t: unpermute_tokens(t, rows()), (M * K, H)),
    "sum, weighted": (lambda t: unpermute_tokens(t, rows(), meta(M, K)), (M * K, H)),
    "sum, weights": (lambda t: unpermute_tokens(meta(M * K, H), rows(), t), (M, K)),
    "sum, out": (lambda t: unpermute_tokens(t, rows(), out=meta(M, H)), (M * K, H)),
    "sum, weights, out": (lambda t: unpermute_tokens(meta(M * K, H), rows(), t, out=meta(M, H)), (M, K)),
    "sum, gradient": (lambda t: unpermute_tokens_backward(t, meta(M * K, H), rows(), meta(M, K)), (M, H)),
    "sum, gradient, rows": (lambda t: unpermute_tokens_backward(meta(M, H), t, rows(), meta(M, K)),
                            (M * K, H)),
    "quantisation": (lambda t: quantize_rows_int8(t), (M, H)),
    "quantisation, out": (lambda t: quantize_rows_int8(t, out=meta(M, H, dtype=torch.int8)), (M, H)),
    "product, scales": (lambda t: product(t, meta(E, 16)), (E, 4)),
    "product, weights' scales": (lambda t: product(meta(E, 4), t), (E, 16)),
}


@pytest.mark.parametrize("name", FLOATING)
@pytest.mark.parametrize("recorded", [False, True])
def test_tangents_are_refused(name, recorded):
    call, shape = FLOATING[name]
    t = meta(*shape)
    call(t)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t.requires_grad_(recorded), meta(*shape))
        with pytest.raises((RuntimeError, ValueError), match="tangent|gradient"):
            call(dual)
    if not recorded:
        with pytest.raises(RuntimeError, match="tangent"):
            torch.func.jvp(call, (t,), (meta(*shape),))


def test_tangents_through_a_gradient_are_refused():
    """Forward over reverse: the gradient's own tangent."""
    y, w, g = meta(M * K, H).requires_grad_(), meta(M, K).requires_grad_(), meta(M, H)
    out = unpermute_tokens(y, rows(), w)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            torch.autograd.grad(out, (y, w), forward_ad.make_dual(g, meta(M, H)))


# Calls that write tensors: what they write.
WRITING = {
    "copy": lambda o: permute_tokens(meta(M, H), rows(), out=o[0]),
    "quantising copy": lambda o: permute_tokens_int8(meta(M, H), rows(), out=o[1], out_scale=o[2]),
    "sum": lambda o: unpermute_tokens(meta(M * K, H), rows(), out=o[0][:M]),
    "quantisation": lambda o: quantize_rows_int8(meta(M * K, H), out=o[1], out_scale=o[2]),
    "product": lambda o: product(meta(E, 4), meta(E, 16), out=o[3], status=o[4]),
}


def buffers():
    return [meta(M * K, H), meta(M * K, H, dtype=torch.int8), meta(M * K),
            meta(E, 4, 16, dtype=torch.bfloat16), meta(1, dtype=torch.int32)]


@pytest.mark.parametrize("name", WRITING)
def test_written_tensors_count_as_changed(name):
    written = {"copy": [0], "sum": [0], "product": [3, 4]}.get(name, [1, 2])
    o = buffers()
    WRITING[name](o)
    assert [t._version for t in o] == [int(i in written) for i in range(5)]
    with torch.no_grad():
        WRITING[name](o)
    assert [t._version for t in o] == [2 * int(i in written) for i in range(5)]
    with torch.inference_mode():
        WRITING[name](buffers())  # (tensors without a version)
    inference = buffers()
    with torch.inference_mode():
        inference = buffers()
    WRITING[name](inference)


def test_a_saved_tensor_that_is_overwritten_is_noticed():
    x, out = meta(M * K, H).requires_grad_(), meta(M * K, H)
    y = (x * out).sum()
    permute_tokens(meta(M, H), rows(), out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("name", WRITING)
def test_written_tensors_that_require_a_gradient_are_refused(name):
    o = buffers()
    for t in o:
        if t.is_floating_point():
            t.requires_grad_()
    with torch.no_grad():
        WRITING[name](o)
    with pytest.raises((RuntimeError, ValueError), match="gradient"):
        WRITING[name](o)


def test_gradients_leave_the_saved_tensors_alone():
    """The backward pass writes its results only."""
    y, w = meta(M * K, H).requires_grad_(), meta(M, K).requires_grad_()
    where = rows()
    unpermute_tokens(y, where, w).sum().backward()
    unpermute_tokens_backward(meta(M, H), y.detach(), where, w.detach())
    assert y._version == w._version == where.row_of._version == 0


@pytest.mark.parametrize("capacity", [0, 4])
@pytest.mark.parametrize("of_rows,of_weights", [(True, True), (True, False), (False, True)])
def test_rows_are_kept_for_the_gradient_of_the_weights_only(capacity, of_rows, of_weights):
    """A frozen router: the gradient of the rows needs the weights and the grad, not the rows."""
    where = sort_by_expert(meta(M, K, dtype=torch.int32), E, capacity)
    y, w = meta(*where.shape(), H).requires_grad_(of_rows), meta(M, K).requires_grad_(of_weights)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.shape) or t, lambda t: t):
        out = unpermute_tokens(y, where, w)
    assert (y.shape in kept) == of_weights
    out.sum().backward()
    assert (y.grad is not None) == of_rows and (w.grad is not None) == of_weights
    assert not of_rows or y.grad.shape == y.shape
    assert not of_weights or w.grad.shape == w.shape


def test_gradient_of_the_weights_without_rows_is_refused():
    where = rows()
    with pytest.raises(RuntimeError, match="needs y"):
        torch.ops.pplx_kernels_b200.unpermute_tokens_backward(
            meta(M, H), None, where.counts, where.offsets, where.row_of, 0, meta(M, K), None, meta(M, K))


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex64, torch.float8_e4m3fn])
def test_types_without_a_gradient_are_refused_at_once(dtype):
    x = meta(M, H, dtype=dtype)
    assert permute_tokens(x, rows()).dtype == dtype
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="bfloat16, float16 or float32"):
        permute_tokens(x, rows())
    with torch.no_grad():
        assert permute_tokens(x, rows()).dtype == dtype


def test_scales_of_a_product_that_require_a_gradient_are_refused():
    for of_rows in (True, False):
        scales = meta(E, 4).requires_grad_(of_rows), meta(E, 16).requires_grad_(not of_rows)
        with pytest.raises(ValueError, match="gradient"):
            product(*scales)
        with torch.no_grad():
            assert product(*scales).shape == (E, 4, 16)


@pytest.mark.parametrize("name", WRITING)
def test_written_tensors_count_as_changed_in_inference_mode(name):
    written = {"copy": [0], "sum": [0], "product": [3, 4]}.get(name, [1, 2])
    o = buffers()
    with torch.inference_mode():
        WRITING[name](o)
    assert [t._version for t in o] == [int(i in written) for i in range(5)]
