"""Results that overlap themselves or an input are refused by the operators of the experts of one GPU."""

import pytest
import torch

from pplx_kernels_b200.ops.expert_rows import (
    permute_tokens,
    permute_tokens_int8,
    sort_by_expert,
    unpermute_tokens,
)
from pplx_kernels_b200.ops.grouped_gemm import grouped_gemm_int8
from pplx_kernels_b200.ops.quant import quantize_rows_int8

E, ROWS, N, K = 5, 4, 16, 64


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def product(out, experts=E, rows=ROWS, xq=None):
    xq = meta(experts, rows, K, dtype=torch.int8) if xq is None else xq
    return grouped_gemm_int8(xq, meta(experts, rows, dtype=torch.float32), meta(experts, N, K, dtype=torch.int8),
                             meta(experts, N, dtype=torch.float32), out=out)


@pytest.mark.parametrize("out", [
    meta(1, ROWS, N).expand(E, ROWS, N),
    meta(E * N * ROWS).as_strided((E, ROWS, N), (N, N, 1)),
    meta(E * 2 * N * ROWS).as_strided((E, ROWS, N), (N * ROWS - 8, N, 1)),
    meta(E * 2 * N * ROWS).as_strided((E, ROWS, N), (8, E * N, 1)),
], ids=["one plane for all", "plane per row", "planes that overlap", "columns that overlap"])
def test_results_of_experts_that_overlap(out):
    with pytest.raises(RuntimeError, match="must not overlap"):
        product(out)


@pytest.mark.parametrize("out", [
    meta(E, ROWS, N),
    meta(ROWS, E, N).transpose(0, 1),  # the experts' columns side by side
    meta(E, ROWS + 3, N + 8)[:, :ROWS, :N],
    meta(ROWS, E, N + 8).transpose(0, 1)[:, :, :N],
    meta(E * ROWS * N).as_strided((E, ROWS, N), (ROWS * N, N, 1)),
])
def test_results_of_experts_that_do_not(out):
    assert product(out) is out


def test_results_of_one_row_or_expert():
    product(meta(1, ROWS, N).as_strided((1, ROWS, N), (0, N, 1)), experts=1)
    product(meta(E, 1, N).as_strided((E, 1, N), (N, 0, 1)), rows=1)
    product(meta(E, 0, N), rows=0)
    with pytest.raises(RuntimeError, match="must not overlap"):
        product(meta(1, 1, N).expand(E, 1, N), rows=1)


M, TOPK, H = 6, 2, 64


def table(m=M, topk=TOPK):
    return sort_by_expert(meta(m, topk, dtype=torch.int32), E)


def bytes_of(t):
    return t.view(torch.int8)


@pytest.mark.parametrize("call", [
    lambda b: permute_tokens(b[:M], table(), out=b[: M * TOPK]),
    lambda b: permute_tokens(b[:M], table(M, 1), out=b[:M]),
    lambda b: unpermute_tokens(b[: M * TOPK], table(), out=b[M : 2 * M]),
    lambda b: unpermute_tokens(b[:M], table(M, 1), meta(M, 1, dtype=torch.float32), out=b[:M]),
    lambda b: quantize_rows_int8(b[:M], out=bytes_of(b[:M]).view(2 * M, H)[:M]),
    lambda b: permute_tokens_int8(b[:M], table(), out=bytes_of(b[:M]).view(2 * M, H)),
    lambda b: product(b.flatten()[: E * ROWS * N].view(E, ROWS, N), xq=b.flatten().view(torch.int8)[
        : E * ROWS * K].view(E, ROWS, K)),
])
def test_results_in_the_memory_of_the_input(call):
    with pytest.raises(RuntimeError, match="must not share memory"):
        call(meta(40, H))


def test_results_beside_the_input():
    """Other rows of one tensor, or other columns."""
    b = meta(40, H)
    permute_tokens(b[:M], table(), out=b[M : M + M * TOPK])
    unpermute_tokens(b[: M * TOPK], table(), out=b[20 : 20 + M])
    wide = meta(M, 2 * H)
    unpermute_tokens(permute_tokens(wide[:, :H], table()), table(), out=wide[:, H:])
