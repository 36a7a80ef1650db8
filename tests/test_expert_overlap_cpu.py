"""Results that overlap themselves or an input are refused by the operators of the experts of one GPU."""

import pytest
import torch

from pplx_kernels_b200.ops.grouped_gemm import grouped_gemm_int8

E, ROWS, N, K = 5, 4, 16, 64


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def product(out, experts=E, rows=ROWS):
    return grouped_gemm_int8(meta(experts, rows, K, dtype=torch.int8), meta(experts, rows, dtype=torch.float32),
                             meta(experts, N, K, dtype=torch.int8), meta(experts, N, dtype=torch.float32), out=out)


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
