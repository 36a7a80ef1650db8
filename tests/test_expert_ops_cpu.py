"""Operators of the experts of one GPU, as far as no GPU is needed: the oracle of the sort against its
definition, and what the operators refuse (Meta tensors pass the checks of the CUDA ones)."""

import pytest
import torch

from pplx_kernels_b200.ops.expert_rows import (
    ExpertRows,
    permute_tokens,
    permute_tokens_backward,
    permute_tokens_int8,
    sort_by_expert,
    sort_by_expert_reference,
    unpermute_tokens,
    unpermute_tokens_backward,
)
from pplx_kernels_b200.ops.grouped_gemm import grouped_gemm_int8, grouped_gemm_int8_reference
from pplx_kernels_b200.ops.quant import quantize_rows_int8, quantize_rows_int8_reference

M, K, E, H = 6, 3, 5, 64


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def meta_rows(m=M, k=K, experts=E, capacity=0):
    return sort_by_expert(meta(m, k, dtype=torch.int32), experts, capacity)


@pytest.mark.parametrize("capacity,bound_m", [(0, None), (4, None), (0, 7), (2, 0)])
def test_oracle_of_the_sort(capacity, bound_m):
    gen = torch.Generator().manual_seed(1)
    idx = torch.randint(-2, E + 2, (20, K), generator=gen, dtype=torch.int32)
    rows = sort_by_expert_reference(idx, E, capacity, bound_m)
    assert rows.offsets[0] == 0 and rows.offsets.numel() == E + 1
    seen = 0
    for e in range(E):
        mine = [(t, k) for t in range(20) for k in range(K)
                if idx[t, k] == e and (bound_m is None or t < bound_m)]
        kept = mine[:capacity] if capacity else mine
        assert rows.counts[e] == len(kept)
        for i, (t, k) in enumerate(kept):
            assert rows.row_of[t, k] == rows.offsets[e] + i
        seen += len(kept)
    assert int((rows.row_of >= 0).sum()) == seen
    assert rows.shape() == ((E, capacity) if capacity else (60,))


def test_oracle_of_the_quantisation():
    x = torch.tensor([[127.0, -63.5, 0.5, 0.0], [0.0, 0.0, 0.0, 0.0], [1e-3, 2e-3, -4e-3, 3e-3]])
    q, s = quantize_rows_int8_reference(x)
    assert q[0].tolist() == [127, -64, 0, 0] and q[1].tolist() == [0] * 4 and q[2, 2] == -127
    # Half a step of the scale, and the rounding of x * (127 / a): at most 127 * 2^-23 steps.
    assert ((q * s[:, None] - x).abs() <= 0.50002 * s[:, None]).all()


def test_oracle_of_the_product():
    gen = torch.Generator().manual_seed(2)
    x = torch.randint(-127, 128, (7, 32), generator=gen, dtype=torch.int8)
    w = torch.randint(-127, 128, (2, 8, 32), generator=gen, dtype=torch.int8)
    sx, sw = torch.rand(7, generator=gen), torch.rand(2, 8, generator=gen)
    counts, offsets = torch.tensor([3, 2]), torch.tensor([0, 3])
    y = grouped_gemm_int8_reference(x, sx, w, sw, counts, offsets)
    r, n = 4, 5
    want = sum(int(a) * int(b) for a, b in zip(x[r].tolist(), w[1, n].tolist())) \
        * float(sx[r]) * float(sw[1, n])
    assert abs(float(y[r, n]) - want) <= 1e-12 * abs(want) and (y[5:] == 0).all()


def test_shapes():
    rows = meta_rows()
    assert permute_tokens(meta(M, H, dtype=torch.float8_e4m3fn), rows).shape == (M * K, H)
    q, s = permute_tokens_int8(meta(M, H), meta_rows(capacity=9))
    assert q.shape == (E, 9, H) and s.shape == (E, 9) and q.dtype == torch.int8
    assert unpermute_tokens(meta(M * K, H), rows, meta(M, K)).shape == (M, H)
    assert permute_tokens_backward(meta(M * K, H), rows).shape == (M, H)
    gy, gw = unpermute_tokens_backward(meta(M, H), meta(M * K, H), rows, meta(M, K), need_y=False)
    assert gy is None and gw.shape == (M, K)
    assert quantize_rows_int8(meta(E, 4, H))[1].shape == (E, 4)


@pytest.mark.parametrize("call,text", [
    (lambda: sort_by_expert(meta(M, K), E), "int32, uint32 or int64"),
    (lambda: sort_by_expert(meta(M, 0, dtype=torch.int32), E), "contiguous"),
    (lambda: sort_by_expert(meta(K, M, dtype=torch.int32).t(), E), "contiguous"),
    (lambda: sort_by_expert(meta(M, K, dtype=torch.int32), 1025), "num_experts"),
    (lambda: sort_by_expert(meta(M, K, dtype=torch.int32), E, -1), "capacity"),
    (lambda: sort_by_expert(meta(M, K, dtype=torch.int32), E, 1 << 29), "rows"),
    (lambda: sort_by_expert(meta(M, K, dtype=torch.int32), E, 0, meta(1)), "bound_m"),
    (lambda: sort_by_expert(meta(M, K, dtype=torch.int32), E, 0, meta(2, dtype=torch.int32)),
     "bound_m"),
    (lambda: permute_tokens(meta(M + 1, H), meta_rows()), "token count"),
    (lambda: permute_tokens(meta(H, M).t(), meta_rows()), "contiguous"),
    (lambda: permute_tokens(meta(1, H).expand(M, H), meta_rows()), "overlap"),
    (lambda: permute_tokens(meta(M, H), meta_rows(), out=meta(M * K, H + 1)), "must be"),
    (lambda: permute_tokens(meta(M, H), meta_rows(), out=meta(M * K, H, dtype=torch.int32)), "type"),
    (lambda: permute_tokens(meta(M, H), meta_rows(capacity=4), out=meta(E * 4, H)), "must be"),
    (lambda: permute_tokens(meta(M, H).requires_grad_(), meta_rows(), out=meta(M * K, H)), "gradient"),
    (lambda: permute_tokens(meta(M, H).requires_grad_(), meta_rows(), zero_rest=False), "gradient"),
    (lambda: permute_tokens(meta(M, H), ExpertRows(meta(E), meta(E + 1), meta(M, K))), "int32"),
    (lambda: permute_tokens_int8(meta(M, H, dtype=torch.int8), meta_rows()), "bfloat16"),
    (lambda: permute_tokens_int8(meta(M, H), meta_rows(), out_scale=meta(M)), "out_scale"),
    (lambda: permute_tokens_int8(meta(M, H).requires_grad_(), meta_rows()), "gradient"),
    (lambda: unpermute_tokens(meta(M * K - 1, H), meta_rows()), "must be"),
    (lambda: unpermute_tokens(meta(M * K, H, dtype=torch.int32), meta_rows()), "bfloat16"),
    (lambda: unpermute_tokens(meta(M * K, H), meta_rows(), meta(M, K, dtype=torch.bfloat16)),
     "float32"),
    (lambda: unpermute_tokens(meta(M * K, H), meta_rows(), meta(M, K + 1)), "weights"),
    (lambda: unpermute_tokens(meta(M * K, H), meta_rows(), out=meta(M - 1, H)), "fewer rows"),
    (lambda: unpermute_tokens(meta(M * K, H), meta_rows(), out=meta(M, H, dtype=torch.float16)),
     "type"),
    (lambda: unpermute_tokens(meta(M * K, H), meta_rows(), out=meta(1, H).expand(M, H)), "overlap"),
    (lambda: unpermute_tokens_backward(meta(M, H), meta(M * K, H, dtype=torch.float16), meta_rows(),
                                       meta(M, K)), "type"),
    (lambda: quantize_rows_int8(meta(H)), "must be"),
    (lambda: quantize_rows_int8(meta(E, 4, H).transpose(0, 1)), "evenly"),
    (lambda: quantize_rows_int8(meta(4, H), counts=meta(E, dtype=torch.int32)), "counts"),
    (lambda: quantize_rows_int8(meta(E, 4, H), counts=meta(E, dtype=torch.int64)), "counts"),
    (lambda: quantize_rows_int8(meta(4, H).requires_grad_()), "gradient"),
])
def test_refusals(call, text):
    with pytest.raises((RuntimeError, ValueError), match=text):
        call()


def gemm(**changes):
    i8, i32 = torch.int8, torch.int32
    args = dict(xq=meta(E, 4, H, dtype=i8), x_scale=meta(E, 4), wq=meta(E, 16, H, dtype=i8),
                w_scale=meta(E, 16), counts=meta(E, dtype=i32))
    args.update(changes)
    return grouped_gemm_int8(**args)


def test_product_shapes():
    i8, i32 = torch.int8, torch.int32
    assert gemm().shape == (E, 4, 16)
    assert gemm(counts=None, swiglu=True, out_dtype=torch.float16).shape == (E, 4, 8)
    assert gemm(xq=meta(9, H, dtype=i8), x_scale=meta(9), offsets=meta(E + 1, dtype=i32)).shape == (9, 16)


@pytest.mark.parametrize("changes,text", [
    ({"xq": meta(E, 4, H)}, "int8"),
    ({"x_scale": meta(E, 5)}, "x_scale"),
    ({"w_scale": meta(E, 8)}, "w_scale"),
    ({"w_scale": meta(16, E).t()}, "w_scale"),
    ({"wq": meta(E, 16, 2 * H, dtype=torch.int8)}, "wq must be"),
    ({"xq": meta(E, 4, H, dtype=torch.int8)[:, :, :40], "wq": meta(E, 16, H, dtype=torch.int8)[:, :, :40]},
     "multiple of 16"),
    ({"xq": meta(E, 4, H + 8, dtype=torch.int8)[:, :, :H]}, "multiples of 16 bytes"),
    ({"xq": meta(1, 1, 1 << 17, dtype=torch.int8), "x_scale": meta(1, 1), "counts": None,
      "wq": meta(1, 16, 1 << 17, dtype=torch.int8), "w_scale": meta(1, 16)}, "at most 131071"),
    ({"wq": meta(E, 12, H, dtype=torch.int8), "w_scale": meta(E, 12)}, "multiple of 8"),
    ({"wq": meta(E, 15, H, dtype=torch.int8), "w_scale": meta(E, 15), "swiglu": True}, "wq must be"),
    ({"out": meta(E, 4, 16)}, "bfloat16 or float16"),
    ({"out": meta(E, 5, 16, dtype=torch.bfloat16)}, "disagree"),
    ({"counts": meta(E, dtype=torch.int64)}, "counts"),
    ({"counts": meta(E + 1, dtype=torch.int32)}, "counts"),
    ({"offsets": meta(E, dtype=torch.int32)}, "where offsets are given"),
    ({"xq": meta(9, H, dtype=torch.int8), "x_scale": meta(9), "counts": None,
      "offsets": meta(E, dtype=torch.int32)}, "offsets need counts"),
    ({"status": meta(1, dtype=torch.int64)}, "status"),
    ({"expected_rows": -1}, "expected_rows"),
])
def test_product_refusals(changes, text):
    with pytest.raises(RuntimeError, match=text):
        gemm(**changes)


def test_cpu_tensors_are_refused():
    with pytest.raises((RuntimeError, NotImplementedError)):
        sort_by_expert(torch.zeros(2, 2, dtype=torch.int32), 4)
