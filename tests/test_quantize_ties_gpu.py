"""Rows to 8-bit integers, value by value: the factor of a row is 127 times the rounded reciprocal of its
largest magnitude, its scale the largest times the rounded 1/127, each step rounded to fp32.  That is
what ``127.0 / a`` and ``a / 127.0`` of a tensor compute on a GPU, and it decides values that lie on the
border of two integers."""

import numpy as np
import pytest
import torch

from pplx_kernels_b200.ops.expert_rows import permute_tokens_int8, sort_by_expert
from pplx_kernels_b200.ops.quant import quantize_rows_int8, quantize_rows_int8_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def plain(x):
    v = x.float()
    a = v.abs().amax(dim=-1).clamp(min=1e-30)
    q = torch.round(v * (127.0 / a).unsqueeze(-1)).clamp(-127, 127).to(torch.int8)
    return q, a / 127.0


def step_by_step(x):
    v = x.float().cpu().numpy()
    a = np.maximum(np.abs(v).max(axis=-1), np.float32(1e-30))
    factor = np.float32(127) * (np.float32(1) / a)
    q = np.clip(np.rint(v * factor[..., None]), -127, 127).astype(np.int8)
    scale = a * (np.float32(1) / np.float32(127))
    assert q.dtype == np.int8 and scale.dtype == np.float32 and factor.dtype == np.float32
    return torch.from_numpy(q).to(x.device), torch.from_numpy(scale).to(x.device)


def tied(rows, k, dtype, seed):
    """Rows of which many values are exact halves of their factor: amplitudes that are whole numbers of
    sixteenths, values (2 j + 1) / 254 of them where the type has those."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, k, generator=gen, device=DEV)
    x *= torch.exp2(2 * torch.rand(rows, 1, generator=gen, device=DEV) - 1)
    half = torch.randint(0, 127, (rows // 2, k), generator=gen, device=DEV) + 0.5
    x[: rows // 2] = half * torch.randint(1, 256, (rows // 2, 1), generator=gen, device=DEV) / 64
    x[: rows // 2, 0] = 127 * (x[: rows // 2, 1] / half[:, 1])
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k", [(4000, 768), (2000, 401), (500, 7168), (200, 20000), (64, 1)])
def test_every_value(dtype, rows, k):
    x = tied(rows, k, dtype, seed=k) if k > 1 else torch.randn(rows, 1, device=DEV).to(dtype)
    q, s = quantize_rows_int8(x)
    for want_q, want_s in (plain(x), step_by_step(x), quantize_rows_int8_reference(x),
                           quantize_rows_int8_reference(x.cpu())):
        assert torch.equal(q, want_q.to(DEV)) and torch.equal(s, want_s.to(DEV))
    topk, experts = 3, 8
    indices = torch.randint(0, experts, (rows, topk), device=DEV)
    where = sort_by_expert(indices, experts)
    rows_q, rows_s = permute_tokens_int8(x, where)
    at = where.row_of.long()
    assert torch.equal(rows_q[at], q[:, None].expand(-1, topk, -1))
    assert torch.equal(rows_s[at], s[:, None].expand(-1, topk))


def test_largest_and_smallest_rows():
    """Largest magnitudes whose reciprocal is below the normal numbers, and rows below 1e-30."""
    x = torch.randn(40, 300, device=DEV).clamp_(-3, 3) / 3
    x[:, 0] = 1
    size = torch.logspace(-44, 38.5, 40, dtype=torch.float64).clamp(max=3.4e38).float().to(DEV)
    x *= size[:, None]
    q, s = quantize_rows_int8(x)
    want_q, want_s = step_by_step(x)
    assert torch.equal(q, want_q) and torch.equal(s, want_s)
    assert (q[size > 1e-30].abs().amax(1) == 127).all()
