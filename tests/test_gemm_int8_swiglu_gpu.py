"""SwiGLU of the 8-bit expert GEMM over the whole range of gates, the far negative ones too, whose
products with a large up projection are ordinary numbers."""

import pytest
import torch

from pplx_kernels_b200.ops.grouped_gemm import grouped_gemm_int8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1.0, 1e10, 1e30])
@pytest.mark.parametrize("hint", [0, 1])
def test_range_of_gates(dtype, size, hint):
    """Row r, column n: a gate of (r - 64) * gate_scale[n] and an up of size * up_scale[n]."""
    rows, n, k = 129, 64, 16
    xq = torch.zeros(1, rows, k, dtype=torch.int8, device=DEV)
    xq[0, :, 0] = torch.arange(rows, device=DEV) - 64
    xq[0, :, 1] = 1
    wq = torch.zeros(1, 2 * n, k, dtype=torch.int8, device=DEV)
    wq[0, :n, 0] = 1
    wq[0, n:, 1] = 1
    gate_scale = torch.linspace(1e-3, 3.2, n, device=DEV)
    up_scale = size * torch.linspace(0.5, 2, n, device=DEV)
    sx, sw = torch.ones(1, rows, device=DEV), torch.cat([gate_scale, up_scale])[None].contiguous()
    out = grouped_gemm_int8(xq, sx, wq, sw, swiglu=True, out_dtype=dtype, expected_rows=1000 if hint else 0)
    gate = xq[0, :, :1].double() * gate_scale.double()
    up = up_scale.double().expand_as(gate)
    assert float(gate.min()) < -200 and float(gate.max()) > 200
    want = gate * torch.sigmoid(gate) * up
    # Roundings: both products, exp (2 + 1.173 |gate| steps of 2^-23, and the gate's own error), its
    # product, the sum, the quotient (2 steps) and the last product.  exp(-|gate|) below 2^-126
    # has an absolute error of a step or two of 2^-149, which the gate and up multiply.
    info = torch.finfo(dtype)
    rel = 2 * U * (8 + 4 * gate.abs()) + info.eps / 2 * 1.01
    limit = want.abs() * rel + info.smallest_normal * info.eps / 2 + 3 * 2.0 ** -149 * gate.abs() * up
    want = want.clamp(-3e38, 3e38)
    big = want.abs() > info.max  # (beyond the type)
    got = out[0].double()
    assert ((got - want).abs() <= limit)[~big].all(), float(((got - want).abs() / limit)[~big].max())
    far = (gate < -87.4) & (gate > -100) & ~big & (want.abs() > 1e-7)
    assert size < 1e30 or int(far.sum()) > 0  # (so the range is among the values)
    assert (got[far] != 0).all()
