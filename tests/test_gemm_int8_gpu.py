"""The grouped GEMM of 8-bit integers against its statement in 64 bits, and the experts of one GPU as a
whole: sorted, quantised, multiplied and brought back."""

import pytest
import torch

from pplx_kernels_b200.ops.expert_rows import (
    permute_tokens,
    permute_tokens_int8,
    sort_by_expert,
    unpermute_tokens,
)
from pplx_kernels_b200.ops.grouped_gemm import (
    grouped_gemm,
    grouped_gemm_int8,
    grouped_gemm_int8_reference,
)
from pplx_kernels_b200.ops.quant import quantize_rows_int8, quantize_rows_int8_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24


def ints(*shape, seed=1):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=gen, device=DEV, dtype=torch.int8)


def scales(*shape, seed=2, size=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (0.5 + torch.rand(shape, generator=gen, device=DEV)) * size


def bound(want, dtype, gate=None, up=None):
    """An exact sum, to fp32, times two scales: 3 roundings.  With SwiGLU those of both products, of
    exp (2 + 1.173 |gate| steps of 2^-23), of the sum, quotient (2 steps) and product; the gate's own
    error counts 1 + |gate| times.  A quotient by more than 2^126 is 0 by its definition
    (__fdividef): that takes exp(-gate) > 2^126, gate < -87.33, where |silu| is below
    87.4 * 2^-126 = 1.03e-36; that, times |up|, is lost.  Then one rounding to the result's type."""
    info = torch.finfo(dtype)
    rel = 3 * U if gate is None else 2 * U * (8 + 4 * gate.abs())
    lost = 0 if up is None else 1.1e-36 * up.abs()
    return want.abs() * (rel + info.eps / 2 * 1.01) + info.smallest_normal * info.eps / 2 + 1e-37 + lost


def check(out, xq, sx, wq, sw, counts, offsets, swiglu, dtype):
    want = grouped_gemm_int8_reference(xq, sx, wq, sw, counts, offsets, swiglu)
    gate = up = None
    if swiglu:
        n = wq.size(1) // 2
        gate, up = (grouped_gemm_int8_reference(xq, sx, wq[:, h], sw[:, h].contiguous(), counts, offsets)
                    for h in (slice(0, n), slice(n, 2 * n)))
    limit = bound(want, dtype, gate, up)
    for e in range(wq.size(0)):
        m = xq.size(-2) if counts is None else int(counts[e])
        mine = slice(int(offsets[e]), int(offsets[e]) + m) if offsets is not None else (e, slice(0, m))
        err = (out[mine].double() - want[mine]).abs()
        assert (err <= limit[mine]).all(), (e, m, float((err / limit[mine]).max()))


COUNTS = [
    [1],
    [300, 0, 1, 17],
    [0, 0, 0, 0, 0],
    [16, 32, 33, 64, 128, 129, 255, 256, 257],
    [513, 2, 700, 0, 96],
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("k,n", [(16, 8), (272, 136), (1024, 264)])
def test_both_layouts(dtype, swiglu, counts, k, n):
    E, rows = len(counts), max(counts) + 3
    wq, sw = ints(E, 2 * n if swiglu else n, k), scales(E, 2 * n if swiglu else n, size=0.02 / k)
    cnt = torch.tensor(counts, dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for hint in (0, sum(counts)):
        # [experts, rows, k]: rows beyond a count are neither read into a result nor written.
        xq, sx = ints(E, rows, k, seed=3), scales(E, rows, seed=4)
        for e, m in enumerate(counts):
            sx[e, m:] = float("nan")
        out = torch.full((E, rows, n), float("nan"), dtype=dtype, device=DEV)
        grouped_gemm_int8(xq, sx, wq, sw, cnt, swiglu=swiglu, out=out, status=status, expected_rows=hint)
        check(out, xq, sx, wq, sw, cnt, None, swiglu, dtype)
        for e, m in enumerate(counts):
            assert out[e, m:].isnan().all()
        # One expert's rows after the other's, with a gap and a tail that belong to none.
        first = torch.cumsum(cnt + 1, 0).to(torch.int32) - cnt
        total = int(first[-1]) + counts[-1] + 2
        xq, sx = ints(total, k, seed=5), scales(total, seed=6)
        mine = torch.zeros(total, dtype=torch.bool, device=DEV)
        for e, m in enumerate(counts):
            mine[int(first[e]) : int(first[e]) + m] = True
        out = torch.full((total, n), float("nan"), dtype=dtype, device=DEV)
        grouped_gemm_int8(xq, sx, wq, sw, cnt, first, swiglu, out, status=status, expected_rows=hint)
        check(out, xq, sx, wq, sw, cnt, first, swiglu, dtype)
        assert out[~mine].isnan().all()
    assert int(status) == 0


@pytest.mark.parametrize("rows,k,n", [(1, 4096, 512), (5, 14336, 72), (200, 131056, 40), (1000, 2816, 2048),
                                      (2500, 192, 1032)])
def test_plain_product(rows, k, n):
    """One matrix, no counts.  All values -128 where K is largest: the largest sum there can be."""
    xq, wq = ints(1, rows, k), ints(1, n, k, seed=2)
    if k > 100000:
        xq.fill_(-128)
        wq.fill_(-128)
    sx, sw = scales(1, rows), scales(1, n, size=1e-6)
    out = grouped_gemm_int8(xq, sx, wq, sw)
    check(out, xq, sx, wq, sw, None, None, False, torch.bfloat16)


def test_strides_and_counts_that_do_not_fit():
    E, rows, k, n = 3, 40, 96, 24
    xq, wq = ints(E, rows, 2 * k)[:, :, 16 : 16 + k], ints(2 * E, n, k + 16)[::2, :, :k]
    sx, sw = scales(E, rows), scales(E, n, size=1e-3)
    wide = torch.full((E, rows, n + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    cnt = torch.tensor([rows + 1000, -5, 13], dtype=torch.int32, device=DEV)
    grouped_gemm_int8(xq, sx, wq, sw, cnt, out=wide[:, :, :n])
    fits = torch.tensor([rows, 0, 13], dtype=torch.int32, device=DEV)
    check(wide[:, :, :n], xq, sx, wq, sw, fits, None, False, torch.bfloat16)
    assert (wide[:, :, n:] == 7).all() and (wide[1] == 7).all() and (wide[2, 13:] == 7).all()
    x2 = xq[0]
    out = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device=DEV)
    cnt = torch.tensor([2 ** 31 - 1, 5, 6], dtype=torch.int32, device=DEV)
    first = torch.tensor([30, -(2 ** 31), 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    grouped_gemm_int8(x2, sx[0], wq, sw, cnt, first, out=out)
    fits, first = torch.tensor([10, 5, 0]), torch.tensor([30, 0, 40])
    check(out, x2, sx[0], wq, sw, fits, first, False, torch.bfloat16)
    assert (out[5:30] == 7).all()


def test_no_rows():
    out = grouped_gemm_int8(ints(2, 0, 64), scales(2, 0), ints(2, 16, 64), scales(2, 16))
    assert out.shape == (2, 0, 16)


def test_rows_that_are_not_finite():
    """A scale that is not finite makes its row so, and no other."""
    xq, wq = ints(1, 20, 64), ints(1, 16, 64)
    sx, sw = scales(1, 20), scales(1, 16, size=1e-3)
    sx[0, 3], sx[0, 11] = float("nan"), float("inf")
    out = grouped_gemm_int8(xq, sx, wq, sw)[0]
    finite = out.isfinite().all(1)
    assert not finite[3] and not out[11].isfinite().any() and int(finite.sum()) == 18


def test_many_experts_and_large_tensors():
    """1024 experts; weights beyond 4 GB, so offsets pass 32 bits."""
    E, k, n = 1024, 2048, 2176
    wq = torch.empty(E, n, k, dtype=torch.int8, device=DEV)
    wq.copy_(ints(1, n, k).expand(E, n, k))
    wq[:, 0, 0] = (torch.arange(E, device=DEV) % 100).to(torch.int8)
    sw = scales(E, n, size=1e-4)
    cnt = torch.zeros(E, dtype=torch.int32, device=DEV)
    cnt[0], cnt[500], cnt[1023] = 3, 40, 20
    first = torch.cumsum(cnt, 0).to(torch.int32) - cnt
    xq, sx = ints(63, k), scales(63)
    out = grouped_gemm_int8(xq, sx, wq, sw, cnt, first)
    for e in (0, 500, 1023):
        mine = slice(int(first[e]), int(first[e] + cnt[e]))
        want = grouped_gemm_int8_reference(xq[mine][None], sx[mine][None], wq[e : e + 1], sw[e : e + 1])[0]
        assert ((out[mine].double() - want).abs() <= bound(want, torch.bfloat16)).all()


def test_graph_follows_the_counts():
    E, k, n = 6, 256, 128
    xq, sx, wq, sw = ints(80, k), scales(80), ints(E, 2 * n, k), scales(E, 2 * n, size=1e-3)
    cnt = torch.tensor([5, 0, 3, 60, 1, 2], dtype=torch.int32, device=DEV)
    first = (torch.cumsum(cnt, 0) - cnt).to(torch.int32)
    out = torch.zeros(80, n, dtype=torch.bfloat16, device=DEV)
    grouped_gemm_int8(xq, sx, wq, sw, cnt, first, True, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grouped_gemm_int8(xq, sx, wq, sw, cnt, first, True, out)
    for counts in ([0, 80, 0, 0, 0, 0], [1, 1, 1, 1, 1, 1]):
        cnt.copy_(torch.tensor(counts))
        first.copy_(torch.cumsum(cnt, 0) - cnt)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check(out, xq, sx, wq, sw, cnt, first, True, torch.bfloat16)
        assert out[sum(counts):].isnan().all()


@pytest.mark.parametrize("m", [1, 61, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_experts_in_8_bits(m, dtype):
    """The operators in a row; each against its statement on what the one before it gave."""
    E, topk, hidden, ffn = 16, 4, 512, 384
    gen = torch.Generator(device=DEV).manual_seed(m)
    x = torch.randn(m, hidden, generator=gen, device=DEV).to(dtype)
    idx = torch.rand(m, E, generator=gen, device=DEV).topk(topk, dim=1).indices
    weights = torch.softmax(torch.randn(m, topk, generator=gen, device=DEV), -1)
    w13 = torch.randn(E, 2 * ffn, hidden, generator=gen, device=DEV) * hidden ** -0.5
    w2 = torch.randn(E, hidden, ffn, generator=gen, device=DEV) * ffn ** -0.5
    q13, s13 = quantize_rows_int8(w13)
    q2, s2 = quantize_rows_int8(w2)
    rows = sort_by_expert(idx, E)
    q, s = permute_tokens_int8(x, rows)
    h = grouped_gemm_int8(q, s, q13, s13, rows.counts, rows.offsets, swiglu=True, out_dtype=dtype)
    check(h, q, s, q13, s13, rows.counts, rows.offsets, True, dtype)
    hq, hs = quantize_rows_int8(h)
    want_q, want_s = quantize_rows_int8_reference(h)
    assert torch.equal(hq, want_q) and torch.equal(hs, want_s)
    y = grouped_gemm_int8(hq, hs, q2, s2, rows.counts, rows.offsets, out_dtype=dtype)
    check(y, hq, hs, q2, s2, rows.counts, rows.offsets, False, dtype)
    out = unpermute_tokens(y, rows, weights)
    # The whole against experts in 64 bits that nothing is quantised in: a value is off by half a
    # step of its row's largest (2^-8 of it, uniformly), in x, h and both weights.  Relative to the
    # size of a row of a product the four errors are at most 4 * amax / rms / 254 / sqrt(3), amax /
    # rms of these normal rows below 6 (h: a product of two, below 12), so 0.08 in the mean; an
    # error in x or w13 passes SwiGLU at most doubled.
    xd = x.double()
    want = torch.zeros_like(xd)
    for k in range(topk):
        w = w13[idx[:, k]].double()
        gu = torch.einsum("mh,mfh->mf", xd, w) if m < 100 else None
        if gu is None:
            gu = torch.stack([xd[t] @ w13[idx[t, k]].double().t() for t in range(m)])
        hd = torch.nn.functional.silu(gu[:, :ffn]) * gu[:, ffn:]
        yd = torch.stack([hd[t] @ w2[idx[t, k]].double().t() for t in range(m)])
        want += weights[:, k : k + 1].double() * yd
    assert float((out.double() - want).norm() / want.norm()) < 0.16


def test_experts_of_a_training_step():
    """Rows with a capacity, the experts' products by torch.bmm, and back; all gradients against the
    same step in 64 bits without sorting.  And the forward pass on the bf16 expert GEMM."""
    m, E, topk, hidden, ffn, cap = 90, 8, 2, 64, 48, 20
    gen = torch.Generator(device=DEV).manual_seed(3)

    def rand(*s):
        return torch.randn(s, generator=gen, device=DEV)

    idx = torch.rand(m, E, generator=gen, device=DEV).topk(topk, dim=1).indices
    x, logits, w = rand(m, hidden), rand(m, topk), rand(E, hidden, hidden) * hidden ** -0.5
    g = rand(m, hidden)
    leaves = [t.clone().requires_grad_() for t in (x, logits, w)]
    rows = sort_by_expert(idx, E, capacity=cap)
    assert int((rows.row_of < 0).sum()) > 0  # some are dropped
    xr = permute_tokens(leaves[0], rows)
    out = unpermute_tokens(torch.tanh(torch.bmm(xr, leaves[2])), rows, torch.softmax(leaves[1], -1))
    out.backward(g)
    plain = [t.double().requires_grad_() for t in (x, logits, w)]
    sm = torch.softmax(plain[1], -1)
    kept = (rows.row_of >= 0).double()
    want = sum((sm[:, k] * kept[:, k])[:, None]
               * torch.tanh(torch.einsum("mh,mho->mo", plain[0], plain[2][idx[:, k]]))
               for k in range(topk))
    want.backward(g.double())
    # Sums of at most hidden + 20 terms in fp32, at most four such in a row: relative to the norm
    # of the result well below 4 * 84 * 2^-24 = 2e-5 (matrix products in full fp32).
    for got, ref in [(out.detach(), want.detach())] + [(a.grad, b.grad) for a, b in zip(leaves, plain)]:
        assert float((got.double() - ref).norm() / ref.norm()) < 2e-5
    xb = permute_tokens(x.bfloat16(), rows)
    y = grouped_gemm(xb, w.transpose(1, 2).contiguous().bfloat16(), rows.counts)
    got = unpermute_tokens(y, rows)
    ref = sum(kept[:, k : k + 1] * torch.einsum(
        "mh,mho->mo", x.bfloat16().double(), w.bfloat16().double()[idx[:, k]]) for k in range(topk))
    # Two roundings to bf16 (2^-9 each in the mean square at most 2^-8 / sqrt(3)).
    assert float((got.double() - ref).norm() / ref.norm()) < 2 ** -8 * 1.2
