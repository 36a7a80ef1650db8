"""Tokens sorted by expert and back, and rows of 8-bit integers, against plain statements in 64 bits.

Tolerances count roundings: one of the result's type (half a step, eps / 2 of the value) behind sums
in fp32 (2^-24 of the sum of magnitudes per term)."""

import pytest
import torch

from pplx_kernels_b200.ops.expert_rows import (
    permute_tokens,
    permute_tokens_backward,
    permute_tokens_int8,
    sort_by_expert,
    sort_by_expert_reference,
    unpermute_tokens,
    unpermute_tokens_backward,
)
from pplx_kernels_b200.ops.quant import quantize_rows_int8, quantize_rows_int8_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
FLOATS = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def routing(m, topk, experts, seed=0, wild=0.0, dtype=torch.int32):
    """Random experts, the same one twice among them; with `wild`, numbers that are none."""
    gen = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, experts, (m, topk), generator=gen)
    if wild:
        bad = torch.rand(m, topk, generator=gen) < wild
        idx = torch.where(bad, torch.randint(0, 2, (m, topk), generator=gen) * (experts + 1) - 1, idx)
    if dtype == torch.uint32:
        return idx.to(torch.int32).to(DEV).view(torch.uint32)
    return idx.to(dtype).to(DEV)


def data(*shape, dtype=torch.float32, seed=1):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


def token_of(rows, total):
    """Token of every row on the host, -1 for none."""
    m, topk = rows.row_of.shape
    token = torch.full((total,), -1, dtype=torch.int64)
    row = rows.row_of.cpu().flatten().long()
    token[row[row >= 0]] = (torch.arange(m * topk) // topk)[row >= 0]
    return token.to(DEV)


def half_step(want, dtype):
    """Rounding of `want` to dtype: half a step, of the smallest numbers too."""
    info = torch.finfo(dtype)
    return info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2


@pytest.mark.parametrize("m,topk,experts,capacity,wild,dtype", [
    (0, 2, 4, 0, 0, torch.int32),
    (0, 2, 4, 3, 0, torch.int64),
    (1, 8, 256, 0, 0, torch.uint32),
    (1, 1, 1, 1, 0, torch.int32),
    (3, 8, 8, 2, 0.3, torch.int64),
    (37, 1, 1, 0, 0.5, torch.uint32),
    (77, 8, 256, 0, 0.75, torch.int32),
    (129, 6, 64, 13, 0.1, torch.int32),
    (1000, 8, 1024, 0, 0, torch.int64),
    (1000, 40, 3, 9999, 0, torch.int32),
    (4095, 8, 256, 100, 0, torch.uint32),
    (40001, 8, 127, 0, 0.01, torch.int32),
    (140001, 2, 1000, 300, 0.01, torch.int32),
])
def test_sort(m, topk, experts, capacity, wild, dtype):
    idx = routing(m, topk, experts, wild=wild, dtype=dtype)
    for bound in (None, 0, m // 3, m, m + 5) if m in (3, 77, 4095) else (None,):
        bound_m = None if bound is None else torch.tensor([bound], dtype=torch.int32, device=DEV)
        rows = sort_by_expert(idx, experts, capacity, bound_m)
        plain = idx.view(torch.int32) if dtype == torch.uint32 else idx
        want = sort_by_expert_reference(plain.cpu(), experts, capacity, bound)
        assert torch.equal(rows.counts.cpu(), want.counts)
        assert torch.equal(rows.offsets.cpu(), want.offsets)
        assert torch.equal(rows.row_of.cpu(), want.row_of)


def test_sort_of_one_expert():
    """All entries to one expert, the last, and 64-bit numbers whose low words are experts."""
    idx = torch.full((5000, 4), 299, device=DEV, dtype=torch.int64)
    rows = sort_by_expert(idx, 300)
    assert torch.equal(rows.row_of.flatten().cpu(), torch.arange(20000, dtype=torch.int32))
    rows = sort_by_expert(idx + (1 << 32), 300)
    assert int(rows.counts.sum()) == 0 and (rows.row_of == -1).all() and (rows.offsets == 0).all()


@pytest.mark.parametrize("dtype", [torch.uint8, torch.float8_e4m3fn, torch.bfloat16, torch.float32,
                                   torch.float64])
@pytest.mark.parametrize("hidden", [1, 7, 129, 256, 1000, 2048, 7168])
@pytest.mark.parametrize("capacity", [0, 5])
def test_permute(dtype, hidden, capacity):
    m, topk, experts = 33, 3, 8
    rows = sort_by_expert(routing(m, topk, experts, wild=0.2), experts, capacity)
    wide = data(m, hidden + 16).to(dtype)
    for x in (wide[:, :hidden], wide[:, :hidden].contiguous(), wide[:, 1 : hidden + 1]):
        total = experts * capacity if capacity else m * topk
        out = torch.full((*rows.shape(), hidden), 3, device=DEV).to(dtype)
        before = out.clone()
        permute_tokens(x, rows, out=out)
        token = token_of(rows, total)
        there = (token >= 0).view(*rows.shape(), 1)

        def as_bytes(t):
            return t.contiguous().view(torch.uint8)

        size = dtype.itemsize
        want = as_bytes(x)[token.clamp(min=0)].view(*rows.shape(), hidden * size)
        assert torch.equal(as_bytes(out), torch.where(there, want, as_bytes(before)))
        out = permute_tokens(x, rows, zero_rest=True, out=out)
        assert torch.equal(as_bytes(out), torch.where(there, want, torch.zeros_like(want)))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,topk,hidden,capacity", [
    (1, 1, 1, 0), (1, 8, 7168, 0), (5, 2, 129, 3), (33, 9, 1000, 0), (64, 6, 2048, 40),
    (130, 3, 4096, 0), (31, 17, 258, 0),
])
def test_unpermute_and_gradients(dtype, m, topk, hidden, capacity):
    experts = 8
    rows = sort_by_expert(routing(m, topk, experts, wild=0.2), experts, capacity)
    total = experts * capacity if capacity else m * topk
    y = data(total, hidden, dtype=dtype)
    token = token_of(rows, total)
    y[token < 0] = float("nan")  # rows without a token reach no result
    y = y.view(*rows.shape(), hidden)
    w = torch.rand(m, topk, device=DEV) - 0.3
    g = data(m, hidden, dtype=dtype, seed=5)
    row = rows.row_of.long()
    there = row >= 0
    picked = torch.where(there[:, :, None], y.view(total, hidden)[row.clamp(min=0)].double(), 0.0)
    for weights in (w, None):
        wd = torch.ones_like(w).double() if weights is None else w.double()
        terms = picked * wd[:, :, None]
        want, size = terms.sum(1), terms.abs().sum(1) * (topk + 1) * U
        out = unpermute_tokens(y, rows, weights)
        assert ((out.double() - want).abs() <= size + 1.01 * half_step(want.abs() + size, dtype)).all()
    # The same with a gradient: forward, rows, weights.
    yl, wl = y.clone().requires_grad_(), w.clone().requires_grad_()
    out2 = unpermute_tokens(yl, rows, wl)
    assert torch.equal(out2.detach(), unpermute_tokens(y, rows, w))
    out2.backward(g)
    grad_y, grad_w = unpermute_tokens_backward(g, y, rows, w)
    assert torch.equal(grad_y, yl.grad) and torch.equal(grad_w, wl.grad)
    only_y, none = unpermute_tokens_backward(g, y, rows, w, need_weights=False)
    assert none is None and torch.equal(only_y, grad_y)
    none, only_w = unpermute_tokens_backward(g, y, rows, w, need_y=False)
    assert none is None and torch.equal(only_w, grad_w)
    want_w = (picked * g.double()[:, None, :]).sum(-1)
    size = (picked * g.double()[:, None, :]).abs().sum(-1) * (hidden + 1) * U
    assert ((grad_w.double() - want_w).abs() <= size + 1.01 * half_step(want_w, torch.float32)).all()
    assert (grad_w[~there] == 0).all()
    each = (w.double()[:, :, None] * g.double()[:, None, :]).view(m * topk, hidden)
    want_y = torch.zeros(total, hidden, dtype=torch.float64, device=DEV)
    want_y[row[there]] = each[there.flatten()]
    err = (grad_y.view(total, hidden).double() - want_y).abs()
    assert (err <= U * want_y.abs() + 1.01 * half_step(want_y, dtype)).all()
    assert (grad_y.view(total, hidden)[token < 0] == 0).all()
    # The gradient of permute: the sum of a token's rows.
    gr = data(total, hidden, dtype=dtype, seed=6).view(*rows.shape(), hidden)
    x = data(m, hidden, dtype=dtype, seed=7).requires_grad_()
    out3 = permute_tokens(x, rows)
    assert (out3.detach().view(total, hidden)[token < 0] == 0).all()
    out3.backward(gr)
    terms = torch.where(there[:, :, None], gr.view(total, hidden)[row.clamp(min=0)].double(), 0.0)
    want, size = terms.sum(1), terms.abs().sum(1) * (topk + 1) * U
    assert ((x.grad.double() - want).abs() <= size + 1.01 * half_step(want.abs() + size, dtype)).all()
    assert torch.equal(x.grad, permute_tokens_backward(gr, rows))


def test_gradients_against_differences():
    """permute -> a product per row -> unpermute is linear in the tokens and in the weights: a
    difference over any distance is the gradient.  fp32, so a result is off by its roundings alone."""
    m, topk, experts, hidden = 9, 3, 4, 40
    rows = sort_by_expert(routing(m, topk, experts, wild=0.1), experts, 6)
    scale = data(experts, 6, 1, seed=3)
    x, w = data(m, hidden).requires_grad_(), torch.rand(m, topk, device=DEV).requires_grad_()
    g = data(m, hidden, seed=4)

    def loss(x, w):
        out = unpermute_tokens(permute_tokens(x, rows) * scale, rows, w)
        return (out * g).sum(), (out.detach().double() * g.double()).sum()

    loss(x, w)[0].backward()
    for leaf, other in ((x, False), (w, True)):
        d = torch.randn_like(leaf)
        with torch.no_grad():
            ends = [loss(x, w + s * d)[1] if other else loss(x + s * d, w)[1] for s in (1.0, -1.0)]
        slope, want = float(ends[0] - ends[1]) / 2, float((leaf.grad.double() * d.double()).sum())
        # Each result is a sum of topk products of three numbers below 6 in size (of |x| + |d|,
        # scale, weights), off by 6 roundings; `size` bounds the sum over all of them.
        size = m * hidden * topk * 10.0 * 4.0 * 4.0 * 4.0
        assert abs(slope - want) <= 6 * U * size, (slope, want)


def test_expanded_gradient_and_strided_tokens():
    """The gradient of a sum is an expanded tensor; tokens may be columns of a wider tensor."""
    m, topk, hidden = 12, 2, 48
    rows = sort_by_expert(routing(m, topk, 4), 4)
    y = data(m * topk, hidden).requires_grad_()
    w = torch.rand(m, topk, device=DEV)
    unpermute_tokens(y, rows, w).sum().backward()
    assert torch.equal(y.grad[rows.row_of.flatten().long()], w.view(-1, 1).expand(-1, hidden))
    x = data(m, 3 * hidden).requires_grad_()
    permute_tokens(x[:, hidden : 2 * hidden], rows).sum().backward()
    assert (x.grad[:, hidden : 2 * hidden] == topk).all() and (x.grad[:, :hidden] == 0).all()
    out = torch.full((m + 2, 2 * hidden), 7.0, device=DEV)
    got = unpermute_tokens(y.detach(), rows, w, out=out[:, :hidden])
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(out[:m, :hidden], unpermute_tokens(y.detach(), rows, w))
    assert (out[:, hidden:] == 7).all() and (out[m:] == 7).all()


def test_bound_m():
    m, topk, hidden, bound = 20, 2, 64, 13
    rows = sort_by_expert(routing(m, topk, 4), 4, bound_m=torch.tensor(bound, device=DEV, dtype=torch.int32))
    x = data(m, hidden)
    x[bound:] = float("nan")
    y = permute_tokens(x, rows, out=torch.full((m * topk, hidden), 5.0, device=DEV))
    assert (y[bound * topk:] == 5).all() and not y.isnan().any()
    out = torch.full((m, hidden), 7.0, device=DEV)
    unpermute_tokens(y, rows, out=out)
    assert (out[bound:] == 7).all()
    assert torch.equal(out[:bound], topk * x[:bound])
    assert (unpermute_tokens(y, rows)[bound:] == 0).all()
    leaf = x.clone().requires_grad_()
    permute_tokens(leaf, rows).sum().backward()
    assert (leaf.grad[:bound] == topk).all() and (leaf.grad[bound:] == 0).all()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,k", [(0, 64), (1, 1), (1, 16), (3, 127), (7, 768), (5, 1001), (40, 2048),
                                    (9, 7168), (3, 16384), (2, 40010), (300, 512)])
def test_quantize(dtype, rows, k):
    x = data(rows, k + 8, dtype=dtype) * torch.exp2(torch.arange(rows, device=DEV) % 9 - 4)[:, None]
    x = x.to(dtype)
    if rows > 2:
        x[1] = 0
        x[2] = 0
        x[2, k // 2] = 3e-8 if dtype == torch.float16 else 2e-38
    for v in (x[:, :k], x[:, :k].contiguous(), x[:, 1 : k + 1]):
        q, s = quantize_rows_int8(v)
        want_q, want_s = quantize_rows_int8_reference(v)
        assert torch.equal(q, want_q) and torch.equal(s, want_s)


def test_quantize_with_counts():
    x = data(3, 50, 264, dtype=torch.bfloat16)
    counts = torch.tensor([0, 50, 17], dtype=torch.int32, device=DEV)
    q = torch.full((3, 50, 264), 9, dtype=torch.int8, device=DEV)
    s = torch.full((3, 50), 9.0, device=DEV)
    for e, n in enumerate(counts.tolist()):
        x[e, n:] = float("nan")
    quantize_rows_int8(x, counts, q, s)
    for e, n in enumerate(counts.tolist()):
        want_q, want_s = quantize_rows_int8_reference(x[e, :n]) if n else (q[e, :0], s[e, :0])
        assert torch.equal(q[e, :n], want_q) and torch.equal(s[e, :n], want_s)
        assert (q[e, n:] == 9).all() and (s[e, n:] == 9).all()


def test_quantize_what_is_not_finite():
    x = data(4, 300)
    x[0, 5], x[1, 7], x[2, 299], x[2, 0] = float("inf"), float("nan"), float("-inf"), float("nan")
    q, s = quantize_rows_int8(x)
    assert s[0] == float("inf") and s[1].isnan() and s[2].isnan() and s[3].isfinite()
    assert (q[:3] == 0).all()
    want_q, want_s = quantize_rows_int8_reference(x[3:])
    assert torch.equal(q[3:], want_q) and torch.equal(s[3:], want_s)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,topk,hidden,capacity", [(1, 8, 7168, 0), (33, 3, 1000, 5), (70, 6, 2048, 0),
                                                    (10, 2, 129, 0), (3, 33, 16400, 0)])
def test_permute_int8(dtype, m, topk, hidden, capacity):
    experts = 8
    rows = sort_by_expert(routing(m, topk, experts, wild=0.2), experts, capacity)
    total = experts * capacity if capacity else m * topk
    x = data(m, hidden, dtype=dtype)
    want_q, want_s = quantize_rows_int8_reference(x)
    token = token_of(rows, total)
    there = token >= 0
    q = torch.full((*rows.shape(), hidden), 9, dtype=torch.int8, device=DEV)
    s = torch.full(rows.shape(), 9.0, device=DEV)
    for rest in (False, True):
        permute_tokens_int8(x, rows, zero_rest=rest, out=q, out_scale=s)
        q2, s2 = q.view(total, hidden), s.view(total)
        assert torch.equal(q2[there], want_q[token[there]]) and torch.equal(s2[there], want_s[token[there]])
        fill = 0 if rest else 9
        assert (q2[~there] == fill).all() and (s2[~there] == fill).all()


@pytest.mark.parametrize("hidden", [33, 256, 2048])
def test_gradients_that_are_not_finite(hidden):
    """An infinity or a NaN reaches its own token's entries, and of those only the ones with a row."""
    m, topk, experts = 12, 5, 4
    indices = routing(m, topk, experts)
    indices[::2, 3] = -1
    indices[4] = -1
    rows = sort_by_expert(indices, experts)
    y, w = data(m * topk, hidden), torch.rand(m, topk, device=DEV) + 0.5
    g = data(m, hidden, seed=3)
    want_y, want_w = unpermute_tokens_backward(g, y, rows, w)
    bad = g.clone()
    bad[2, 0], bad[4, hidden - 1], bad[6] = float("inf"), float("nan"), float("-inf")
    grad_y, grad_w = unpermute_tokens_backward(bad, y, rows, w)
    there = rows.row_of >= 0
    hit = torch.zeros(m, 1, dtype=torch.bool, device=DEV)
    hit[[2, 4, 6]] = True
    assert torch.equal(grad_w[~(hit & there)], want_w[~(hit & there)])
    assert (grad_w[~there] == 0).all() and not grad_w[hit & there].isfinite().any()
    touched = torch.zeros(m * topk, dtype=torch.bool, device=DEV)
    touched[rows.row_of[hit & there].long()] = True
    assert torch.equal(grad_y[~touched], want_y[~touched])
    assert not grad_y[touched].isfinite().all(1).any()


def test_rows_out_of_range_are_skipped():
    """A table that does not fit the tensors: the kernels leave such entries out."""
    m, topk, hidden = 4, 2, 32
    rows = sort_by_expert(routing(m, topk, 4), 4)
    rows.row_of[0, 0] = m * topk
    rows.row_of[1, 1] = 2 ** 31 - 1
    rows.row_of[2, 0] = -(2 ** 31)
    x = data(m, hidden)
    out = permute_tokens(x, rows, out=torch.zeros(m * topk, hidden, device=DEV))
    back = unpermute_tokens(out, rows)
    grad_y, grad_w = unpermute_tokens_backward(x, out, rows, torch.ones(m, topk, device=DEV))
    q, s = permute_tokens_int8(x, rows)
    left = torch.tensor([1.0, 1.0, 1.0, 2.0], device=DEV)[:, None]
    assert torch.equal(back, left * x)
    assert grad_w[0, 0] == grad_w[1, 1] == grad_w[2, 0] == 0


def test_streams_and_graphs():
    """Two graphs captured on a side stream, replayed with other routing, next to eager calls; the
    functional gradients are captured while an eager graph of the same leaves lives."""
    m, topk, experts, hidden = 50, 4, 16, 512
    idx = [routing(m, topk, experts, seed=s) for s in (1, 2, 3)]
    x, w = data(m, hidden, dtype=torch.bfloat16), torch.rand(m, topk, device=DEV)
    g = data(m, hidden, dtype=torch.bfloat16, seed=9)
    live = idx[0].clone()

    def step():
        rows = sort_by_expert(live, experts)
        y = permute_tokens(x.detach(), rows)
        out = unpermute_tokens(y, rows, w.detach())
        grad_y, grad_w = unpermute_tokens_backward(g, y, rows, w.detach())
        return out, permute_tokens_backward(grad_y, rows), grad_w, permute_tokens_int8(x.detach(), rows)

    xl, wl = x.requires_grad_(), w.requires_grad_()
    eager_rows = sort_by_expert(live, experts)
    eager = unpermute_tokens(permute_tokens(xl, eager_rows), eager_rows, wl)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = step()
        graphs.append((graph, result))
    for i in (1, 2, 0):
        live.copy_(idx[i])
        want = step()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            for a, b in zip(got[:3], want[:3]):
                assert torch.equal(a, b)
            assert torch.equal(got[3][0], want[3][0]) and torch.equal(got[3][1], want[3][1])
    eager.backward(g)
    assert torch.equal(x.grad, want[1]) and torch.equal(w.grad, want[2])


def test_captured_backward_with_leaves_of_its_own():
    """Forward and backward captured as autograd records them, with leaves made in the capture, while an
    eager graph of the tensors behind them lives."""
    m, topk, experts, hidden = 24, 2, 4, 128
    x, w = data(m, hidden).requires_grad_(), torch.rand(m, topk, device=DEV).requires_grad_()
    g = data(m, hidden, seed=2)
    idx = routing(m, topk, experts)

    def step(x, w):
        rows = sort_by_expert(idx, experts)
        out = unpermute_tokens(torch.tanh(permute_tokens(x, rows)), rows, w)
        out.backward(g)
        return out.detach(), x.grad, w.grad

    rows = sort_by_expert(idx, experts)
    eager = unpermute_tokens(torch.tanh(permute_tokens(x, rows)), rows, w)  # lives until the end
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x.detach().requires_grad_(), w.detach().requires_grad_())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x.detach().requires_grad_(), w.detach().requires_grad_())
    with torch.no_grad():
        x.mul_(-0.5)
    idx.copy_(routing(m, topk, experts, seed=9))
    graph.replay()
    want = step(x.detach().requires_grad_(), w.detach().requires_grad_())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert eager.shape == (m, hidden)


def test_second_derivatives():
    """The copy and the plain sum are linear, so their gradients have gradients; that of the weighted
    sum is refused."""
    m, topk, hidden = 6, 2, 32
    rows = sort_by_expert(routing(m, topk, 4), 4)
    x, y = data(m, hidden).requires_grad_(), data(m * topk, hidden, seed=2).requires_grad_()
    g = data(m, hidden, seed=3).requires_grad_()
    (gy,) = torch.autograd.grad(unpermute_tokens(y, rows), y, g, create_graph=True)
    (gg,) = torch.autograd.grad(gy.sum(), g)
    assert (gg == topk).all()
    gr = data(m * topk, hidden, seed=4).requires_grad_()
    (gx,) = torch.autograd.grad(permute_tokens(x, rows), x, gr, create_graph=True)
    (gg,) = torch.autograd.grad(gx.sum(), gr)
    assert (gg == 1).all()
    w = torch.rand(m, topk, device=DEV).requires_grad_()
    with pytest.raises(RuntimeError, match="no derivative of its own"):
        torch.autograd.grad(unpermute_tokens(y, rows, w), w, g, create_graph=True)


def test_rows_behind_four_gigabytes():
    """Offsets into the rows pass 32 bits."""
    m, topk, hidden = 70000, 8, 4096  # 4.6 GB of rows
    rows = sort_by_expert(torch.arange(m * topk, device=DEV, dtype=torch.int32).view(m, topk) % 7, 7)
    x = data(m, hidden, dtype=torch.bfloat16)
    y = permute_tokens(x, rows)
    at = torch.tensor([0, 1, m // 2, m - 1], device=DEV)
    for k in range(topk):
        assert torch.equal(y[rows.row_of[at, k].long()], x[at])
    out = unpermute_tokens(y, rows)
    assert torch.equal(out, topk * x)  # eight times a bf16 is one
    q, s = permute_tokens_int8(x, rows)
    want_q, want_s = quantize_rows_int8_reference(x[at])
    for k in range(topk):
        assert torch.equal(q[rows.row_of[at, k].long()], want_q)


def test_compile():
    m, topk, experts, hidden = 20, 2, 4, 64
    idx, x, w = routing(m, topk, experts), data(m, hidden), torch.rand(m, topk, device=DEV)

    def fn(idx, x, w):
        rows = sort_by_expert(idx, experts)
        return unpermute_tokens(permute_tokens(x, rows) * 2, rows, w)

    got = torch.compile(fn, backend="eager", fullgraph=True)(idx, x, w)
    assert torch.equal(got, fn(idx, x, w))
