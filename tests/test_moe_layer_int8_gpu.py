"""The int8 MoE layer: on one GPU (sorted rows) and as ranks of an all-to-all (int8 payload with one
scale per token), against its plain statement."""

import pytest
import torch

from pplx_kernels_b200.models.configs import TINY, MoEModelConfig
from pplx_kernels_b200.models.moe import MoELayerInt8, moe_reference_int8
from pplx_kernels_b200.utils.testing import as_index_tensor, routing

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def inputs(cfg, m, seed=3):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, cfg.hidden_dim, generator=gen).to(torch.bfloat16)
    idx = routing(m, cfg.num_experts, cfg.experts_per_token, gen)
    w = torch.softmax(torch.randn(m, cfg.experts_per_token, generator=gen), dim=-1)
    return x.to(DEV), idx.to(DEV), w.to(DEV)


def check(out, want):
    """The kernels' sums are exact, the statement's in fp32: the bf16 of h can differ by one step
    (2^-8 of the value) where it is next to a border, and its 8-bit value by one step of 1/127 of the
    row's largest.  Both are rare, so a result is off by the final roundings (2^-8 of each of top-k
    terms, 2^-9 twice) and by a few of up to `ffn` terms moved by one step each: against the row's
    norm, sqrt(share moved) / 127 * (largest / rms, below 12), below 1e-2 for a share of 1 %."""
    err, size = (out.double() - want.double()), want.double()
    assert float(err.norm() / size.norm()) < 2 ** -7
    assert float(err.abs().max()) <= 2 ** -7 * float(size.abs().max()) + 0.03 * float(size.norm(dim=1).max())


@pytest.mark.parametrize("cfg,m", [(TINY, 1), (TINY, 40), (MoEModelConfig("a", 4, 2, 512, 272), 200),
                                   (MoEModelConfig("b", 2, 2, 256, 256), 700)])
def test_one_gpu(cfg, m):
    layer = MoELayerInt8(cfg, max_num_tokens=m + 3, init_std=0.05)
    x, idx, w = inputs(cfg, m)
    want = moe_reference_int8(x, idx, w, *layer.dequantized_weights())
    out = layer(x, as_index_tensor(idx, DEV), w)
    check(out[:m], want)
    assert torch.equal(layer(x, idx.long(), w)[:m], out[:m])
    assert int(layer.counts.sum()) == m * cfg.experts_per_token
    # A padded batch: tokens at or beyond bound_m change nothing.
    bound = m // 2
    x2 = x.clone()
    x2[bound:] = float("nan")
    mine = torch.full((m, cfg.hidden_dim), 7.0, dtype=torch.bfloat16, device=DEV)
    layer(x2, idx, w, out=mine, bound_m=torch.tensor([bound], dtype=torch.int32, device=DEV))
    assert torch.equal(mine[:bound], out[:bound]) and (mine[bound:] == 7).all()
    layer.check_status()
    with pytest.raises(ValueError, match="room for"):
        layer(torch.zeros(m + 4, cfg.hidden_dim, dtype=torch.bfloat16, device=DEV), idx, w)
    layer.destroy()


def test_graph():
    cfg, m = TINY, 32
    layer = MoELayerInt8(cfg, max_num_tokens=m, init_std=0.05)
    x, idx, w = inputs(cfg, m)
    idx = as_index_tensor(idx, DEV)
    out = torch.zeros(m, cfg.hidden_dim, dtype=torch.bfloat16, device=DEV)
    layer(x, idx, w, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x, idx, w, out=out)
    for seed in (4, 5):
        x2, idx2, w2 = inputs(cfg, m, seed)
        x.copy_(x2), idx.copy_(as_index_tensor(idx2, DEV)), w.copy_(w2)
        graph.replay()
        check(out, moe_reference_int8(x2, idx2, w2, *layer.dequantized_weights()))
    layer.check_status()


@pytest.mark.parametrize("world,dp_size", [(2, 1), (4, 2)])
def test_ranks(world, dp_size):
    """The layers of all ranks on one GPU, each step launched for all ranks before the next."""
    import pplx_kernels_b200 as pk
    from pplx_kernels_b200.ops.grouped_gemm import grouped_gemm_int8
    from pplx_kernels_b200.ops.quant import quantize_rows_int8

    cfg, m = MoEModelConfig("r", 8, 2, 512, 256), 60
    atas = pk.AllToAll.local_world(m, cfg.num_experts, cfg.experts_per_token, world, dp_size,
                                   cfg.hidden_dim, cfg.hidden_dim, 4)
    layers = [MoELayerInt8(cfg, m, rank=r, world_size=world, dp_size=dp_size, device=DEV, ata=atas[r],
                           init_std=0.05) for r in range(world)]
    data = [inputs(cfg, m, seed=g) for g in range(world // dp_size)]
    mine = [data[r // dp_size] for r in range(world)]
    idx = [as_index_tensor(d[1], DEV) for d in mine]
    outs = [torch.full((m, cfg.hidden_dim), float("nan"), dtype=torch.bfloat16, device=DEV)
            for _ in range(world)]
    deq = [l.dequantized_weights() for l in layers]
    w13, w2 = torch.cat([d[0] for d in deq]), torch.cat([d[1] for d in deq])
    q = [quantize_rows_int8(d[0]) for d in mine]
    pk.dispatch_group(atas, [l.counts for l in layers], [l.expert_x for l in layers],
                      [l.expert_scale.unsqueeze(-1) for l in layers], [a for a, _ in q],
                      [b.unsqueeze(-1) for _, b in q], idx, [None] * world)
    for l in layers:
        grouped_gemm_int8(l.expert_x, l.expert_scale, l.w13_q, l.w13_s, l.counts, swiglu=True, out=l.h,
                          status=l.gemm_status)
        quantize_rows_int8(l.h, l.counts, out=l.h_q, out_scale=l.h_scale)
        grouped_gemm_int8(l.h_q, l.h_scale, l.w2_q, l.w2_s, l.counts, out=l.expert_y,
                          status=l.gemm_status)
    pk.combine_group(atas, outs, idx, [d[2] for d in mine], [l.expert_y for l in layers], [None] * world)
    torch.cuda.synchronize()
    for r, l in enumerate(layers):
        l.check_status()
        x, i, w = mine[r]
        check(outs[r], moe_reference_int8(x, i, w, w13, w2))
        l.destroy()


def test_one_rank_of_an_all_to_all():
    """The layer's own way through dispatch and combine, in a world of one rank."""
    import pplx_kernels_b200 as pk

    cfg, m = TINY, 40
    ata = pk.AllToAll.intranode(m, cfg.num_experts, cfg.experts_per_token, 0, 1, 1, cfg.hidden_dim,
                                cfg.hidden_dim, 4)
    through, local = MoELayerInt8(cfg, m, init_std=0.05, ata=ata), MoELayerInt8(cfg, m, init_std=0.05)
    x, idx, w = inputs(cfg, m)
    idx = as_index_tensor(idx, DEV)
    a, b = through(x, idx, w), local(x, idx, w)
    torch.cuda.synchronize()
    through.check_status()
    # The same products; the sums of top-2 terms in fp32 in the same order, rounded once.
    assert torch.equal(through.counts, local.counts)
    assert ((a.float() - b.float()).abs() <= 2 ** -7 * b.float().abs() + 1e-6).all()
    through.destroy()
