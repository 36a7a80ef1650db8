"""A padded batch through the int8 layer of one GPU: rows that no token has are not worked on."""

import pytest
import torch

from pplx_kernels_b200.models.configs import TINY
from pplx_kernels_b200.models.moe import MoELayerInt8
from pplx_kernels_b200.utils.testing import as_index_tensor, routing

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("m,bound", [(40, 17), (40, 0), (40, 40), (40, 99), (1, 0), (0, 0)])
@pytest.mark.parametrize("captured", [False, True])
def test_rows_behind_the_last_expert(m, bound, captured):
    layer = MoELayerInt8(TINY, max_num_tokens=44, init_std=0.05)
    gen = torch.Generator().manual_seed(m + bound)
    topk = TINY.experts_per_token
    x = torch.randn(m, TINY.hidden_dim, generator=gen).to(torch.bfloat16).to(DEV)
    idx = as_index_tensor(routing(m, TINY.num_experts, topk, gen), DEV)
    w = torch.softmax(torch.randn(m, topk, generator=gen), dim=-1).to(DEV)
    live = min(m, bound)
    want = layer(x[:live].contiguous(), idx[:live], w[:live])[:live].clone()
    bound_m = torch.tensor([bound], dtype=torch.int32, device=DEV)
    buffers = [layer.expert_x, layer.expert_scale, layer.h, layer.h_q, layer.h_scale, layer.expert_y]
    out = torch.zeros(44, TINY.hidden_dim, dtype=torch.bfloat16, device=DEV)

    def run():
        layer(x, idx, w, out=out, bound_m=bound_m)

    run()
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        run = graph.replay
    for b in buffers:
        b.fill_(9)
    out.fill_(7)
    run()
    torch.cuda.synchronize()
    layer.check_status()
    assert torch.equal(out[:live], want) and (out[live:] == 7).all()
    for b in buffers:
        assert (b[live * topk:] == 9).all()
