"""The layer benchmark with 8-bit integers: figures of the form that ran and of no other."""

import pytest
import torch

from pplx_kernels_b200.utils.bench_moe import measure

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
def test_measure(graph):
    got = measure("tiny", 4, 2, 1, 0, 1, torch.device("cuda", 0), graph=graph, int8=True)
    assert got["composed_us_p50"] > 0 and got["composed_tokens_per_s"] > 0
    assert 0 < got["best_frac_of_roofline"] < 1
    assert not any("fused" in key for key in got)
    assert "reference" in got["output_checked"]
