"""What the layer benchmark reports of the forms that ran."""

import pytest

from pplx_kernels_b200.utils import bench_moe

FLOORS = {"compute_us": 40.0}


def test_both_forms():
    got = bench_moe._figures({"composed": 100.0, "fused": 80.0}, 16, FLOORS, 40.0)
    assert got == {"composed_us_p50": 100.0, "fused_us_p50": 80.0, "fused_tokens_per_s": pytest.approx(2e5),
                   "composed_tokens_per_s": pytest.approx(1.6e5), "floors_us": FLOORS,
                   "fused_frac_of_roofline": 0.5, "best_frac_of_roofline": 0.5}


def test_a_layer_without_a_fused_form():
    got = bench_moe._figures({"composed": 100.0}, 16, FLOORS, 40.0)
    assert not any("fused" in key for key in got)
    assert got["composed_us_p50"] == 100.0 and got["best_frac_of_roofline"] == pytest.approx(0.4)
