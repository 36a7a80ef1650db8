"""Calls of several threads at once, whose launches take different amounts of shared memory."""

import threading

import pytest
import torch

from pplx_kernels_b200.ops.expert_rows import sort_by_expert
from pplx_kernels_b200.ops.grouped_gemm import grouped_gemm_int8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def in_threads(calls, times):
    """Each call `times` times in a thread and stream of its own, checked against its first result."""
    wanted = [call() for call in calls]
    torch.cuda.synchronize()
    failures = []

    def work(call, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(times):
                    got = call()
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        except BaseException as e:  # noqa: B902 (handed to the test's own thread)
            failures.append(e)

    threads = [threading.Thread(target=work, args=pair) for pair in zip(calls, wanted)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[0]


def test_sorts():
    def call(experts):
        indices = torch.arange(4000, device=DEV, dtype=torch.int32).view(-1, 4) * 7 % experts

        def sort():
            rows = sort_by_expert(indices, experts)
            return rows.counts, rows.offsets, rows.row_of
        return sort

    in_threads([call(e) for e in (1024, 700, 900, 800)], 1500)


def test_products():
    def call(experts):
        gen = torch.Generator(device=DEV).manual_seed(experts)
        x = torch.randint(-99, 99, (experts, 2, 128), generator=gen, device=DEV, dtype=torch.int8)
        w = torch.randint(-99, 99, (experts, 16, 128), generator=gen, device=DEV, dtype=torch.int8)
        sx, sw = (torch.rand(experts, n, generator=gen, device=DEV) for n in (2, 16))
        return lambda: (grouped_gemm_int8(x, sx, w, sw),)

    in_threads([call(e) for e in (1, 40, 90, 200)], 1500)
