"""The grouped GEMM of 8-bit integers where a worker has many tiles: accumulators, scale tables and stages
are taken in turn, wide tiles are two halves, and tiles lie behind the table that is looked up in advance.

`plan` restates how a launch is cut, so that every case says (and asserts) what it reaches."""

import pytest
import torch

from pplx_kernels_b200.ops.grouped_gemm import grouped_gemm_int8

from .test_gemm_int8_gpu import check, ints, scales

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def cut(rows, unit, limit):
    """Widths of an expert's token tiles."""
    units = -(-rows // unit)
    tiles = -(-units * unit // limit)
    return [(units // tiles + (i < units % tiles)) * unit for i in range(tiles)]


def plan(counts, n, k, swiglu, pairs, sms=148):
    """(tiles of the fullest worker, widest tile, widths of all tiles in order)."""
    unit, most, workers = (32, 512, sms // 2) if pairs else (16, 256, sms)
    blocks = -(-n // ((64 if swiglu else 128) * (2 if pairs else 1)))
    limit = most
    if max(counts) > 256:
        best = None
        for cand in range(most, 0, -unit):
            if 4 * cand < most:
                break
            widths = [w for c in counts for w in cut(c, unit, cand)]
            w = sum(widths) // len(widths)
            each = max(330 + 5 * w // 3, 220 + 11 * w // 5, 18 * max(w, 100) // 5 - 340)
            drain = 0 if cand <= 256 else 6 if cand <= 320 else 10
            cost = -(-len(widths) * blocks // workers) * (-(-k // 128) * each + drain * w)
            if best is None or cost < best:
                best, limit = cost, cand
    widths = [w for c in counts for w in cut(c, unit, limit)]
    return -(-len(widths) * blocks // workers), max(widths), widths


MIX = [700, 3, 0, 300, 17, 512, 40, 260, 1, 333, 0, 96, 480, 257, 256, 20]
CASES = {
    # name: (counts, n, k, pairs, least tiles of the fullest worker, widest tile from .. to)
    "three accumulators": ([300] * 37, 1024, 2048, True, 2, 257, 320),
    "three accumulators, odd k": ([289, 290, 320, 319] * 9, 2048, 1200, True, 4, 257, 320),
    "three accumulators, behind the table": ([320, 319, 290] * 37, 6144, 1040, True, 33, 257, 320),
    "halves in two accumulators": ([352] * 37, 1024, 2048, True, 2, 321, 512),
    "halves, many turns": ([352] * 37, 6144, 2048, True, 12, 321, 512),
    "halves of 192": ([384, 400] * 12, 2048, 2048, True, 4, 321, 512),
    "halves of 240": ([500, 470, 512] * 9, 768, 1664, True, 2, 321, 512),
    "wide experts in narrow tiles": ([352] * 37, 4096, 96, True, 8, 65, 256),
    "one accumulator per tile, pairs": ([200, 256, 224] * 13, 1024, 400, True, 2, 193, 256),
    "behind the table": ([20] * 128, 8192, 64, False, 33, 17, 256),
    "near the end of the table, pairs": ([70] * 64, 8192, 80, True, 27, 65, 256),
    "behind the table, pairs": ([270, 300] * 16, 16384, 48, True, 33, 65, 256),
    "more experts than threads": ([3, 40, 0, 17] * 100, 512, 272, False, 8, 33, 256),
    "more experts than threads, pairs": ([3, 40, 0, 17] * 100, 512, 272, True, 8, 33, 256),
    "narrow and wide": (MIX * 4, 1536, 2048, True, 4, 321, 512),
    "narrow and wide, many turns": (MIX * 4, 4096, 1664, True, 8, 321, 512),
    "narrow and wide, single CTAs": (MIX, 4096, 1040, False, 3, 193, 256),
}


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_many_tiles(name, swiglu):
    counts, n, k, pairs, tiles, least, most = CASES[name]
    n = n // 2 if swiglu else n  # (the same number of weight rows and tiles)
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    per_worker, widest, _ = plan(counts, n, k, swiglu, pairs, sms)
    if sms == 148:
        assert per_worker >= tiles and least <= widest <= most, (per_worker, widest)
    E = len(counts)
    hint = 65 * E if pairs else 1
    wq = ints(E, 2 * n if swiglu else n, k, seed=11)
    sw = scales(E, wq.size(1), seed=12, size=0.02 / k)
    cnt = torch.tensor(counts, dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    # One expert's rows after the other's.
    first = (torch.cumsum(cnt, 0) - cnt).to(torch.int32)
    total = sum(counts)
    xq, sx = ints(total + 5, k, seed=13), scales(total + 5, seed=14)
    out = torch.full((total + 5, n), float("nan"), dtype=torch.bfloat16, device=DEV)
    grouped_gemm_int8(xq, sx, wq, sw, cnt, first, swiglu, out, status=status, expected_rows=hint)
    check(out, xq, sx, wq, sw, cnt, first, swiglu, torch.bfloat16)
    assert out[total:].isnan().all()
    # The same rows in planes: the same bits.
    rows = max(counts) + 1
    planes, plane_scales = ints(E, rows, k, seed=15), scales(E, rows, seed=16)
    got = torch.full((E, rows, n), float("nan"), dtype=torch.bfloat16, device=DEV)
    for e, m in enumerate(counts):
        mine = slice(int(first[e]), int(first[e]) + m)
        planes[e, :m], plane_scales[e, :m] = xq[mine], sx[mine]
    for _ in range(3):
        grouped_gemm_int8(planes, plane_scales, wq, sw, cnt, None, swiglu, got, status=status,
                          expected_rows=hint)
    for e, m in enumerate(counts):
        assert torch.equal(got[e, :m], out[int(first[e]) : int(first[e]) + m])
        assert got[e, m:].isnan().all()
    assert int(status) == 0
