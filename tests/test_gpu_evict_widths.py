"""Eviction from tables of every width at which the host takes another form of the kernel, and one entry less or more: rows that fill their
table, rows over their budget by one block, rows at it and under it."""
import numpy as np
import pytest

import bounded_ref as bref
from test_gpu_evict import I32, books, run_evict, same

pytestmark = pytest.mark.gpu

WIDTHS = [1, 2, 63, 64, 1023, 1024, 1025, 4095, 4096, 4097, 8191, 8192, 8193, 16383, 16384, 16385, 40000]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("masses", ["random", "ties", "zeros", "null"])
def test_evict_at_full_width(width, masses):
    rng = np.random.default_rng(700 + width)
    full = 16 * width
    for budget in sorted({max(1, width // 3), max(1, width - 1)} | ({1, width} if width < 5000 else set())):
        sink, recent = min(1, budget - 1), min(max(1, budget // 4), 5)
        lens = [full, full - 15, 16 * budget + 1, 16 * budget, max(0, 16 * budget - 16), full // 2, 0]
        nb, tables, refs = books(rng, lens, width, shared=width > 2)
        m = rng.exponential(2.0, tables.shape).astype(np.float32)
        if masses == "ties":
            m = rng.integers(0, 3, tables.shape).astype(np.float32)
        elif masses == "zeros":  # rows that no attention has weighed yet
            m[:] = 0
        elif masses == "null":
            m = None
        lens = np.array(lens, I32)
        want = bref.evict(tables, lens, m, sink, recent, budget, refs)
        same(run_evict(nb, tables, lens, m, sink, recent, budget, refs), want)
        if budget < width:
            assert want[4][0] == width - budget


@pytest.mark.parametrize("width", [1024, 4096, 8192, 16384])
@pytest.mark.parametrize("with_mass", [True, False])
def test_evict_moves_the_last_entry_of_a_full_table(width, with_mass):
    """The last register of the last thread: its block stays as the newest, moves with blocks reserved behind it, or is the one that goes."""
    rng = np.random.default_rng(710)
    nb, tables, refs = books(rng, [16 * width] * 3, width, shared=False)
    m = rng.exponential(2.0, tables.shape).astype(np.float32) if with_mass else None
    lens = np.array([16 * width, 16 * (width - 1), 16 * (width - 200) - 3], I32)  # 0, 1, 200 blocks reserved ahead
    for budget in (width - 201, width // 2):
        want = bref.evict(tables, lens, m, 0, 1, budget, refs)
        got = run_evict(nb, tables, lens, m, 0, 1, budget, refs)
        same(got, want)
        for i in range(3):
            assert tables[i, -1] in got[0][i]
    if with_mass:  # all but the newest weigh the same, and the one before it nothing
        m[:] = 1
        m[:, -2] = 0
        lens[:] = 16 * width
        want = bref.evict(tables, lens, m, 0, 1, width - 1, refs)
        same(run_evict(nb, tables, lens, m, 0, 1, width - 1, refs), want)
        assert all(tables[i, -2] not in want[0][i] for i in range(3))
