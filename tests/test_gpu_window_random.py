"""Small random calls of the operators for bounded caches against the 64-bit forms of bounded_ref.py: types, heads, lengths, windows, sinks,
bounds, tables with entries that are none, what stands in unused slots. The same calls every time."""
import random

import numpy as np
import pytest

import bounded_ref as bref
import longctx_ref as ref
from test_gpu_evict import books, run_evict, same
from test_gpu_window import I32, INT8, TYPES, close, close_mass, gpu_pool, masses, run_decode, run_mass, run_prefill, spoil

# (the plain form multiplies what stands in the place of no block by 0)
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:invalid value")]

FAR = 2 ** 31 - 1


def a_pool(rnd, seed):
    """(pool, lengths)"""
    kv, q = rnd.choice(TYPES)
    d = rnd.choice([64, 128, 256] if kv == INT8 else [32, 64, 128, 256])
    hkv, group = rnd.choice([1, 1, 2, 3, 8]), rnd.choice([1, 2, 4, 8, 16])
    while hkv * group * d > 4096:
        hkv, group = 1, max(1, group // 2)
    n = rnd.choice([1, 2, 5, 17, 40])
    most = int(2 ** rnd.uniform(0, 10.5 if n < 10 else 7.5))
    lens = [rnd.randint(0, most) for _ in range(n)]
    lens[rnd.randrange(n)] = most
    p = ref.Pool(5000 + seed, lens, hkv * group, hkv, d, kv, q, width=(most + 15) // 16 + rnd.choice([0, 0, 1, 5]))
    p.cfg.scale = rnd.choice([0.0, 0.0, 0.3, 2.0 / d])
    if rnd.random() < 0.3:
        for _ in range(3):
            p.tables[rnd.randrange(n), rnd.randrange(p.width)] = rnd.choice([-1, p.nb, FAR, -FAR - 1])
    if kv != INT8 and rnd.random() < 0.4:
        for s, t in enumerate(lens):
            if t % 16 and 0 <= p.tables[s, t // 16] < p.nb:
                spoil(p, s, range(t, (t // 16 + 1) * 16), rnd.choice([np.nan, np.inf, -np.inf]))
    return p, lens


@pytest.mark.parametrize("first", range(0, 1000, 100))
def test_attention_and_masses(first):
    for seed in range(first, first + 100):
        rnd = random.Random(seed)
        p, lens = a_pool(rnd, seed)
        window = rnd.choice([0, 0, 1, rnd.randint(1, 60), rnd.randint(1, 2000), FAR])
        sink = rnd.choice([0, 0, 1, rnd.randint(1, 100), FAR])
        most = rnd.choice([max(lens), max(lens), rnd.randint(0, max(lens) + 40)])
        what = f"seed {seed}: types {p.kv} {p.q}, heads {p.hq} {p.hkv} {p.d}, {lens[:5]}, window {window}, sink {sink}, most {most}"
        g, qs, before = gpu_pool(p), p.queries(len(lens)), masses(p)
        out, tol, _, _, added, mass_tol = bref.decode(p, qs, lens, sink, window, most)
        got, mass = run_decode(p, g, qs, lens, sink, window, before, max_len=most)
        close(got, out, tol, what)
        close_mass(mass, before, added, mass_tol)
        chunks = [min(t, rnd.choice([0, 1, 2, 5, rnd.randint(0, 150)])) for t in lens]
        if sum(chunks) == 0 or sum(chunks) * p.hq > 6000:
            continue
        bound = rnd.choice([max(chunks), max(chunks) + rnd.randint(0, 5), 5000])
        rows, at = bref.chunk_rows(lens, chunks)
        qs = p.queries(len(rows))
        want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, sink, window, [lens[s] for s in rows], most)
        got, glse = run_prefill(p, g, qs, lens, chunks, sink, window, max_len=most, max_chunk=bound)
        seen = np.isfinite(lse)
        close(got, want, tol, f"{what}, chunks {chunks[:5]}, bound {bound}")
        close(glse[seen], lse[seen], lse_tol[seen], what)
        assert (glse[~seen] == -np.inf).all() and (got[~seen] == 0).all(), what
        last = rnd.choice([1, 3, 64, 200])
        added, mass_tol = bref.prompt_mass(p, qs, glse, lens, chunks, last, sink, window, most)
        close_mass(run_mass(p, g, qs, glse, lens, chunks, last, sink, window, before, most), before, added, mass_tol)


@pytest.mark.parametrize("first", range(0, 400, 100))
def test_eviction(first):
    for seed in range(first, first + 100):
        rnd, rng = random.Random(seed), np.random.default_rng(seed)
        width = int(2 ** rnd.uniform(0, 13.5))
        rows = rnd.choice([1, 2, 5, 9]) if width > 1000 else rnd.choice([1, 3, 20])
        budget = rnd.randint(1, width + 2)
        recent = rnd.randint(1, min(budget, rnd.choice([20, budget])))
        sink = rnd.randint(0, min(budget - recent, rnd.choice([5, budget])))
        lens = [rnd.choice([rnd.randint(-3, 16 * width + 40), 16 * width, 16 * min(width, budget), 16 * min(width, budget) + 1]) for _ in range(rows)]
        nb, tables, refs = books(rng, lens, width)
        for _ in range(rnd.choice([0, 0, 3])):
            tables[rnd.randrange(rows), rnd.randrange(width)] = rnd.choice([-1, nb, FAR, -7])
        kind = rnd.choice(["random", "ties", "zeros", "odd", "none"])
        m = None if kind == "none" else rng.exponential(2.0, tables.shape).astype(np.float32)
        if kind == "ties":
            m = rng.integers(0, 3, tables.shape).astype(np.float32)
        elif kind == "zeros":
            m[:] = 0
        elif kind == "odd":
            m = rng.choice(np.array([np.inf, -np.inf, np.nan, -1, 0, -0.0, 1e-42, 3e38, 1], np.float32), tables.shape)
        lens = np.array(lens, I32)
        same(run_evict(nb, tables, lens, m, sink, recent, budget, refs), bref.evict(tables, lens, m, sink, recent, budget, refs))


@pytest.mark.parametrize("first", range(0, 300, 100))
def test_values_that_are_not_finite(first):
    """They reach the queries that see their tokens, in their channels, and nothing else."""
    for seed in range(first, first + 100):
        rnd = random.Random(10 ** 6 + seed)
        p, lens = a_pool(rnd, seed)
        if p.kv == INT8 or sum(lens) == 0:
            continue
        p.tables[:] = -1
        at = 0
        for s, t in enumerate(lens):  # every block in one place (the pool may have renamed some)
            p.tables[s, :(t + 15) // 16] = np.arange(at, at + (t + 15) // 16)
            at += (t + 15) // 16
        p.k[:], p.v[:] = (ref.of_type(p.rng.standard_normal(x.shape, np.float32), p.kv) for x in (p.k, p.v))
        window, sink = rnd.choice([0, 0, rnd.randint(1, 60), rnd.randint(1, 1000)]), rnd.choice([0, 1, rnd.randint(1, 100)])
        chunks = [min(t, rnd.choice([0, 1, 5, rnd.randint(0, 150)])) for t in lens]
        if sum(chunks) == 0 or sum(chunks) * p.hq > 6000:
            continue
        rows, at = bref.chunk_rows(lens, chunks)
        qs, one = p.queries(len(rows)), p.queries(len(lens))
        want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, sink, window, [lens[s] for s in rows])
        dwant, dtol, _, _, _, _ = bref.decode(p, one, lens, sink, window)
        touched, dtouched = np.zeros(want.shape, bool), np.zeros(dwant.shape, bool)
        for _ in range(rnd.choice([1, 3, 30])):
            s = rnd.choice([s for s, t in enumerate(lens) if t])
            t, h, c = rnd.randrange(max(0, lens[s] - 2 * chunks[s] - 40), lens[s]), rnd.randrange(p.hkv), rnd.randrange(p.d)
            p.v[p.tables[s, t // 16], h, c, t % 16] = ref.of_type(np.full(1, rnd.choice([np.nan, np.inf, -np.inf]), np.float32), p.kv)[0]
            heads = slice(h * (p.hq // p.hkv), (h + 1) * (p.hq // p.hkv))
            for r, (x, pos) in enumerate(zip(rows, at)):
                if x == s and bref.seen(pos, t, sink, window):
                    touched[r, heads, c] = True
            if bref.seen(lens[s] - 1, t, sink, window):
                dtouched[s, heads, c] = True
        g = gpu_pool(p)
        got, glse = run_prefill(p, g, qs, lens, chunks, sink, window, max_chunk=rnd.choice([max(chunks), 5000]))
        what = f"seed {seed}: types {p.kv} {p.q}, heads {p.hq} {p.hkv} {p.d}, {lens[:5]}, {chunks[:5]}, window {window}, sink {sink}"
        seen = np.isfinite(lse)
        close(glse[seen], lse[seen], lse_tol[seen], what)
        for x, w, t, hit in ((got, want, tol, touched), (run_decode(p, g, one, lens, sink, window)[0], dwant, dtol, dtouched)):
            assert not np.isfinite(x[hit]).any(), what
            close(x[~hit], w[~hit], np.broadcast_to(t, w.shape)[~hit], what)
