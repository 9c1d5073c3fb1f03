"""Eviction by mass on the GPU against its plain form (bounded_ref.py), and a serving loop that runs the operators for bounded
caches together, eagerly and from a graph."""
import numpy as np
import pytest

import bounded_ref as bref
import longctx_ref as ref
import paged_attention as pa
from helpers import empty_gpu, to_gpu, to_np
from test_gpu_window import close, close_mass, gpu_pool, run_mass, run_prefill

pytestmark = pytest.mark.gpu

I32 = np.int32


def run_evict(nb, tables, lens, mass, sink, recent, budget, refs, count=True):
    import torch
    cfg = pa.make_config(num_q_heads=2, num_kv_heads=2, head_dim=64, kv_dtype=1, num_blocks=nb)
    t, l, r = to_gpu(tables), to_gpu(lens), to_gpu(refs)
    m = None if mass is None else to_gpu(mass)
    gone = empty_gpu((len(lens) + 1,), I32)
    gone.fill_(-7)
    pa.evict_blocks(None, cfg, t, l, m, len(lens), tables.shape[1], sink, recent, budget, r, gone if count else None)
    torch.cuda.synchronize()
    gone = to_np(gone)
    assert gone[len(lens)] == -7
    return to_np(t), to_np(l), None if m is None else to_np(m), to_np(r), gone[:len(lens)]


def same(got, want, count=True):
    for a, b in zip(got[:4 + count], want):
        if b is not None:
            np.testing.assert_array_equal(a, b)


def books(rng, lens, width, shared=True):
    need = [min(width, (max(0, t) + 15) // 16) for t in lens]
    nb = sum(need) + 5
    ids = rng.permutation(nb).astype(I32)
    tables, at = np.full((len(lens), width), -1, I32), 0
    for i, n in enumerate(need):
        tables[i, :n] = ids[at:at + n]
        at += n
        if shared and i % 3 == 1:
            half = min(n, need[i - 1]) // 2
            tables[i, :half] = tables[i - 1, :half]
    return nb, tables, np.bincount(tables[tables >= 0], minlength=nb).astype(I32)


LENS = [1, 16, 500, 497, 0, 2000, 1999, -5, 16 * 40, 16 * 41, 16 * 40 + 1, 3333]


@pytest.mark.parametrize("masses", ["random", "ties", "zeros", "equal digits", "null"])
@pytest.mark.parametrize("sink,recent,budget", [(0, 1, 1), (1, 1, 2), (1, 2, 40), (3, 8, 41), (0, 40, 40), (20, 20, 40), (1, 4, 1000)])
def test_evict(masses, sink, recent, budget):
    rng = np.random.default_rng(500 + budget)
    for width in (209, 300):
        nb, tables, refs = books(rng, LENS, width)
        m = rng.exponential(2.0, tables.shape).astype(np.float32)
        if masses == "ties":
            m = rng.integers(0, 4, tables.shape).astype(np.float32)
        elif masses == "zeros":
            m[rng.random(m.shape) < 0.7] = 0
            m[rng.random(m.shape) < 0.3] = -0.0
        elif masses == "equal digits":  # apart in their lowest bits alone
            m = (np.float32(1.5).view(np.uint32) + rng.integers(0, 9, tables.shape)).astype(np.uint32).view(np.float32)
        elif masses == "null":
            m = None
        lens = np.array(LENS, I32)
        want = bref.evict(tables, lens, m, sink, recent, budget, refs)
        same(run_evict(nb, tables, lens, m, sink, recent, budget, refs), want)
        same(run_evict(nb, tables, lens, m, sink, recent, budget, refs, count=False), want, count=False)
        assert (want[4] > 0).any() or budget == 1000


def test_evict_masses_of_every_kind():
    """Infinities, NaN of both signs, negative values, denormals, the largest."""
    rng = np.random.default_rng(510)
    nb, tables, refs = books(rng, [16 * 200] * 4, 200)
    kinds = np.array([np.inf, -np.inf, np.nan, -1.0, 1e-42, -1e-42, 3.4e38, -3.4e38, 0.0, -0.0, 1.0], np.float32)
    m = rng.choice(kinds, tables.shape)
    m.view(np.uint32)[2, 50:60] = 0xffc00000
    lens = np.full(4, 16 * 200, I32)
    for budget in (10, 60, 120, 199):
        same(run_evict(nb, tables, lens, m, 2, 3, budget, refs), bref.evict(tables, lens, m, 2, 3, budget, refs))


@pytest.mark.parametrize("blocks", [1024, 1025, 8192, 16384, 40000, 140000])
@pytest.mark.parametrize("with_mass", [True, False])
def test_evict_long_rows(blocks, with_mass):
    rng = np.random.default_rng(520)
    lens = [16 * blocks - 3, 16 * blocks // 2, 100]
    nb, tables, refs = books(rng, lens, blocks + 3, shared=False)
    m = rng.exponential(2.0, tables.shape).astype(np.float32) if with_mass else None
    lens = np.array(lens, I32)
    for budget in (16, blocks // 3, blocks - 1):
        same(run_evict(nb, tables, lens, m, 1, 5, budget, refs), bref.evict(tables, lens, m, 1, 5, budget, refs))


def test_evict_entries_that_are_none_and_reserved_ahead():
    rng = np.random.default_rng(530)
    lens = np.array([16 * 50, 16 * 50 - 7, 9999999], I32)
    nb, tables, refs = books(rng, [16 * 60] * 3, 64, shared=False)  # ten blocks behind the length, or none
    tables[0, [5, 6, 20]] = -1, nb, 2 ** 31 - 1
    m = rng.exponential(2.0, tables.shape).astype(np.float32)
    m[0, [5, 6, 20]] = 0
    for budget in (3, 20, 49):
        same(run_evict(nb, tables, lens, m, 1, 1, budget, refs), bref.evict(tables, lens, m, 1, 1, budget, refs))


def test_evict_without_rows_or_width():
    cfg = pa.make_config(num_q_heads=2, num_kv_heads=2, head_dim=64, kv_dtype=1, num_blocks=4)
    refs = to_gpu(np.ones(4, I32))
    pa.evict_blocks(None, cfg, refs, refs, None, 0, 5, 0, 1, 1, refs)
    pa.evict_blocks(None, cfg, refs, refs, None, 3, 0, 0, 1, 1, refs)
    assert to_np(refs).tolist() == [1] * 4


class Serving:
    """Rows of a bounded cache on the device, and the same in plain form: prompts, then steps of one token each, with eviction."""

    def __init__(self, kv, q, window, sink, budget):
        self.lens0 = [150, 33, 260, 90]
        self.kv, self.q, self.window, self.sink, self.budget = kv, q, window, sink, budget
        p = self.p = ref.Pool(540 + kv, self.lens0, 8, 2, 64, kv, q, extra=0, width=40)
        more = 60  # free blocks
        p.nb += more
        p.cfg.num_blocks = p.nb
        for name in ("k", "v"):
            a = getattr(p, name)
            setattr(p, name, np.concatenate([a, np.zeros((more,) + a.shape[1:], a.dtype)]))
        if p.stats:
            p.stats = [np.concatenate([s, np.zeros((more, p.hkv), np.float32)]) for s in p.stats]
        self.refs = np.bincount(p.tables[p.tables >= 0], minlength=p.nb).astype(I32)
        self.lens = np.array(self.lens0, I32)
        self.mass = np.zeros(p.tables.shape, np.float32)


@pytest.mark.parametrize("kv,q,window,sink,budget", [(1, 1, 0, 0, 8), (2, 0, 0, 3, 6), (0, 0, 0, 0, 5), (1, 1, 64, 16, 6)])
@pytest.mark.parametrize("graph", [False, True])
def test_serving_from_a_bounded_cache(kv, q, window, sink, budget, graph):
    """Prompts are attended to and weighed, evicted to their budget, and decoded token by token: room reserved, the token
    appended, attention with its masses, eviction. Every device result is checked against the plain forms of the same
    step on the device's own cache; from a graph the steps are replayed with work of the program's own between them."""
    import torch
    S = Serving(kv, q, window, sink, budget)
    p = S.p
    B, width = len(S.lens0), p.width
    with_mass = window == 0  # a sliding window needs none: what lies between sinks and window goes
    g = gpu_pool(p)
    rows, at = bref.chunk_rows(S.lens0, S.lens0)
    qs = p.queries(len(rows))
    out, lse = run_prefill(p, g, qs, S.lens0, S.lens0, sink, window)
    want = bref.attend(p, qs, rows, at, sink, window, [S.lens0[s] for s in rows])
    close(out, want[0], want[1])
    close(lse, want[2], want[3])
    mass = S.mass
    if with_mass:
        added, tol = bref.prompt_mass(p, qs, lse, S.lens0, S.lens0, 16, sink, window)
        mass = run_mass(p, g, qs, lse, S.lens0, S.lens0, 16, sink, window, S.mass)
        close_mass(mass, S.mass, added, tol)

    dev = pa.Device(0)
    ts = pa.Stream(dev)
    tstream = torch.cuda.ExternalStream(ts.native(), device="cuda:0")
    tables, lens, refs, gm = g["tables"], to_gpu(S.lens), to_gpu(S.refs), to_gpu(mass)
    one, off = to_gpu(np.ones(B, I32)), to_gpu(np.arange(B, dtype=I32))
    pairs, status, slots, gone = empty_gpu((B, 2), I32), empty_gpu((2,), I32), empty_gpu((B,), np.int64), empty_gpu((B,), I32)
    act = np.float32 if q == 0 else np.uint16
    kn, vn, dq = (empty_gpu((B, h, p.d), act) for h in (p.hkv, p.hkv, p.hq))
    dout = empty_gpu((B, p.hq, p.d), np.float32)
    most = width * 16
    ws_b, rs_b = pa.window_decode_workspace_size(p.cfg, B, most, sink, window, with_mass), pa.pages_workspace_size(p.cfg, B, width)
    ws, rs = empty_gpu((ws_b,), np.uint8), empty_gpu((max(rs_b, 16),), np.uint8)
    sink_blocks, recent = (sink + 15) // 16, (window + 14) // 16 + 1 if window else 2

    def evict():
        pa.evict_blocks(ts, p.cfg, tables, lens, gm if with_mass else None, B, width, sink_blocks, recent, budget, refs, gone)

    def step():
        pa.pages_reserve(ts, p.cfg, tables, lens, one, B, width, 1, refs, pairs, status, rs, rs_b)
        pa.build_slot_mapping(ts, p.cfg, tables, width, lens, one, off, B, 1, slots)
        pa.kv_append(ts, p.cfg, kn, vn, slots, B, g["k"], g["v"], *g["stats"])
        with torch.cuda.stream(tstream):
            lens.add_(one)
        pa.window_decode(ts, p.cfg, dout, dq, g["k"], g["v"], g["stats"][0], g["stats"][1], tables, lens, B, width, most, sink,
                         window, gm if with_mass else None, ws, ws_b)
        evict()

    torch.cuda.synchronize()
    with torch.cuda.stream(tstream):  # (loaded before a capture)
        lens.add_(one).sub_(one)
    evict()
    ts.synchronize()
    state = bref.evict(p.tables, S.lens, mass if with_mass else None, sink_blocks, recent, budget, S.refs)

    def check_books():
        np.testing.assert_array_equal(to_np(tables), state[0])
        np.testing.assert_array_equal(to_np(lens), state[1])
        np.testing.assert_array_equal(to_np(refs), state[3])
        np.testing.assert_array_equal(to_np(gone), state[4])
        if with_mass:
            np.testing.assert_array_equal(to_np(gm), state[2])

    check_books()
    assert (state[4] > 0).any()
    gr = None
    if graph:
        gr = pa.Graph().capture(ts)
        step()
        gr.end()
    rng, left = np.random.default_rng(7), 0
    for n in range(40):
        new = [ref.of_type(rng.standard_normal((B, h, p.d), np.float32), q) for h in (p.hkv, p.hkv, p.hq)]
        for a, b in zip((kn, vn, dq), new):
            a.copy_(to_gpu(b))
        before = to_np(gm).copy()
        torch.cuda.synchronize()
        if gr:
            gr.launch(ts)
        else:
            step()
        ts.synchronize()
        junk = torch.randn(1 << 18, device="cuda:0").sum()  # the program's own work between replays
        torch.cuda.synchronize()
        del junk
        assert to_np(status)[1] == 0
        t2, r2, _, _ = ref.reserve(state[0], state[1], np.ones(B, I32), state[3])
        l2 = state[1] + 1
        # the cache as the device holds it: the append is another operator's
        p.tables, p.k, p.v = t2, to_np(g["k"], ref.NP_DTYPE[kv]), to_np(g["v"], ref.NP_DTYPE[kv])
        if p.stats:
            p.stats = [to_np(s) for s in g["stats"]]
        want, tol, _, _, added, mass_tol = bref.decode(p, new[2], l2, sink, window)
        close(to_np(dout), want, tol, f"step {n}")
        m2 = None
        if with_mass:  # the device's masses before this step's eviction: what stayed is told by the tables, the rest by the sums
            m2 = before + added
            got_t, got_m = to_np(tables), to_np(gm)
            for i in range(B):
                kept = [list(t2[i]).index(b) for b in got_t[i] if b >= 0]
                close(got_m[i, :len(kept)], m2[i, kept], mass_tol[i, kept] + 2 * bref.EPS * m2[i, kept])
                m2[i, kept] = got_m[i, :len(kept)]
                gap = np.setdiff1d(np.nonzero(t2[i] >= 0)[0], kept)
                if len(gap):  # what left was lighter than all that could have stayed, up to the masses' tolerance
                    may = [b for b in kept if sink_blocks <= b < (l2[i] + 15) // 16 - recent]
                    assert all(m2[i, x] <= m2[i, b] + 2 * mass_tol[i].max() for x in gap for b in may)
                    m2[i, gap] = -1.0  # so the plain form picks them
        state = bref.evict(t2, l2, m2, sink_blocks, recent, budget, r2)
        if with_mass:
            state = (state[0], state[1], state[2].astype(np.float32), *state[3:])
        check_books()
        left += state[4].sum()
    assert left > 0
    if gr:
        gr.destroy()
    ts.destroy()
    dev.close()


def test_evict_the_same_block_twice():
    """A block that stands twice in a row, and in another row: a count for every entry that leaves."""
    tables = np.array([[3, 3, 4, 3, 5, -1], [3, 6, 6, 7, -1, -1]], I32)
    lens, mass = np.array([70, 64], I32), np.array([[1, 2, 0, 3, 4, 9], [0, 0, 5, 1, 9, 9]], np.float32)
    refs = np.bincount(tables[tables >= 0], minlength=9).astype(I32)
    for m in (mass, None):
        got = run_evict(9, tables, lens, m, 0, 1, 2, refs)
        same(got, bref.evict(tables, lens, m, 0, 1, 2, refs))
        np.testing.assert_array_equal(got[3], np.bincount(got[0][got[0] >= 0], minlength=9))
