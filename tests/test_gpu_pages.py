"""The page books on the GPU (fork, reserve, compact) and the copies they ask for, against their forms that work one row
and one block at a time (longctx_ref.py): whole numbers and bytes, equal bit for bit."""
import numpy as np
import pytest

import longctx_ref as ref
import paged_attention as pa
from helpers import empty_gpu, to_gpu, to_np

pytestmark = pytest.mark.gpu


def config(nb, kv=1, hkv=2, d=64):
    return pa.make_config(num_q_heads=hkv, num_kv_heads=hkv, head_dim=d, kv_dtype=kv, num_blocks=nb)


def books(seed, lens, nb, width=None, share=0.0):
    """Tables, lengths and refcounts; row i starts with blocks of row i - 1 with probability `share`."""
    rng = np.random.default_rng(seed)
    width = width or max([(t + 15) // 16 for t in lens] + [1]) + 2
    ids = list(rng.permutation(nb))
    tables = np.full((len(lens), width), -1, np.int32)
    for i, t in enumerate(lens):
        n = (t + 15) // 16
        common = 0
        if i and rng.random() < share:
            common = int(rng.integers(0, min(n, (lens[i - 1] + 15) // 16) + 1))
            tables[i, :common] = tables[i - 1, :common]
        for j in range(common, n):
            tables[i, j] = ids.pop()
    refs = np.zeros(nb, np.int32)
    np.add.at(refs, tables[tables >= 0], 1)
    return tables, np.array(lens, np.int32), refs


def run_fork(cfg, tables, lens, src, refs):
    import torch
    n, w = len(src), tables.shape[1]
    out, out_lens, r = empty_gpu((max(n, 1), w), np.int32), empty_gpu((max(n, 1),), np.int32), to_gpu(refs)
    out.fill_(99)
    pa.pages_fork(None, cfg, to_gpu(tables), to_gpu(lens), len(tables), to_gpu(np.array(src, np.int32)), out, out_lens, n, w, r)
    torch.cuda.synchronize()
    return to_np(out)[:n], to_np(out_lens)[:n], to_np(r)


def run_reserve(cfg, tables, lens, num_new, refs, most=None):
    import torch
    t, r, pairs, st = to_gpu(tables), to_gpu(refs), empty_gpu((len(lens), 2), np.int32), empty_gpu((2,), np.int32)
    size = pa.pages_workspace_size(cfg, len(lens), tables.shape[1])
    ws = empty_gpu((size,), np.uint8)
    ws.fill_(0x5A)
    pairs.fill_(77)
    pa.pages_reserve(None, cfg, t, to_gpu(np.array(lens, np.int32)), to_gpu(np.array(num_new, np.int32)), len(lens),
                     tables.shape[1], max(num_new) if most is None else most, r, pairs, st, ws, size)
    torch.cuda.synchronize()
    return to_np(t), to_np(r), to_np(pairs), to_np(st)


def run_compact(cfg, tables, refs, moves):
    import torch
    t, r, pairs, st = to_gpu(tables), to_gpu(refs), empty_gpu((max(moves, 1), 2), np.int32), empty_gpu((2,), np.int32)
    size = pa.pages_workspace_size(cfg, len(tables), tables.shape[1])
    ws = empty_gpu((size,), np.uint8)
    ws.fill_(0x5A)
    pairs.fill_(77)
    pa.pages_compact(None, cfg, t, len(tables), tables.shape[1], r, moves, pairs, st, ws, size)
    torch.cuda.synchronize()
    return to_np(t), to_np(r), to_np(pairs)[:moves], to_np(st)


def same(got, want, what=""):
    for i, (a, b) in enumerate(zip(got, want)):
        np.testing.assert_array_equal(a, b, err_msg=f"{what}: result {i}")


@pytest.mark.parametrize("rows,src", [
    (1, [0]), (1, [0] * 9), (1, []), (1, [-1]), (4, [3, 2, 1, 0]), (4, [1, 1, -1, 3, 1, 7, -2 ** 31, 2 ** 31 - 1]), (4, [-1] * 4),
    (70, list(range(0, 70, 3)) * 2), (300, [(7 * i) % 300 if i % 5 else -1 for i in range(777)]),
])
def test_fork(rows, src):
    lens = [(37 * i) % 400 for i in range(rows)]
    tables, lens, refs = books(1, lens, 30 * rows + 5, share=0.4)
    same(run_fork(config(len(refs)), tables, lens, src, refs), ref.fork(tables, lens, src, refs), f"{rows} rows")


def test_fork_from_no_rows_and_counts_of_other_owners():
    tables, lens, refs = books(2, [100, 50], 20)
    refs[tables[0, 0]] += 3  # a prefix cache holds it too
    same(run_fork(config(20), tables, lens, [1, 1, -1], refs), ref.fork(tables, lens, [1, 1, -1], refs))
    import torch
    out, n, r = empty_gpu((2, 5), np.int32), empty_gpu((2,), np.int32), to_gpu(refs)
    pa.pages_fork(None, config(20), None, None, 0, to_gpu(np.zeros(2, np.int32)), out, n, 2, 5, r)
    torch.cuda.synchronize()
    assert (to_np(out) == -1).all() and (to_np(n) == 0).all() and (to_np(r) == refs).all()


@pytest.mark.parametrize("num_new", [0, 1, 15, 16, 17, 40])
def test_reserve_new_blocks(num_new):
    lens = [0, 1, 15, 16, 17, 31, 32, 100, 5, -3]
    tables, _, refs = books(3, [max(t, 0) for t in lens], 100, width=9)
    new = [num_new] * 8 + [0, num_new]
    same(run_reserve(config(100), tables, lens, new, refs, most=num_new), ref.reserve(tables, lens, new, refs))


def test_reserve_stops_at_the_table_and_at_the_bound():
    tables, lens, refs = books(4, [30, 33], 40, width=3)
    same(run_reserve(config(40), tables, lens, [1000, 2 ** 31 - 1], refs), ref.reserve(tables, lens, [1000, 1000], refs))
    tables, lens, refs = books(4, [30, 33], 40, width=30)
    # a bound of 18 tokens: three blocks a row at most
    same(run_reserve(config(40), tables, lens, [400, 400], refs, most=18), ref.reserve(tables, lens, [16 * 4 - 30, 16 * 5 - 33], refs))


@pytest.mark.parametrize("src,new", [
    ([0, 0, 0], [1, 1, 1]),          # all who hold the block ask: the last keeps it
    ([0, 0, 0], [1, 0, 1]),          # one does not: both others copy
    ([0, 1, 1, 1, 0, 2], [1, 20, 3, 1, 1, 1]),
    ([2, 2, 2, 2], [16, 1, 40, 1]),  # full last block: no copy, blocks of their own
])
def test_reserve_copies_on_write(src, new):
    tables, lens, refs = books(5, [100, 37, 64], 60, width=12)
    tables, lens, refs = ref.fork(tables, lens, src, refs)
    got = run_reserve(config(60), tables, lens, new, refs)
    same(got, ref.reserve(tables, lens, new, refs))


def test_reserve_counts_other_owners_and_reserved_blocks():
    tables, lens, refs = books(6, [40, 20], 30, width=8)
    refs[tables[0, 2]] += 1  # held by somebody outside the tables: copied even if the only row asks
    same(run_reserve(config(30), tables, lens, [1, 1], refs), ref.reserve(tables, lens, [1, 1], refs))
    # blocks reserved ahead, then forked: each row gets its own
    t, r, _, _ = ref.reserve(tables, lens, [50, 50], refs)
    t, n, r = ref.fork(t, lens, [0, 0, 1, 1], r)
    same(run_reserve(config(30), t, n, [30, 50, 1, 2], r), ref.reserve(t, n, [30, 50, 1, 2], r))


@pytest.mark.parametrize("free", [0, 1, 2, 3, 4])
def test_reserve_is_all_or_nothing(free):
    tables, lens, refs = books(7, [16, 40, 40], 9, width=6)
    tables, lens, refs = ref.fork(tables, lens, [0, 1, 1, 2], refs)  # needs 1 + 1 + 0 + 0
    refs[np.nonzero(refs == 0)[0][free:]] = 1
    new = [17, 1, 1, 1]  # two blocks for the first row, one copy
    got = run_reserve(config(9), tables, lens, new, refs)
    same(got, ref.reserve(tables, lens, new, refs))
    assert (got[3] == ([3, 0] if free >= 3 and (refs == 0).sum() >= 3 else [0, 3 - (refs == 0).sum()])).all()


def test_reserve_large():
    """More demands than a workgroup has threads, a pool of many slabs, shared tails everywhere."""
    tables, lens, refs = books(8, [(61 * i) % 900 for i in range(260)], 20000, width=70, share=0.5)
    src = [(i * 3) % 260 for i in range(700)]
    tables, lens, refs = ref.fork(tables, lens, src, refs)
    new = [(i * 7) % 60 for i in range(700)]
    same(run_reserve(config(len(refs)), tables, lens, new, refs), ref.reserve(tables, lens, new, refs))


@pytest.mark.parametrize("rows", [200, 511, 1024])
def test_reserve_as_many_demands_as_threads(rows):
    """A demand for each thread, nearly all of them for shared blocks, in a pool whose free blocks lie behind its first
    thousands."""
    nb = 30000
    tables, lens, refs = books(10, [20 + i % 400 for i in range(60)], nb, width=30)
    src = [(i * 7) % 60 for i in range(rows)]
    tables, lens, refs = ref.fork(tables, lens, src, refs)
    refs[:nb - 1100][refs[:nb - 1100] == 0] = 1
    new = [1 if i % 9 else 0 for i in range(rows)]
    same(run_reserve(config(nb), tables, lens, new, refs), ref.reserve(tables, lens, new, refs))


def test_reserve_one_block_held_by_all():
    tables, lens, refs = books(11, [5], 1100, width=2)
    tables, lens, refs = ref.fork(tables, lens, [0] * 1024, refs)
    for new in ([1] * 1024, [1] * 1000 + [0] * 24):
        same(run_reserve(config(1100), tables, lens, new, refs), ref.reserve(tables, lens, new, refs))


@pytest.mark.parametrize("nb,live,moves", [(20000, 9000, 10 ** 5), (300001, 70000, 10 ** 6), (600000, 299000, 1000), (530000, 529000, 10 ** 6)])
def test_compact_large_pools(nb, live, moves):
    """Pools past one round of the counting, checked against the definition in whole arrays."""
    rng = np.random.default_rng(nb)
    refs = np.zeros(nb, np.int32)
    ids = rng.permutation(nb)[:live].astype(np.int32)
    refs[ids] = rng.integers(1, 4, live)
    tables = ids.reshape(-1, 100)
    moves = min(moves, nb)
    t, r, pairs, st = run_compact(config(nb), tables, refs, moves)
    up, down = np.nonzero(refs > 0)[0][::-1], np.nonzero(refs == 0)[0]
    k = min(len(up), len(down), moves)
    up, down = up[:k], down[:k]
    up, down = up[down < up], down[down < up]
    want = refs.copy()
    want[down], want[up] = refs[up], 0
    name = np.arange(nb, dtype=np.int32)
    name[up] = down
    np.testing.assert_array_equal(pairs[:len(up)], np.stack([up, down], 1))
    assert (pairs[len(up):] == -1).all()
    np.testing.assert_array_equal(r, want)
    np.testing.assert_array_equal(t, name[tables])
    assert st.tolist() == [len(up), np.nonzero(want > 0)[0][-1] + 1]


@pytest.mark.parametrize("moves", [0, 1, 7, 10 ** 4])
@pytest.mark.parametrize("rows,nb", [(1, 3), (6, 60), (40, 1024), (200, 3001)])
def test_compact(rows, nb, moves):
    lens = [(53 * i) % (16 * (nb // rows)) for i in range(rows)]
    tables, lens, refs = books(9, lens, nb, share=0.2)
    src = [i if i % 3 else -1 for i in range(rows)]
    tables, lens, refs = ref.fork(tables, lens, src, refs)
    moves = min(moves, nb)
    same(run_compact(config(nb), tables, refs, moves), ref.compact(tables, refs, moves))


def test_compact_full_empty_and_compact_pools():
    for refs in (np.zeros(50, np.int32), np.ones(50, np.int32), np.array([1] * 20 + [0] * 30, np.int32),
                 np.array([0] * 49 + [1], np.int32)):
        tables = np.full((2, 4), -1, np.int32)
        same(run_compact(config(50), tables, refs, 50), ref.compact(tables, refs, 50))


@pytest.mark.parametrize("kv,hkv,d", [(0, 2, 32), (0, 3, 64), (1, 8, 128), (1, 1, 64), (2, 8, 128), (2, 2, 256)])
@pytest.mark.parametrize("count", [None, 0, 5, 100])
def test_copy_pages(kv, hkv, d, count):
    import torch
    p = ref.Pool(80, [16 * 60], hkv, hkv, d, kv)
    pairs = p.rng.permutation(p.nb)[:40].reshape(20, 2).astype(np.int32)
    pairs[3, 1], pairs[6, 0], pairs[9] = pairs[3, 0], -1, (pairs[9, 0], p.nb)
    n = len(pairs) if count is None else min(count, len(pairs))
    for bounds in (True, False):
        arrays = [p.k, p.v] + ([p.bounds] if bounds else []) + (p.stats or [])
        g = [to_gpu(a) for a in arrays]
        st = g[2 + bounds:] or [None] * 4
        num = None if count is None else to_gpu(np.array([count, -5], np.int32))
        pa.copy_pages(None, p.cfg, g[0], g[1], *st, g[2] if bounds else None, to_gpu(pairs), len(pairs), num)
        torch.cuda.synchronize()
        ok = [(a, b) for a, b in pairs[:n] if a != b and a >= 0 and b < p.nb]
        for a, t in zip(arrays, g):
            want = a.copy()
            for x, y in ok:
                want[y] = a[x]
            np.testing.assert_array_equal(to_np(t, a.dtype), want)


@pytest.mark.parametrize("kv", [1, 2])
def test_beam_search_steps_in_a_graph(kv):
    """Steps of a beam search with the books on the device: beams reordered, blocks reserved, shared ones copied, the new tokens
    appended and attended, captured once and replayed. Every beam's attention is that over its own tokens, kept
    apart on the host; no block leaks; and a compaction moves all of it without changing a result."""
    import torch
    B, hq, hkv, d, steps, nb, width = 6, 4, 2, 64, 22, 90, 12
    rng = np.random.default_rng(90 + kv)
    cfg = pa.make_config(num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=kv, q_dtype=0, num_blocks=nb)
    dt = ref.NP_DTYPE[kv]
    k, v, bounds = empty_gpu((nb, hkv, 16, d), dt), empty_gpu((nb, hkv, d, 16), dt), empty_gpu((nb, hkv, 2, d), dt)
    stats = [empty_gpu((nb, hkv), np.float32) for _ in range(4)] if kv == 2 else [None] * 4
    tables = [empty_gpu((B, width), np.int32), empty_gpu((B, width), np.int32)]
    lens = [empty_gpu((B,), np.int32), empty_gpu((B,), np.int32)]
    tables[0].fill_(-1)
    refs, src, one = empty_gpu((nb,), np.int32), empty_gpu((B,), np.int32), to_gpu(np.ones(B, np.int32))
    pairs, status = empty_gpu((B, 2), np.int32), empty_gpu((2,), np.int32)
    size = pa.pages_workspace_size(cfg, B, width)
    ws, off, slots = empty_gpu((size,), np.uint8), to_gpu(np.arange(B, dtype=np.int32)), empty_gpu((B,), np.int64)
    q, kn, vn, out = (empty_gpu((B, h, d), np.float32) for h in (hq, hkv, hkv, hq))
    sel = to_gpu(np.tile(np.arange(width, dtype=np.int32), (B, hkv, 1)))
    n2 = pa.sparse_workspace_size(cfg, B, width)
    ws2, len1 = empty_gpu((max(8, n2),), np.uint8), empty_gpu((B,), np.int32)
    dev = pa.Device(0)
    ts = pa.Stream(dev)
    tstream = torch.cuda.ExternalStream(ts.native(), device="cuda:0")

    def step(a, b):
        pa.pages_fork(ts, cfg, tables[a], lens[a], B, src, tables[b], lens[b], B, width, refs)
        pa.pages_reserve(ts, cfg, tables[b], lens[b], one, B, width, 1, refs, pairs, status, ws, size)
        pa.copy_pages(ts, cfg, k, v, *stats, bounds, pairs, B)
        pa.build_slot_mapping(ts, cfg, tables[b], width, lens[b], one, off, B, 1, slots)
        pa.kv_append(ts, cfg, kn, vn, slots, B, k, v, *stats)
        pa.key_bounds_update(ts, cfg, k, tables[b], width, lens[b], one, B, 1, bounds)
        with torch.cuda.stream(tstream):
            lens[b].add_(1)
        pa.sparse_decode(ts, cfg, out, q, k, v, stats[0], stats[1], tables[b], B, width, None, lens[b], B, 16 * width, sel, width,
                         ws2, n2)

    torch.cuda.synchronize()
    graphs = []
    for a, b in ((0, 1), (1, 0)):
        gr = pa.Graph().capture(ts)
        step(a, b)
        graphs.append(gr.end())
    torch.cuda.synchronize()
    host = [[] for _ in range(B)]  # (k, v) of every token of a beam
    for n in range(steps):
        parents = rng.integers(0, B, B)
        if n == steps - 2:
            parents[1] = parents[4] = -1  # finished: an empty beam starts anew
        x = [rng.standard_normal(s, np.float32) for s in ((B, hq, d), (B, hkv, d), (B, hkv, d))]
        for t, a in zip((q, kn, vn), x):
            t.copy_(to_gpu(a))
        src.copy_(to_gpu(parents.astype(np.int32)))
        torch.cuda.synchronize()
        graphs[n % 2].launch(ts)
        ts.synchronize()
        host = [list(host[s]) if s >= 0 else [] for s in parents]
        for i in range(B):
            host[i].append((x[1][i], x[2][i]))
        now = (n + 1) % 2
        t, r, ln = to_np(tables[now]), to_np(refs), to_np(lens[now])
        assert (ln == [len(h) for h in host]).all() and to_np(status)[1] == 0
        count = np.zeros(nb, np.int32)
        np.add.at(count, t[t >= 0], 1)
        np.testing.assert_array_equal(r, count)
        if n in (9, 16):  # a compaction in between
            cp, cs = empty_gpu((nb, 2), np.int32), empty_gpu((2,), np.int32)
            pa.pages_compact(ts, cfg, tables[now], B, width, refs, nb, cp, cs, ws, size)
            pa.copy_pages(ts, cfg, k, v, *stats, bounds, cp, nb, cs)
            ts.synchronize()
            assert to_np(cs)[1] == (to_np(refs) > 0).sum()
        got = to_np(out)
        for i in range(B):
            kk, vv = (np.stack([h[j] for h in host[i]]) for j in (0, 1))
            if kv == 1:
                kk, vv = (ref.f64(ref.bf16_of(a)) for a in (kk, vv))
            for h in range(hq):
                s = kk[:, h // 2] @ x[0][i, h].astype(np.float64) / np.sqrt(d)
                w = np.exp(s - s.max())
                want = w @ vv[:, h // 2] / w.sum()
                # int8: codes requantised as the block's largest value grows, half a step of 4 / 127 each time
                np.testing.assert_allclose(got[i, h], want, atol=1e-4 if kv == 1 else 0.3, rtol=0)
    for gr in graphs:
        gr.destroy()
    ts.destroy()
    dev.close()
