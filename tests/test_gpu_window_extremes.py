"""The operators for bounded caches at the ends of what they take: contexts of 400000 tokens, tens of thousands of sequences, hundreds
of query heads; a captured call whose chunks, prefixes and tables change between replays. Against the 64-bit forms of
bounded_ref.py, a sample of rows where there are many."""
import numpy as np
import pytest

import bounded_ref as bref
import longctx_ref as ref
import paged_attention as pa
from helpers import empty_gpu, to_gpu, to_np
from test_gpu_window import BF16, FP32, I32, INT8, close, close_mass, gpu_pool, masses, run_decode, run_mass, run_prefill
from test_gpu_window_forms import check_decode, forked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,q,hq,hkv,d", [(BF16, BF16, 2, 1, 32), (INT8, FP32, 2, 1, 64), (FP32, FP32, 2, 1, 32)])
def test_hundreds_of_thousands_of_tokens(kv, q, hq, hkv, d):
    """One row in more parts than a wave has lanes; keys of a few queries cut over workgroups; masses of 25001 blocks."""
    t = 400003
    p = ref.Pool(1000 + kv, [t], hq, hkv, d, kv, q)
    for sink, window in ((0, 0), (5, 300000)):
        check_decode(p, [t], sink, window, [0])
    g, chunk = gpu_pool(p), 3
    for sink, window in ((0, 0), (7, 200001)):
        rows, at = bref.chunk_rows([t], [chunk])
        qs = p.queries(chunk)
        want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, sink, window, [t] * chunk)
        got, glse = run_prefill(p, g, qs, [t], [chunk], sink, window)
        close(got, want, tol)
        close(glse, lse, lse_tol)
        before = masses(p)
        added, mass_tol = bref.prompt_mass(p, qs, glse, [t], [chunk], 2, sink, window)
        close_mass(run_mass(p, g, qs, glse, [t], [chunk], 2, sink, window, before), before, added, mass_tol)


def test_as_many_sequences_as_a_call_takes():
    """65535 chunks of one and two tokens, their masses, and as many single tokens, over the blocks of one text."""
    n = 65535
    lens = [1 + 7 * i % 90 for i in range(n)]
    p = forked(1010, n, lens, 2, 1, 32, BF16, BF16)
    g, before = gpu_pool(p), masses(p)
    sample = [0, 1, 2, 4095, 4096, 30000, 65533, 65534]
    chunks = [min(t, 1 + i % 2) for i, t in enumerate(lens)]
    start = np.concatenate([[0], np.cumsum(chunks)])
    qs = p.queries(int(start[-1]))
    got, glse = run_prefill(p, g, qs, lens, chunks, 2, 40)
    mass = run_mass(p, g, qs, glse, lens, chunks, 5, 2, 40, before)
    assert np.isfinite(got).all() and np.isfinite(glse).all()
    for s in sample:
        r = range(start[s], start[s + 1])
        at = [lens[s] - len(r) + i for i in range(len(r))]
        want, tol, lse, lse_tol, added, mass_tol = bref.attend(p, qs[r], [s] * len(r), at, 2, 40, [lens[s]] * len(r))
        close(got[r], want, tol, f"sequence {s}")
        close(glse[r], lse, lse_tol, f"sequence {s}")
        close_mass(mass[s], before[s], added[s], mass_tol[s])
    total = (mass.astype(np.float64) - before).sum(1)
    # (a weight is off by what its logarithm is; at most 4 a row, by 2^-16 with any of this length, and the entries round)
    assert np.abs(total - 2 * np.array(chunks)).max() < 1e-3
    check_decode(p, lens, 2, 40, sample)


@pytest.mark.parametrize("kv,q,hq,hkv", [(BF16, BF16, 160, 20), (BF16, FP32, 130, 130), (FP32, FP32, 256, 64), (BF16, BF16, 512, 32)])
def test_hundreds_of_heads(kv, q, hq, hkv):
    """More query heads than the masses' launch holds at a time."""
    lens = [70, 1, 333, 16, 200]
    p = ref.Pool(1020 + kv, lens, hq, hkv, 32, kv, q)
    for sink, window in ((0, 0), (3, 100)):
        check_decode(p, lens, sink, window, range(5))
    chunks = [3, 1, 20, 16, 2]
    rows, at = bref.chunk_rows(lens, chunks)
    qs, g, before = p.queries(len(rows)), gpu_pool(p), masses(p)
    want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, 3, 100, [lens[s] for s in rows])
    got, glse = run_prefill(p, g, qs, lens, chunks, 3, 100)
    close(got, want, tol)
    close(glse, lse, lse_tol)
    added, mass_tol = bref.prompt_mass(p, qs, glse, lens, chunks, 9, 3, 100)
    close_mass(run_mass(p, g, qs, glse, lens, chunks, 9, 3, 100, before), before, added, mass_tol)


@pytest.mark.parametrize("kv,q", [(BF16, BF16), (INT8, FP32), (FP32, FP32)])
@pytest.mark.parametrize("bound", [40, 3000])
def test_a_captured_call_takes_what_its_arrays_hold_at_each_replay(kv, q, bound):
    """Chunks, prefixes, lengths, tables and masses change between replays of one graph; sizes on the host are bounds (bound of the chunks:
    waves that share columns, that own them)."""
    import torch
    hq, hkv, d, n, most, sink, window = 8, 2, 64, 3, 3000, 4, 900
    p = ref.Pool(1030 + kv, [most] * n, hq, hkv, d, kv, q)
    steps = [([3000, 50, 7], [40, 40, 7]), ([1, 2999, 0], [1, 2, 0]), ([0, 0, 0], [0, 0, 0]), ([700, 1600, 2222], [33, 16, 1]), ([3000, 3000, 3000], [40, 1, 40])]
    rows = 120
    g, tables0 = gpu_pool(p), p.tables.copy()
    tables, mass = to_gpu(tables0), to_gpu(np.zeros(tables0.shape, np.float32))
    start, prefix, lens = (to_gpu(np.zeros(k, I32)) for k in (n + 1, n, n))
    act = np.float32 if q == 0 else np.uint16
    cq, dq = empty_gpu((rows, hq, d), act), empty_gpu((n, hq, d), act)
    out, lse, one = empty_gpu((rows, hq, d), np.float32), empty_gpu((rows, hq), np.float32), empty_gpu((n, hq, d), np.float32)
    wp = pa.window_prefill_workspace_size(p.cfg, n, bound, most, sink, window)
    wd = pa.window_decode_workspace_size(p.cfg, n, most, sink, window, True)
    ws_p, ws_d = empty_gpu((max(wp, 16),), np.uint8), empty_gpu((wd,), np.uint8)

    def run(stream):
        st = pa.Stream(pa.Device(0), stream.cuda_stream)
        pa.window_prefill(st, p.cfg, out, cq, start, prefix, g["k"], g["v"], g["stats"][0], g["stats"][1], tables, n, p.width, bound, most,
                          sink, window, lse, ws_p, wp)
        pa.prefill_mass(st, p.cfg, cq, lse, start, prefix, g["k"], g["stats"][0], tables, n, p.width, most, 16, sink, window, mass)
        pa.window_decode(st, p.cfg, one, dq, g["k"], g["v"], g["stats"][0], g["stats"][1], tables, lens, n, p.width, most, sink, window,
                         mass, ws_d, wd)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(stream)
    rng = np.random.default_rng(1)
    for step, (ts, chunks) in enumerate(steps + steps[:2]):
        p.tables = rng.permutation(tables0.reshape(-1)).reshape(tables0.shape)
        before = masses(p)
        new = p.queries(sum(chunks)), p.queries(n)
        cq[:sum(chunks)].copy_(to_gpu(new[0]))
        dq.copy_(to_gpu(new[1]))
        for dst, src in ((tables, p.tables), (mass, before), (start, np.concatenate([[0], np.cumsum(chunks)]).astype(I32)),
                         (prefix, (np.array(ts) - np.array(chunks)).astype(I32)), (lens, np.array(ts, I32))):
            dst.copy_(to_gpu(src))
        out.fill_(12345.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        junk = torch.randn(1 << 16, device="cuda:0").sum()  # the program's own work between replays
        seqs, at = bref.chunk_rows(ts, chunks)
        k = sum(chunks)
        want, tol, wlse, lse_tol, _, _ = bref.attend(p, new[0], seqs, at, sink, window, [ts[s] for s in seqs])
        close(to_np(out)[:k], want, tol, f"step {step}")
        close(to_np(lse)[:k], wlse, lse_tol, f"step {step}")
        assert (to_np(out)[k:] == 12345.0).all()
        dwant, dtol, _, _, dadd, dmt = bref.decode(p, new[1], ts, sink, window)
        close(to_np(one), dwant, dtol, f"step {step}")
        added, mt = bref.prompt_mass(p, new[0], to_np(lse)[:k], ts, chunks, 16, sink, window)
        close(to_np(mass), before + added + dadd, mt + dmt + 4 * bref.EPS * (before + added + dadd), f"step {step}")
        del junk
