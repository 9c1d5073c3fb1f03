"""Attention over a sliding window and sinks, for single tokens and for chunks, and the masses of blocks, on the GPU against
their 64-bit forms (bounded_ref.py): types, head shapes, lengths, windows, masks that leave nothing, what stands in unseen
places."""
import numpy as np
import pytest

import bounded_ref as bref
import longctx_ref as ref
import paged_attention as pa
from helpers import empty_gpu, to_gpu, to_np

pytestmark = pytest.mark.gpu

FP32, BF16, INT8 = 0, 1, 2
TYPES = [(BF16, BF16), (BF16, FP32), (INT8, BF16), (INT8, FP32), (FP32, FP32), (FP32, BF16)]
SHAPES = [(8, 8, 32), (8, 2, 64), (32, 8, 128), (16, 1, 128), (8, 1, 256), (4, 2, 256), (12, 3, 64)]
I32 = np.int32


def gpu_pool(p):
    g = {"k": to_gpu(p.k), "v": to_gpu(p.v), "tables": to_gpu(p.tables)}
    g["stats"] = [to_gpu(s) for s in p.stats] if p.stats else [None] * 4
    return g


def run_decode(p, g, q, lens, sink, window, mass=None, max_len=None, stream=None):
    """(out, masses)"""
    import torch
    n, most = len(lens), int(max_len if max_len is not None else max(list(lens) + [1]))
    out = empty_gpu((n, p.hq, p.d), np.float32)
    out.fill_(float("nan"))
    gm = None if mass is None else to_gpu(mass)
    size = pa.window_decode_workspace_size(p.cfg, n, most, sink, window, mass is not None)
    ws = empty_gpu((size,), np.uint8)
    ws.fill_(0xFF)
    pa.window_decode(stream, p.cfg, out, to_gpu(q), g["k"], g["v"], g["stats"][0], g["stats"][1], g["tables"],
                     to_gpu(np.array(lens, I32)), n, p.width, most, sink, window, gm, ws, size)
    torch.cuda.synchronize()
    return to_np(out), None if mass is None else to_np(gm)


def run_prefill(p, g, q, lens, chunks, sink, window, lse=True, max_len=None, max_chunk=None, stream=None):
    """(out, lse)"""
    import torch
    n, most = len(lens), int(max_len if max_len is not None else max(list(lens) + [1]))
    longest = int(max_chunk if max_chunk is not None else max(chunks))
    rows = sum(chunks)
    out, gl = empty_gpu((rows + 1, p.hq, p.d), np.float32), empty_gpu((rows + 1, p.hq), np.float32)
    out.fill_(12345.0)
    gl.fill_(12345.0)
    size = pa.window_prefill_workspace_size(p.cfg, n, longest, most, sink, window)
    ws = empty_gpu((max(size, 16),), np.uint8)
    ws.fill_(0xFF)
    pa.window_prefill(stream, p.cfg, out, to_gpu(q), to_gpu(np.concatenate([[0], np.cumsum(chunks)]).astype(I32)),
                      to_gpu((np.array(lens) - np.array(chunks)).astype(I32)), g["k"], g["v"], g["stats"][0], g["stats"][1],
                      g["tables"], n, p.width, longest, most, sink, window, gl if lse else None, ws, size)
    torch.cuda.synchronize()
    out, gl = to_np(out), to_np(gl)
    assert (out[rows] == 12345.0).all() and (gl[rows] == 12345.0).all(), "rows behind the last sequence were written"
    if not lse:
        assert (gl == 12345.0).all()
    return out[:rows], gl[:rows]


def run_mass(p, g, q, lse, lens, chunks, last, sink, window, mass, max_len=None):
    import torch
    gm = to_gpu(mass)
    pa.prefill_mass(None, p.cfg, to_gpu(q), to_gpu(lse), to_gpu(np.concatenate([[0], np.cumsum(chunks)]).astype(I32)),
                    to_gpu((np.array(lens) - np.array(chunks)).astype(I32)), g["k"], g["stats"][0], g["tables"], len(lens),
                    p.width, int(max_len if max_len is not None else max(list(lens) + [1])), last, sink, window, gm)
    torch.cuda.synchronize()
    return to_np(gm)


def close(got, want, tol, what=""):
    assert np.isfinite(got).all(), f"{what}: not finite"
    off = np.abs(got - want) - tol
    assert off.max(initial=-1) <= 0, f"{what}: off by {np.abs(got - want).max():.3e}, tolerance {tol.max():.3e}"


def close_mass(got, before, added, tol):
    """An entry is the sum rounded once more; those that no token is seen in are as they were."""
    close(got, before + added, tol + 2 * bref.EPS * (np.abs(before) + added))
    np.testing.assert_array_equal(got[added == 0], before[added == 0])


def masses(p):
    return p.rng.exponential(3.0, p.tables.shape).astype(np.float32)


LENS = [1, 15, 16, 17, 0, 100, 333, 48, 7, 290]


@pytest.mark.parametrize("kv,q", TYPES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_decode(kv, q, hq, hkv, d):
    if kv == INT8 and d == 32:
        pytest.skip("int8 caches take head_dim 64 and more")
    p = ref.Pool(300 + 10 * kv + q, LENS, hq, hkv, d, kv, q)
    g = gpu_pool(p)
    for sink, window in ((0, 0), (4, 32), (0, 1), (17, 50), (3, 1000), (1000, 5), (0, 2 ** 31 - 1), (2 ** 31 - 1, 3), (16, 16)):
        qs = p.queries(len(LENS))
        out, tol, _, _, added, mass_tol = bref.decode(p, qs, LENS, sink, window)
        before = masses(p)
        got, mass = run_decode(p, g, qs, LENS, sink, window, before)
        close(got, out, tol, f"sink {sink}, window {window}")
        close_mass(mass, before, added, mass_tol)
        plain, _ = run_decode(p, g, qs, LENS, sink, window)
        np.testing.assert_array_equal(plain, got)


@pytest.mark.parametrize("kv,q", [(BF16, BF16), (INT8, FP32), (FP32, FP32)])
@pytest.mark.parametrize("sink,window", [(0, 0), (4, 1024), (100, 3000)])
def test_decode_long_and_ragged(kv, q, sink, window):
    lens = [20000, 3, 5001, 0, 900, 16 * 1024, 70, 1]
    p = ref.Pool(320 + kv, lens, 8, 2, 64, kv, q)
    qs = p.queries(len(lens))
    out, tol, _, _, added, mass_tol = bref.decode(p, qs, lens, sink, window)
    before = masses(p)
    got, mass = run_decode(p, gpu_pool(p), qs, lens, sink, window, before)
    close(got, out, tol)
    close_mass(mass, before, added, mass_tol)


@pytest.mark.parametrize("n,lens", [(40, 1000), (64, 128), (512, 40), (2100, 30), (4100, 3)])
@pytest.mark.parametrize("hkv", [1, 8])
def test_decode_rows_of_one_length(n, lens, hkv):
    """Whole rows a workgroup, several, or ranges; calls of more than one launch."""
    lens = [lens] * n
    lens[-1] = 1
    p = ref.Pool(330, lens, hkv * 4, hkv, 32)
    qs = p.queries(n)
    for sink, window in ((0, 0), (2, 100)):
        out, tol, _, _, added, mass_tol = bref.decode(p, qs, lens, sink, window)
        before = masses(p)
        got, mass = run_decode(p, gpu_pool(p), qs, lens, sink, window, before)
        close(got, out, tol)
        close_mass(mass, before, added, mass_tol)


def spoil(p, s, tokens, value):
    """Keys and values of these tokens of a row, all channels."""
    bad = ref.of_type(np.full(1, value, np.float32), p.kv)[0]
    for t in tokens:
        b = p.tables[s, t // 16]
        p.k[b, :, t % 16], p.v[b, :, :, t % 16] = bad, bad


@pytest.mark.parametrize("kv,q", [(BF16, BF16), (BF16, FP32), (FP32, FP32)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_unseen_tokens_do_not_matter(kv, q, value):
    """Expired tokens inside the window's first block, those between sinks and window, unused slots of the last block."""
    lens, sink, window = [200, 77, 333, 20], 5, 40
    p = ref.Pool(340, lens, 8, 2, 64, kv, q)
    qs = p.queries(4)
    out, tol, _, _, added, mass_tol = bref.decode(p, qs, lens, sink, window)
    chunks = [3, 1, 2, 20]
    rows, at = bref.chunk_rows(lens, chunks)
    cq = p.queries(len(rows))
    want = bref.attend(p, cq, rows, at, sink, window, [lens[s] for s in rows])
    for s, t in enumerate(lens):
        spoil(p, s, range(t, (t + 15) // 16 * 16), value)
    g = gpu_pool(p)  # what a chunk's oldest query still sees is left for now
    cout, lse = run_prefill(p, g, cq, lens, chunks, sink, window)
    close(cout, want[0], want[1])
    close(lse, want[2], want[3])
    for s, t in enumerate(lens):
        spoil(p, s, range(sink, max(sink, t - window)), value)
    g = gpu_pool(p)
    before = masses(p)
    got, mass = run_decode(p, g, qs, lens, sink, window, before)
    close(got, out, tol)
    close_mass(mass, before, added, mass_tol)
    # single tokens as chunks
    one, _ = run_prefill(p, g, qs, lens, [1] * 4, sink, window)
    close(one, out, tol)


@pytest.mark.parametrize("kv,q", [(BF16, BF16), (FP32, FP32), (BF16, FP32)])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (4, 4, 32), (8, 1, 128), (3, 1, 256)])
def test_a_token_that_only_some_queries_see(kv, q, value, hq, hkv, d):
    """A value that is not finite reaches the queries that see its token and no others: later tokens (causal) and expired ones."""
    for lens, chunks in (([150, 90], [150, 60]), ([600], [5])):
        sink, window = 3, 45
        p = ref.Pool(350, lens, hq, hkv, d, kv, q)
        rows, at = bref.chunk_rows(lens, chunks)
        qs = p.queries(len(rows))
        want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, sink, window, [lens[s] for s in rows])
        bad = ref.of_type(np.full(1, value, np.float32), kv)[0]
        t = lens[0] - 3
        p.v[p.tables[0, t // 16], :, 5, t % 16] = bad  # one channel of one late token
        old = lens[0] - chunks[0] + 1 - window + 1 if chunks[0] < lens[0] else 40  # seen by the first queries alone
        p.v[p.tables[0, old // 16], :, 9, old % 16] = bad
        got, glse = run_prefill(p, gpu_pool(p), qs, lens, chunks, sink, window)
        close(glse, lse, lse_tol)
        touched = np.zeros(got.shape, bool)
        for r, (s, pos) in enumerate(zip(rows, at)):
            if s == 0:
                touched[r, :, 5] = bref.seen(pos, t, sink, window)
                touched[r, :, 9] = bref.seen(pos, old, sink, window)
        assert touched.any() and not touched[:, :, 5].all()
        assert not np.isfinite(got[touched]).any()
        np.testing.assert_array_less(np.abs(got - want)[~touched], (tol + np.zeros(got.shape))[~touched])


def test_nan_queries_and_keys_stay_in_their_rows():
    lens, chunks = [120, 64, 80], [40, 64, 3]
    p = ref.Pool(360, lens, 4, 2, 64, BF16, BF16)
    rows, at = bref.chunk_rows(lens, chunks)
    qs = p.queries(len(rows))
    qs[5, 1] = 0x7fc0
    want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, 4, 30, [lens[s] for s in rows])
    got, glse = run_prefill(p, gpu_pool(p), qs, lens, chunks, 4, 30)
    assert np.isnan(got[5, 1]).all() and np.isnan(glse[5, 1])
    keep = np.ones(len(rows) * 4, bool)
    keep[21] = False
    close(got.reshape(-1, 64)[keep], want.reshape(-1, 64)[keep], np.broadcast_to(tol.reshape(-1, 1), (len(rows) * 4, 64))[keep])
    dq = p.queries(3)
    dq[1, 2] = 0x7fc0
    out, dtol, _, _, _, _ = bref.decode(p, dq, lens, 4, 30)
    dgot, _ = run_decode(p, gpu_pool(p), dq, lens, 4, 30)
    assert np.isnan(dgot[1, 2]).all()
    keep = np.ones(12, bool)
    keep[6] = False
    close(dgot.reshape(-1, 64)[keep], out.reshape(-1, 64)[keep], np.broadcast_to(dtol.reshape(-1, 1), (12, 64))[keep])


@pytest.mark.parametrize("kv", [BF16, INT8, FP32])
def test_blocks_that_are_none_read_as_zeros(kv):
    lens = [100, 64, 200]
    p = ref.Pool(370, lens, 8, 2, 64, kv, FP32)
    p.tables[0, 2], p.tables[1, 0], p.tables[2, 12], p.tables[2, 5] = -1, p.nb, 2 ** 31 - 1, -2 ** 31
    g = gpu_pool(p)
    for sink, window in ((0, 0), (5, 70)):
        qs = p.queries(3)
        out, tol, _, _, added, mass_tol = bref.decode(p, qs, lens, sink, window)
        before = masses(p)
        got, mass = run_decode(p, g, qs, lens, sink, window, before)
        close(got, out, tol)
        close_mass(mass, before, added, mass_tol)
        chunks = [9, 64, 2]
        rows, at = bref.chunk_rows(lens, chunks)
        cq = p.queries(len(rows))
        want = bref.attend(p, cq, rows, at, sink, window, [lens[s] for s in rows])
        cout, lse = run_prefill(p, g, cq, lens, chunks, sink, window)
        close(cout, want[0], want[1])
        close(lse, want[2], want[3])
        added, mt = bref.prompt_mass(p, cq, lse, lens, chunks, 7, sink, window)
        close_mass(run_mass(p, g, cq, lse, lens, chunks, 7, sink, window, before), before, added, mt)


def test_contexts_past_the_bounds():
    """Lengths beyond the table and beyond max_context_len are read up to these; queries whose window lies past them see nothing."""
    lens = [100, 64, 40]
    p = ref.Pool(380, lens, 4, 2, 64)
    g = gpu_pool(p)
    qs = p.queries(3)
    long = [5000, 64, 40]  # the table is 7 blocks wide; 50 tokens are read at most
    out, tol, _, _, _, _ = bref.decode(p, qs, long, 3, 20, 50)
    got, _ = run_decode(p, g, qs, long, 3, 20, max_len=50)
    close(got, out, tol)
    # chunk of 30 at positions 80 .. 109 of a table of 112 tokens, read up to 90: the last see the sinks, or nothing
    rows, at = [0] * 30, list(range(80, 110))
    cq = p.queries(30)
    for sink in (3, 0):
        want = bref.attend(p, cq, rows, at, sink, 8, [110] * 30, 90)
        cout, lse = run_prefill(p, g, cq, [110], [30], sink, 8, max_len=90)
        close(cout, want[0], want[1])
        seen = np.isfinite(want[2])
        assert seen.all() == (sink > 0)
        close(lse[seen], want[2][seen], want[3][seen])
        assert (lse[~seen] == -np.inf).all() and (cout[~seen] == 0).all()


CHUNKS = [([1, 17, 333, 64, 130], [1, 17, 33, 0, 130]), ([700], [700]), ([500, 90], [3, 5]), ([40] * 30, [7] * 30)]


@pytest.mark.parametrize("kv,q", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 32), (8, 2, 64), (32, 8, 128), (16, 1, 128), (3, 1, 256), (20, 4, 64), (6, 6, 128)])
def test_prefill_and_mass(kv, q, hq, hkv, d):
    if kv == INT8 and d == 32:
        pytest.skip("int8 caches take head_dim 64 and more")
    for lens, chunks in CHUNKS:
        if len(lens) == 30 and hq != 8 or lens == [700] and hq > 16:
            continue
        p = ref.Pool(390 + kv + 3 * q, lens, hq, hkv, d, kv, q)
        g = gpu_pool(p)
        rows, at = bref.chunk_rows(lens, chunks)
        for sink, window in ((0, 0), (4, 32), (40, 1), (0, 100), (1000, 7)):
            qs = p.queries(len(rows))
            want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, sink, window, [lens[s] for s in rows])
            got, glse = run_prefill(p, g, qs, lens, chunks, sink, window)
            close(got, want, tol, f"chunks {chunks[:5]}, sink {sink}, window {window}")
            close(glse, lse, lse_tol)
            again, _ = run_prefill(p, g, qs, lens, chunks, sink, window, lse=False)
            np.testing.assert_array_equal(again, got)
            for last in (1, 9, 2000):
                before = masses(p)
                added, mass_tol = bref.prompt_mass(p, qs, glse, lens, chunks, last, sink, window)
                close_mass(run_mass(p, g, qs, glse, lens, chunks, last, sink, window, before), before, added, mass_tol)


@pytest.mark.parametrize("kv,q", [(BF16, BF16), (INT8, BF16), (FP32, FP32)])
@pytest.mark.parametrize("chunk", [1, 4, 9, 33, 100])
@pytest.mark.parametrize("sink,window", [(0, 0), (4, 2500)])
def test_short_chunks_on_long_contexts(kv, q, chunk, sink, window):
    lens = [6000, 200]
    chunks = [chunk, min(chunk, 3)]
    p = ref.Pool(400 + kv, lens, 8, 2, 128, kv, q)
    g = gpu_pool(p)
    rows, at = bref.chunk_rows(lens, chunks)
    qs = p.queries(len(rows))
    want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, sink, window, [lens[s] for s in rows])
    got, glse = run_prefill(p, g, qs, lens, chunks, sink, window)
    close(got, want, tol)
    close(glse, lse, lse_tol)
    before = masses(p)
    added, mass_tol = bref.prompt_mass(p, qs, glse, lens, chunks, 40, sink, window)
    close_mass(run_mass(p, g, qs, glse, lens, chunks, 40, sink, window, before), before, added, mass_tol)


@pytest.mark.parametrize("kv,q", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 32), (8, 2, 64), (8, 1, 64), (32, 8, 128), (3, 1, 256), (20, 4, 128)])
def test_masses_of_many_prompts(kv, q, hq, hkv, d):
    """Calls that fill the chip, of long and short contexts, with block counts that no workgroup divides."""
    if kv == INT8 and d == 32:
        pytest.skip("int8 caches take head_dim 64 and more")
    lens = [310, 17, 130, 0, 270] + [i % 23 + 1 for i in range(65)]
    chunks = [min(t, (7 * i) % 37) for i, t in enumerate(lens)]
    p = ref.Pool(395 + kv + 3 * q, lens, hq, hkv, d, kv, q)
    g = gpu_pool(p)
    rows, at = bref.chunk_rows(lens, chunks)
    for sink, window, last in ((0, 0, 13), (4, 90, 2000)):
        qs = p.queries(len(rows))
        want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, sink, window, [lens[s] for s in rows])
        got, glse = run_prefill(p, g, qs, lens, chunks, sink, window)
        close(got, want, tol)
        close(glse, lse, lse_tol)
        before = masses(p)
        close_mass(run_mass(p, g, qs, glse, lens, chunks, last, sink, window, before), before,
                   *bref.prompt_mass(p, qs, glse, lens, chunks, last, sink, window))


def test_max_chunk_len_bounds_what_is_computed():
    lens, chunks = [100, 50], [40, 6]
    p = ref.Pool(410, lens, 4, 2, 64)
    rows, at = bref.chunk_rows(lens, chunks)
    qs = p.queries(len(rows))
    got, lse = run_prefill(p, gpu_pool(p), qs, lens, chunks, 0, 16, max_chunk=9)
    want = bref.attend(p, qs, rows, at, 0, 16, [lens[s] for s in rows])
    keep = [*range(9), *range(40, 46)]
    close(got[keep], want[0][keep], want[1][keep])
    assert (got[9:40] == 12345.0).all() and (lse[9:40] == 12345.0).all()


@pytest.mark.parametrize("scale", [0.01, 3.0])
def test_scales(scale):
    lens, chunks = [300, 40], [30, 40]
    p = ref.Pool(420, lens, 8, 2, 64, BF16, FP32)
    p.cfg.scale = scale
    g = gpu_pool(p)
    qs = p.queries(2)
    out, tol, _, _, added, mass_tol = bref.decode(p, qs, lens, 2, 90)
    before = masses(p)
    got, mass = run_decode(p, g, qs, lens, 2, 90, before)
    close(got, out, tol)
    close_mass(mass, before, added, mass_tol)
    rows, at = bref.chunk_rows(lens, chunks)
    qs = p.queries(len(rows))
    want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, 2, 90, [lens[s] for s in rows])
    got, glse = run_prefill(p, g, qs, lens, chunks, 2, 90)
    close(got, want, tol)
    close(glse, lse, lse_tol)


def test_same_inputs_same_bits():
    lens = [900, 5000, 31, 2500]
    p = ref.Pool(430, lens, 32, 8, 128)
    g = gpu_pool(p)
    qs, before = p.queries(4), masses(p)
    first = run_decode(p, g, qs, lens, 4, 0, before)
    for _ in range(3):
        again = run_decode(p, g, qs, lens, 4, 0, before)
        np.testing.assert_array_equal(again[0], first[0])
        np.testing.assert_array_equal(again[1], first[1])


@pytest.mark.parametrize("old", [2, 40])
def test_scores_of_minus_infinity_weigh_nothing(old):
    """Seen keys of -Inf against queries that are positive throughout, in whole blocks before others whose scores lie far below 0."""
    lens = [old * 16 + 40, 40]
    p = ref.Pool(440, lens, 8, 2, 64)
    p.cfg.scale = 1.0
    qs = ref.of_type(np.abs(p.rng.standard_normal((2, 8, 64))).astype(np.float32) + 1, BF16)
    p.k[:] = ref.of_type(np.full(1, -3, np.float32), BF16)[0]  # scores of -192 and less
    for b in range(old):
        p.k[p.tables[0, b]] = ref.of_type(np.full(1, -np.inf, np.float32), BF16)[0]
    finite = ref.Pool(440, lens, 8, 2, 64)  # the same with those blocks out of the window
    finite.k, finite.v, finite.cfg, finite.tables = p.k.copy(), p.v, p.cfg, p.tables
    for b in range(old):
        finite.k[p.tables[0, b]] = 0
    out, tol, lse, lse_tol, added, mass_tol = bref.decode(finite, qs, lens, 0, 40)
    g, before = gpu_pool(p), masses(p)
    got, glse = run_prefill(p, g, qs, lens, [1, 1], 0, 0)
    close(got, out, tol)
    close(glse, lse, lse_tol)
    close_mass(run_mass(p, g, qs, glse, lens, [1, 1], 1, 0, 0, before), before,
               *bref.prompt_mass(finite, qs, glse, lens, [1, 1], 1, 0, 40))
    got, mass = run_decode(p, g, qs, lens, 0, 0, before)
    close(got, out, tol)
    close_mass(mass, before, added, mass_tol)


def test_caches_past_4_gib():
    """Blocks at both ends of a cache whose offsets need more than 32 bits."""
    import torch
    lens, chunks = [700, 90], [60, 3]
    p = ref.Pool(450, lens, 32, 8, 128)
    far = 150000
    assert far * 8 * 16 * 128 * 2 > 2 ** 32
    g = gpu_pool(p)
    k, v = (torch.empty((far, 8, 16 * 128), dtype=torch.int16, device="cuda") for _ in range(2))
    at = np.arange(p.nb) + np.where(np.arange(p.nb) % 2, far - p.nb, 0)
    index = to_gpu(at.astype(np.int64))
    k[index] = to_gpu(p.k).reshape(p.nb, 8, -1)
    v[index] = to_gpu(p.v).reshape(p.nb, 8, -1)
    g["k"], g["v"], g["tables"] = k, v, to_gpu(np.where(p.tables >= 0, at[p.tables], -1).astype(I32))
    rows, pos = bref.chunk_rows(lens, chunks)
    cq, dq = p.queries(len(rows)), p.queries(2)
    want = bref.attend(p, cq, rows, pos, 4, 300, [lens[s] for s in rows])
    out, tol, _, _, added, mass_tol = bref.decode(p, dq, lens, 4, 300)
    p.cfg.num_blocks = far
    before = masses(p)
    got, mass = run_decode(p, g, dq, lens, 4, 300, before)
    close(got, out, tol)
    close_mass(mass, before, added, mass_tol)
    got, lse = run_prefill(p, g, cq, lens, chunks, 4, 300)
    close(got, want[0], want[1])
    close(lse, want[2], want[3])
    close_mass(run_mass(p, g, cq, lse, lens, chunks, 9, 4, 300, before), before, *bref.prompt_mass(p, cq, lse, lens, chunks, 9, 4, 300))


def test_two_streams_at_once_and_a_replayed_graph():
    """Calls with workspaces of their own on two streams of the caller, and the same calls captured: every outcome is the eager one's."""
    import torch
    lens, chunks = [4000, 90, 33, 1200], [5, 40, 33, 1]
    p = ref.Pool(460, lens, 8, 2, 128)
    g = gpu_pool(p)
    n, rows = len(lens), sum(chunks)
    start, prefix = to_gpu(np.concatenate([[0], np.cumsum(chunks)]).astype(I32)), to_gpu((np.array(lens) - np.array(chunks)).astype(I32))
    glens, zeros = to_gpu(np.array(lens, I32)), np.zeros(p.tables.shape, np.float32)
    qs = [(p.queries(rows), p.queries(n)) for _ in range(4)]
    wp = pa.window_prefill_workspace_size(p.cfg, n, 40, 4000, 4, 3000)
    wd = pa.window_decode_workspace_size(p.cfg, n, 4000, 4, 3000, True)

    class Lane:
        def __init__(self):
            self.cq, self.dq = to_gpu(qs[0][0]), to_gpu(qs[0][1])
            self.out, self.lse, self.one = (empty_gpu(s, np.float32) for s in ((rows, 8, 128), (rows, 8), (n, 8, 128)))
            self.mass = to_gpu(zeros)
            self.wp, self.wd = empty_gpu((wp,), np.uint8), empty_gpu((wd,), np.uint8)

        def run(self, stream):
            st = pa.Stream(pa.Device(0), stream.cuda_stream)
            self.mass.zero_()
            pa.window_prefill(st, p.cfg, self.out, self.cq, start, prefix, g["k"], g["v"], None, None, g["tables"], n, p.width, 40, 4000,
                              4, 3000, self.lse, self.wp, wp)
            pa.prefill_mass(st, p.cfg, self.cq, self.lse, start, prefix, g["k"], None, g["tables"], n, p.width, 4000, 16, 4, 3000,
                            self.mass)
            pa.window_decode(st, p.cfg, self.one, self.dq, g["k"], g["v"], None, None, g["tables"], glens, n, p.width, 4000, 4, 3000,
                             self.mass, self.wd, wd)

        def set(self, q):
            self.cq.copy_(to_gpu(q[0]))
            self.dq.copy_(to_gpu(q[1]))

        def result(self):
            torch.cuda.synchronize()
            return [to_np(x).copy() for x in (self.out, self.lse, self.one, self.mass)]

    eager, want = Lane(), []
    for q in qs:
        eager.set(q)
        eager.run(torch.cuda.current_stream())
        want.append(eager.result())
    out, tol, _, _, _, _ = bref.decode(p, qs[0][1], lens, 4, 3000)
    close(want[0][2], out, tol)
    lanes, streams = [Lane(), Lane()], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, lane in enumerate(lanes):
        lane.set(qs[i])
    torch.cuda.synchronize()
    for _ in range(5):
        for lane, s in zip(lanes, streams):
            with torch.cuda.stream(s):
                lane.run(s)
    for i, lane in enumerate(lanes):
        for a, b in zip(lane.result(), want[i]):
            np.testing.assert_array_equal(a, b)
    graph, lane = torch.cuda.CUDAGraph(), lanes[0]
    with torch.cuda.graph(graph, stream=streams[0]):
        lane.run(streams[0])
    for i in (2, 0, 3, 1, 2):
        lane.set(qs[i])
        graph.replay()
        for a, b in zip(lane.result(), want[i]):
            np.testing.assert_array_equal(a, b)
        eager.set(qs[i - 1])
        eager.run(torch.cuda.current_stream())
