"""The forms of the attention over a window and sinks that the host's rules choose by sizes: chunks whose waves own their columns
or share them, streams longer than what a wave's lanes name at once, single tokens over whole rows, over ranges of several
stretches, one sequence. Against the 64-bit forms of bounded_ref.py.

The rules look at the host's bounds (max_chunk_len, num_seqs), so a loose bound or many tiny sequences bring a form about
while few rows have to be compared; sequences of one long text share its blocks, as forked ones do."""
import numpy as np
import pytest

import bounded_ref as bref
import longctx_ref as ref
import paged_attention as pa
from helpers import check_close, empty_gpu, to_gpu, to_np, tol_for
from test_gpu_window import BF16, FP32, I32, INT8, TYPES, close, close_mass, gpu_pool, masses, run_decode, run_mass, run_prefill

pytestmark = pytest.mark.gpu

FORMS = [(kv, q, d) for kv, q in TYPES for d in (32, 64, 128, 256) if not (kv == INT8 and d == 32)]
HEADS = {32: (8, 2), 64: (8, 2), 128: (4, 2), 256: (2, 2)}
CHUNK_BOUND = {32: 2200, 64: 2200, 128: 4200, 256: 8400}  # 4 (sequence, KV head), over 256 workgroups of 128 columns


def check_chunks(p, lens, chunks, sink, window, bound):
    rows, at = bref.chunk_rows(lens, chunks)
    qs = p.queries(len(rows))
    g = gpu_pool(p)
    want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, sink, window, [lens[s] for s in rows])
    got, glse = run_prefill(p, g, qs, lens, chunks, sink, window, max_chunk=bound)
    close(got, want, tol, f"sink {sink}, window {window}")
    close(glse, lse, lse_tol, f"lse, sink {sink}, window {window}")


@pytest.mark.parametrize("kv,q,d", FORMS)
def test_chunks_with_columns_of_their_own(kv, q, d):
    """Waves that own 32 columns each; contexts of more than the 32 pairs of blocks that a wave's lanes name, past their refill."""
    hq, hkv = HEADS[d]
    lens, chunks = [1500, 70], [45, 70]
    p = ref.Pool(600 + 10 * kv + q, lens, hq, hkv, d, kv, q)
    for sink, window in ((0, 0), (20, 1200), (4, 33)):
        check_chunks(p, lens, chunks, sink, window, CHUNK_BOUND[d])


@pytest.mark.parametrize("kv,q,d", [f for f in FORMS if not (f[0] == FP32 and f[2] == 256)])  # (which never shares)
def test_chunks_with_shared_columns_on_long_contexts(kv, q, d):
    """Four waves that take the pairs of blocks in turn, more than 32 pairs each: 33 sequences of 8 KV heads leave keys uncut."""
    lens = [4500] + [6] * 32
    chunks = [5] + [2] * 32
    p = ref.Pool(610 + 10 * kv + q, lens, 8, 8, d, kv, q)
    for sink, window in ((0, 0), (9, 4300)):
        check_chunks(p, lens, chunks, sink, window, 5)


@pytest.mark.parametrize("kv,q", [(BF16, BF16), (FP32, FP32), (BF16, FP32)])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_a_token_that_only_some_queries_see_in_columns_of_their_own(kv, q, value, d):
    hq, hkv = HEADS[d]
    lens, chunks, sink, window = [1300, 60], [60, 60], 3, 1200
    p = ref.Pool(620, lens, hq, hkv, d, kv, q)
    rows, at = bref.chunk_rows(lens, chunks)
    qs = p.queries(len(rows))
    want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, sink, window, [lens[s] for s in rows])
    bad = ref.of_type(np.full(1, value, np.float32), kv)[0]
    late, old = 1270, 60  # seen by the chunk's last queries alone, by its first alone
    p.v[p.tables[0, late // 16], :, 5, late % 16] = bad
    p.v[p.tables[0, old // 16], :, 9, old % 16] = bad
    got, glse = run_prefill(p, gpu_pool(p), qs, lens, chunks, sink, window, max_chunk=CHUNK_BOUND[d])
    close(glse, lse, lse_tol)
    touched = np.zeros(got.shape, bool)
    for r, (s, pos) in enumerate(zip(rows, at)):
        if s == 0:
            touched[r, :, 5] = bref.seen(pos, late, sink, window)
            touched[r, :, 9] = bref.seen(pos, old, sink, window)
    assert touched[:60, :, 5].any() and not touched[:60, :, 5].all() and touched[:60, :, 9].any() and not touched[:60, :, 9].all()
    assert not np.isfinite(got[touched]).any()
    np.testing.assert_array_less(np.abs(got - want)[~touched], (tol + np.zeros(got.shape))[~touched])


def forked(seed, n, lens, hq, hkv, d, kv, q):
    """n sequences of the given lengths (one, or one each) over the blocks of one text."""
    most = max(lens)
    p = ref.Pool(seed, [most], hq, hkv, d, kv, q)
    p.tables = np.repeat(p.tables, n, axis=0)
    for s, t in enumerate(lens):
        p.tables[s, (t + 15) // 16:] = -1
    return p


def check_decode(p, lens, sink, window, sample):
    """Every row's masses add to the query heads; a sample of rows in full. (A head's weights are divided by their own sum: what
    scores are off by cancels, the roundings of the sums' additions are left, and those of the entries.)"""
    n = len(lens)
    qs, before = p.queries(n), masses(p)
    got, mass = run_decode(p, gpu_pool(p), qs, lens, sink, window, before)
    plain, _ = run_decode(p, gpu_pool(p), qs, lens, sink, window)
    np.testing.assert_array_equal(plain, got)
    assert np.isfinite(got).all()
    sample = sorted({s % n for s in sample})
    out, tol, _, _, added, mass_tol = bref.attend(p, qs[sample], sample, [lens[s] - 1 for s in sample], sink, window,
                                                  [lens[s] for s in sample])
    close(got[sample], out, tol)
    close_mass(mass[sample], before[sample], added[sample], mass_tol[sample])
    total = (mass.astype(np.float64) - before).sum(1)
    slack = 2 * bref.EPS * mass.sum(1) + p.hq * (4 * np.sqrt(max(lens) * p.hq) + 16) * bref.EPS
    assert (np.abs(total - p.hq) <= slack).all()


@pytest.mark.parametrize("kv,q", TYPES)
@pytest.mark.parametrize("length", [1, 16, 17, 129, 1028, 5000])
def test_decode_of_one_sequence(kv, q, length):
    for hq, hkv, d in ((32, 8, 128), (8, 1, 64), (2, 2, 256)):
        p = ref.Pool(630 + kv, [length], hq, hkv, d, kv, q)
        for sink, window in ((0, 0), (4, 1024), (0, 1)):
            check_decode(p, [length], sink, window, [0])


@pytest.mark.parametrize("kv,q,hq,hkv,d", [(BF16, BF16, 32, 8, 128), (BF16, FP32, 8, 8, 64), (INT8, FP32, 16, 4, 128), (FP32, FP32, 8, 4, 256),
                                           (FP32, BF16, 4, 4, 32), (BF16, BF16, 64, 4, 128), (INT8, BF16, 16, 2, 256)])
@pytest.mark.parametrize("blocks", [3, 8, 40])
def test_decode_of_whole_rows(kv, q, hq, hkv, d, blocks):
    """Sequences of truly one length, one or several rows to a workgroup."""
    for n in (256 // hkv, 512 // hkv, 640 // hkv):
        lens = [16 * blocks - 5] * n
        p = forked(640 + kv, n, lens, hq, hkv, d, kv, q)
        check_decode(p, lens, 0, 0, [0, 1, n // 2, n - 1])
        check_decode(p, lens, 5, 16 * blocks - 30, [2, n - 2])


@pytest.mark.parametrize("kv,q,hq,hkv,d", [(BF16, BF16, 32, 8, 128), (BF16, FP32, 8, 8, 64), (INT8, FP32, 16, 8, 128), (FP32, FP32, 8, 8, 256),
                                           (INT8, BF16, 8, 8, 64), (BF16, BF16, 32, 2, 128), (FP32, BF16, 8, 8, 32)])
@pytest.mark.parametrize("even", [True, False])
def test_decode_of_several_stretches(kv, q, hq, hkv, d, even):
    """Workgroups with more than the 256 list entries that their lanes name at once: whole rows of 700 blocks, and ranges that cross rows of
    many lengths."""
    n = 1024 // hkv
    lens = [11195] * n if even else [9000 + 37 * (i % 128) for i in range(n)]
    p = forked(650 + kv, n, lens, hq, hkv, d, kv, q)
    check_decode(p, lens, 0, 0, [77, n - 1])
    check_decode(p, lens, 40, 8000, [5])


@pytest.mark.parametrize("kv,q", [(BF16, BF16), (INT8, FP32), (FP32, FP32)])
@pytest.mark.parametrize("sink,window", [(0, 0), (4, 9)])
def test_prompt_masses_of_contexts_past_the_bounds(kv, q, sink, window):
    """Prompts longer than max_context_len, and than the table: tokens behind either are not seen, blocks behind them as they were."""
    lens, chunks = [110, 40, 112], [30, 40, 3]
    p = ref.Pool(660, lens, 8, 2, 64, kv, q)
    g = gpu_pool(p)
    long = [110, 40, 150]  # the last queries of the third lie past the table of 112 tokens
    rows, at = bref.chunk_rows(long, chunks)
    qs = p.queries(len(rows))
    before = masses(p)
    for most in (90, 150):
        want, tol, lse, lse_tol, _, _ = bref.attend(p, qs, rows, at, sink, window, [long[s] for s in rows], most)
        got, glse = run_prefill(p, g, qs, long, chunks, sink, window, max_len=most)
        close(got, want, tol)
        seen = np.isfinite(lse)
        close(glse[seen], lse[seen], lse_tol[seen])
        assert (glse[~seen] == -np.inf).all()
        for last in (2, 17, 64):
            added, mass_tol = bref.prompt_mass(p, qs, glse, long, chunks, last, sink, window, most)
            close_mass(run_mass(p, g, qs, glse, long, chunks, last, sink, window, before, most), before, added, mass_tol)


@pytest.mark.parametrize("kv,q", [(BF16, BF16), (FP32, FP32)])
def test_single_tokens_and_chunks_past_the_bounds(kv, q):
    """A context that is longer than the host's bounds: for a single token it ends there, window and masses too; a chunk's token keeps its
    position, and where its window lies past the bounds it sees nothing."""
    lens, sink, window, most = [200, 45, 200], 0, 20, 50
    p = ref.Pool(670, lens, 8, 2, 64, kv, q)
    g, qs, before = gpu_pool(p), p.queries(3), masses(p)
    out, tol, _, _, added, mass_tol = bref.attend(p, qs, range(3), [49, 44, 49], sink, window, [50, 45, 50])
    for long in ([200, 45, 5000], [50, 45, 50]):
        got, mass = run_decode(p, g, qs, long, sink, window, before, max_len=most)
        close(got, out, tol)
        close_mass(mass, before, added, mass_tol)
    got, lse = run_prefill(p, g, qs, [200, 45, 5000], [1, 1, 1], sink, window, max_len=most)
    close(got[1:2], out[1:2], tol[1:2])
    assert (got[[0, 2]] == 0).all() and (lse[[0, 2]] == -np.inf).all()


@pytest.mark.parametrize("kv,q", [(BF16, BF16), (INT8, FP32)])
def test_masses_by_the_last_tokens_of_prompts_alone(kv, q):
    """Prompts attended to by the chunks' other kernel, their last tokens once more for the logarithms that their masses need."""
    import torch
    lens, last = [700, 90, 20], 32
    p = ref.Pool(680, lens, 8, 2, 64, kv, q)
    g = gpu_pool(p)
    whole = p.queries(sum(lens))
    start = np.concatenate([[0], np.cumsum(lens)]).astype(I32)
    out = empty_gpu(whole.shape, np.float32)
    pa.chunked_prefill(None, p.cfg, out, to_gpu(whole), to_gpu(start), to_gpu(np.zeros(3, I32)), g["k"], g["v"], g["stats"][0], g["stats"][1],
                       g["tables"], 3, p.width, max(lens))
    torch.cuda.synchronize()
    chunks = [min(last, t) for t in lens]
    tail = np.concatenate([np.arange(start[s + 1] - n, start[s + 1]) for s, n in enumerate(chunks)])
    rows, at = bref.chunk_rows(lens, chunks)
    want, tol, lse, lse_tol, _, _ = bref.attend(p, whole[tail], rows, at, 0, 0, [lens[s] for s in rows])
    check_close(to_np(out)[tail], want, **tol_for(kv), what="chunked prefill")
    again, glse = run_prefill(p, g, whole[tail], lens, chunks, 0, 0)
    close(again, want, tol)
    close(glse, lse, lse_tol)
    before = masses(p)
    added, mass_tol = bref.prompt_mass(p, whole[tail], glse, lens, chunks, last, 0, 0)
    got = run_mass(p, g, whole[tail], glse, lens, chunks, last, 0, 0, before)
    close_mass(got, before, added, mass_tol)
    # a row's weights are the heads of its last tokens, by their own logarithms
    total = (got.astype(np.float64) - before).sum(1)
    slack = 2 * bref.EPS * got.sum(1) + mass_tol.sum(1) + added.sum(1) * lse_tol.max()
    assert (np.abs(total - 8 * np.array(chunks)) <= slack).all()


@pytest.mark.parametrize("kv", [BF16, FP32])
@pytest.mark.parametrize("window", [0, 700])
def test_values_that_are_not_finite_cost_little_time(kv, window):
    """Prompts whose values are NaN throughout, or at one token of many, take a small multiple of the time of finite ones."""
    import torch
    lens = [2048, 2048]
    p = ref.Pool(690, lens, 8, 2, 64, kv, kv)
    g, n = gpu_pool(p), sum(lens)
    q, out = to_gpu(p.queries(n)), empty_gpu((n, 8, 64), np.float32)
    start, prefix = to_gpu(np.array([0, 2048, 4096], I32)), to_gpu(np.zeros(2, I32))
    size = pa.window_prefill_workspace_size(p.cfg, 2, 2048, 2048, 0, window)
    ws = empty_gpu((max(size, 16),), np.uint8)

    def took(v):
        values, times = to_gpu(v), []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            pa.window_prefill(None, p.cfg, out, q, start, prefix, g["k"], values, None, None, g["tables"], 2, p.width, 2048, 2048, 0, window,
                              None, ws, size)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    bad = ref.of_type(np.full(1, np.nan, np.float32), kv)[0]
    one, whole = p.v.copy(), np.full_like(p.v, bad)
    one[p.tables[0, 64], :, 5, 3] = bad
    finite = took(p.v)
    assert took(one) < 10 * finite and took(whole) < 10 * finite
