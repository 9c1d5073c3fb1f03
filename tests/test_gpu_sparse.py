"""Key bounds, block selection and attention over selected blocks on the GPU against their 64-bit forms
(longctx_ref.py): types, head shapes, context lengths around block borders, lists and masks that leave nothing, and the three
together as a decode step uses them, in a graph too."""
import numpy as np
import pytest

import longctx_ref as ref
import paged_attention as pa
from helpers import empty_gpu, to_gpu, to_np

pytestmark = pytest.mark.gpu

FP32, BF16, INT8 = 0, 1, 2
SHAPES = [(8, 8, 32), (8, 2, 64), (32, 8, 128), (16, 1, 128), (8, 1, 256), (4, 2, 256), (16, 1, 64), (3, 3, 128), (12, 3, 64)]


def gpu_pool(p):
    g = {"k": to_gpu(p.k), "v": to_gpu(p.v), "tables": to_gpu(p.tables), "bounds": to_gpu(p.bounds)}
    g["stats"] = [to_gpu(s) for s in p.stats] if p.stats else [None] * 4
    return g


def run_bounds(p, g, start, num_new, stream=None, most=None):
    pa.key_bounds_update(stream, p.cfg, g["k"], g["tables"], p.width, to_gpu(np.array(start, np.int32)),
                         to_gpu(np.array(num_new, np.int32)), len(start), most or max(list(num_new) + [1]), g["bounds"])
    import torch
    torch.cuda.synchronize()
    return to_np(g["bounds"], ref.NP_DTYPE[p.kv])


def run_select(p, g, q, rows, lens, sink, recent, budget, max_len=None, stream=None):
    import torch
    n, most = len(lens), int(max_len if max_len is not None else max(list(lens) + [1]))
    out = empty_gpu((n, p.hkv, budget), np.int32)
    out.fill_(-7)
    size = pa.select_workspace_size(p.cfg, n, most)
    ws = empty_gpu((max(size, 8),), np.uint8)
    ws.fill_(0xFF)
    pa.select_blocks(stream, p.cfg, to_gpu(q), g["bounds"], g["stats"][0], g["tables"], len(p.tables), p.width,
                     None if rows is None else to_gpu(np.array(rows, np.int32)), to_gpu(np.array(lens, np.int32)), n, most, sink,
                     recent, budget, out, ws, size)
    torch.cuda.synchronize()
    return to_np(out)


def run_sparse(p, g, q, rows, lens, selected, max_len=None, stream=None):
    import torch
    n, budget = len(lens), selected.shape[2]
    most = int(max_len if max_len is not None else max(list(lens) + [1]))
    out = empty_gpu((n, p.hq, p.d), np.float32)
    out.fill_(float("nan"))
    size = pa.sparse_workspace_size(p.cfg, n, budget)
    ws = empty_gpu((max(size, 8),), np.uint8)
    ws.fill_(0xFF)
    pa.sparse_decode(stream, p.cfg, out, to_gpu(q), g["k"], g["v"], g["stats"][0], g["stats"][1], g["tables"], len(p.tables),
                     p.width, None if rows is None else to_gpu(np.array(rows, np.int32)), to_gpu(np.array(lens, np.int32)), n,
                     most, to_gpu(np.ascontiguousarray(selected, np.int32)), budget, ws, size)
    torch.cuda.synchronize()
    return to_np(out)


def close(got, want, tol, what=""):
    assert np.isfinite(got).all(), f"{what}: not finite"
    off = np.abs(got - want) - tol
    assert off.max(initial=-1) <= 0, f"{what}: off by {np.abs(got - want).max():.3e}, tolerance {tol.max():.3e}"


def random_lists(p, rows, lens, budget, rng):
    """Distinct blocks of each context in ascending order, its last block among them, -1 behind."""
    sel = np.full((len(lens), p.hkv, budget), -1, np.int32)
    for r, (s, t) in enumerate(zip(rows, lens)):
        n, _ = ref.blocks_of(p, s, t)
        for h in range(p.hkv):
            m = min(n, budget)
            if m:
                pick = np.append(rng.choice(n - 1, m - 1, replace=False), n - 1) if n > 1 else np.array([0])
                sel[r, h, :m] = np.sort(pick)
    return sel


@pytest.mark.parametrize("kv", [FP32, BF16, INT8])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_key_bounds_exact(kv, hq, hkv, d):
    if kv == INT8 and d == 32:
        pytest.skip("int8 caches take head_dim 64 and more")
    lens = [1, 2, 15, 16, 17, 31, 33, 160, 0, 48]
    p = ref.Pool(10 + kv, lens, hq, hkv, d, kv)
    p.tables[7, 3] = -1
    p.tables[7, 5] = p.nb
    start = [0, 1, 0, 15, 16, 3, 32, 0, 0, -1]
    new = [1, 1, 15, 1, 1, 28, 1, 160, 0, 5]
    g = gpu_pool(p)
    got = run_bounds(p, g, start, new)
    np.testing.assert_array_equal(got, ref.key_bounds(p, start, new))


def test_key_bounds_past_the_table_and_the_bound():
    p = ref.Pool(13, [64, 64, 40], kv=BF16)
    start, new = [60, 0, 2 ** 31 - 8], [500, 64, 2 ** 31 - 1]
    g = gpu_pool(p)
    got = run_bounds(p, g, start, new, most=18)  # 18 tokens touch three blocks at most
    np.testing.assert_array_equal(got, ref.key_bounds(p, [60, 0, 0], [4, 48, 0]))


@pytest.mark.parametrize("kv", [FP32, BF16])
def test_key_bounds_infinities_and_nan(kv):
    p = ref.Pool(14, [20, 16], kv=kv)
    inf, ninf, nan = (ref.of_type(np.float32(x).reshape(1), kv)[0] for x in (np.inf, -np.inf, np.nan))
    b = p.tables[0, 0]
    p.k[b, 0, 3, 5], p.k[b, 1, 4, 6], p.k[b, 0, 7, 9] = inf, ninf, nan
    p.k[p.tables[0, 1], :, 4:] = nan  # unused slots
    g = gpu_pool(p)
    got = ref.f64(run_bounds(p, g, [0, 0], [20, 16]))
    np.testing.assert_array_equal(got, ref.f64(ref.key_bounds(p, [0, 0], [20, 16])))
    assert np.isnan(got[b, 0, :, 9]).all() and got[b, 0, 1, 5] == np.inf and not np.isnan(got[p.tables[0, 1]]).any()


@pytest.mark.parametrize("kv,q", [(FP32, FP32), (BF16, BF16), (BF16, FP32), (INT8, BF16), (INT8, FP32), (FP32, BF16)])
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (32, 8, 128), (16, 1, 128), (8, 2, 256), (12, 3, 64)])
def test_select(kv, q, hq, hkv, d):
    lens = [1, 16, 17, 16 * 12, 16 * 12 + 1, 16 * 13, 16 * 64, 16 * 64 + 5, 16 * 200 - 1, 0, 16 * 77 + 9]
    p = ref.Pool(20 + kv, lens, hq, hkv, d, kv, q, values=False)
    qs = p.queries(len(lens))
    g = {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [to_gpu(s) for s in p.stats] if p.stats else [None] * 4}
    rows = range(len(lens))
    for sink, recent, budget in ((0, 1, 1), (1, 2, 12), (2, 3, 5), (1, 4, 40)):
        got = run_select(p, g, qs, None, lens, sink, recent, budget)
        np.testing.assert_array_equal(got, ref.select(p, qs, rows, lens, sink, recent, budget), err_msg=str((sink, recent, budget)))


def test_select_head_dim_32():
    lens = [500, 33, 16 * 40]
    for kv in (FP32, BF16):
        p = ref.Pool(29, lens, 4, 2, 32, kv, values=False)
        g = {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [None] * 4}
        qs = p.queries(3)
        np.testing.assert_array_equal(run_select(p, g, qs, None, lens, 1, 1, 9), ref.select(p, qs, range(3), lens, 1, 1, 9))


@pytest.mark.parametrize("blocks", [1023, 1024, 1025, 2500, 9001, 17000])
def test_select_long_contexts(blocks):
    p = ref.Pool(30, [16 * blocks - 3, 16 * (blocks // 2)], 4, 2, 64, BF16, values=False)
    g = {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [None] * 4}
    qs = p.queries(2)
    got = run_select(p, g, qs, None, p.lens, 1, 2, 100)
    np.testing.assert_array_equal(got, ref.select(p, qs, range(2), p.lens, 1, 2, 100))


@pytest.mark.parametrize("budget", [9, 64, 200])
def test_select_equal_scores_go_to_the_lowest_index(budget):
    p = ref.Pool(31, [16 * 300, 16 * 300, 16 * 300, 16 * 300], 4, 2, 64, BF16, values=False)
    same = p.bounds[0].copy()
    p.bounds[p.tables[0]] = same                       # every block alike
    p.bounds[p.tables[1, ::2]] = same                  # every other one
    p.bounds[p.tables[2, 150:]] = p.bounds[p.tables[2, :150]]  # pairs
    p.bounds[p.tables[3]] = 0
    p.bounds[p.tables[3, ::3]] = 0x8000                # zeros of both signs are equal
    g = {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [None] * 4}
    qs = p.queries(4)
    got = run_select(p, g, qs, None, p.lens, 1, 2, budget)
    np.testing.assert_array_equal(got, ref.select(p, qs, range(4), p.lens, 1, 2, budget))


def test_select_scores_that_differ_in_the_last_bits():
    """Scores near 1 that differ by 2^-30 of it and less: sums in 32 bits could not tell them apart."""
    p = ref.Pool(32, [16 * 400], 1, 1, 64, FP32, FP32, values=False)
    rng = np.random.default_rng(5)
    p.bounds[:] = 0
    step = (rng.permutation(400) * 2.0 ** -33).astype(np.float32)
    p.bounds[p.tables[0], 0, 1, 0] = 1
    p.bounds[p.tables[0], 0, 1, 1] = step
    qs = np.zeros((1, 1, 64), np.float32)
    qs[0, 0, :2] = 1
    g = {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [None] * 4}
    np.testing.assert_array_equal(run_select(p, g, qs, None, p.lens, 1, 2, 50), ref.select(p, qs, [0], p.lens, 1, 2, 50))


def test_select_infinities_nan_and_huge_scores():
    p = ref.Pool(33, [16 * 90] * 4, 4, 2, 64, FP32, FP32, values=False)
    t = p.tables
    p.bounds[t[0, 10], :, 1, 3] = np.nan
    p.bounds[t[0, 50], :, 0, 4] = np.nan
    p.bounds[t[0, 60], :, 1] = np.inf
    p.bounds[t[1, 5:40], :, 0] = -np.inf
    p.bounds[t[2]] *= np.float32(1e30)
    qs = p.queries(4)
    qs[0, :, :] = np.abs(qs[0]) + 0.1   # no zero times infinity
    qs[1, :, :] = np.abs(qs[1]) + 0.1   # -inf meets a zero weight: NaN
    qs[2] *= np.float32(1e8)            # products past fp32's largest
    qs[3, :2, 0] = np.nan
    g = {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [None] * 4}
    got = run_select(p, g, qs, None, p.lens, 1, 2, 20)
    with np.errstate(invalid="ignore"):
        np.testing.assert_array_equal(got, ref.select(p, qs, range(4), p.lens, 1, 2, 20))


@pytest.mark.parametrize("kv", [FP32, BF16, INT8])
def test_select_many_queries_in_any_order(kv):
    """More queries than sequences, of each sequence anywhere in the list, past one look at the list."""
    p = ref.Pool(36 + kv, [16 * 40 + 5, 16 * 25, 16 * 300 + 1, 0, 16 * 12], 8, 2, 64, kv, values=False)
    rng = np.random.default_rng(3)
    rows = rng.integers(-1, 6, 150).tolist()
    lens = [int(rng.integers(0, 16 * 300 + 2)) if 0 <= s < 5 and s == 2 else int(rng.integers(0, 700)) for s in rows]
    lens = [min(t, int(p.lens[s])) if 0 <= s < 5 else t for s, t in zip(rows, lens)]
    qs = p.queries(150)
    g = {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [to_gpu(s) for s in p.stats] if p.stats else [None] * 4}
    np.testing.assert_array_equal(run_select(p, g, qs, rows, lens, 1, 2, 8), ref.select(p, qs, rows, lens, 1, 2, 8))


def test_select_int8_weights_of_any_size():
    """Weights far apart within a query, zeros, and values that are not finite (their scores are NaN: the lowest indices)."""
    p = ref.Pool(39, [16 * 90] * 5, 8, 2, 64, INT8, FP32, values=False)
    qs = p.queries(5)
    qs[0] *= np.float32(1e-30)
    qs[1, :, ::2] *= np.float32(1e6)
    qs[2] = 0
    qs[3, 0, 3] = np.inf
    qs[4, 5, 1] = np.nan
    g = {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [to_gpu(s) for s in p.stats]}
    got = run_select(p, g, qs, None, p.lens, 1, 2, 20)
    want = ref.select(p, np.nan_to_num(qs, nan=np.float32(np.nan), posinf=np.float32(np.nan)), range(5), p.lens, 1, 2, 20)
    np.testing.assert_array_equal(got, want)


def test_select_ignores_bounds_of_the_recent_blocks_and_reads_no_bad_page():
    p = ref.Pool(34, [16 * 60 - 5, 16 * 60], 8, 2, 64, BF16, values=False)
    p.bounds[p.tables[0, 58:]] = 0x7fc0  # not brought up to date: NaN
    p.tables[1, 7], p.tables[1, 20], p.tables[1, 21] = -1, p.nb, 2 ** 31 - 1
    g = {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [None] * 4}
    qs = p.queries(2)
    np.testing.assert_array_equal(run_select(p, g, qs, None, p.lens, 0, 2, 16), ref.select(p, qs, [0, 1], p.lens, 0, 2, 16))


def test_select_several_queries_of_a_sequence():
    p = ref.Pool(35, [16 * 70, 16 * 33 + 4, 16 * 9], 16, 2, 128, BF16, values=False)
    rows = [0, 0, 0, 1, 1, 2, 2, 2, 2, 2, 0, -1, 3, 1]
    lens = [16 * 70 - 2, 16 * 70 - 1, 16 * 70, 16 * 33 + 3, 16 * 33 + 4, 1, 40, 100, 143, 144, 300, 500, 500, 0]
    qs = p.queries(len(rows))
    g = {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [None] * 4}
    got = run_select(p, g, qs, rows, lens, 1, 2, 8)
    np.testing.assert_array_equal(got, ref.select(p, qs, rows, lens, 1, 2, 8))
    # the bound of the context lengths and the table's width cut the contexts
    got = run_select(p, g, qs, rows, [10 ** 6] * len(rows), 1, 2, 8, max_len=900)
    np.testing.assert_array_equal(got, ref.select(p, qs, rows, [10 ** 6] * len(rows), 1, 2, 8, max_len=900))


@pytest.mark.parametrize("kv,q", [(FP32, FP32), (BF16, BF16), (BF16, FP32), (INT8, BF16), (INT8, FP32), (FP32, BF16)])
@pytest.mark.parametrize("hq,hkv,d", [s for s in SHAPES if s[0] != 12])
def test_sparse_decode(kv, q, hq, hkv, d):
    if kv == INT8 and d == 32:
        pytest.skip("int8 caches take head_dim 64 and more")
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 100, 16 * 30 + 7, 16 * 40, 0]
    p = ref.Pool(40 + kv, lens, hq, hkv, d, kv, q)
    qs, rows, g = p.queries(len(lens)), range(len(lens)), gpu_pool(p)
    for budget in (1, 3, 24, 45):
        sel = random_lists(p, rows, lens, budget, p.rng)
        want, tol = ref.attend(p, qs, rows, lens, sel)
        close(run_sparse(p, g, qs, None, lens, sel), want, tol, f"budget {budget}")


@pytest.mark.parametrize("n,budget", [(1, 64), (1, 600), (1, 1300), (3, 130), (40, 33), (90, 20), (50, 77), (700, 9), (129, 64), (190, 24)])
@pytest.mark.parametrize("kv", [BF16, INT8])
def test_sparse_decode_splits(kv, n, budget):
    """Few rows of long lists, in parts, and many rows in one: the same attention."""
    lens = [16 * (budget + 5) - 3 * i for i in range(n)]
    p = ref.Pool(45, lens, 8, 2, 64, kv, BF16)
    qs, g = p.queries(n), gpu_pool(p)
    sel = random_lists(p, range(n), lens, budget, p.rng)
    want, tol = ref.attend(p, qs, range(n), lens, sel)
    close(run_sparse(p, g, qs, None, lens, sel), want, tol)


@pytest.mark.parametrize("n,budget", [(3, 130), (20, 70), (90, 20), (260, 11)])
@pytest.mark.parametrize("kv,hq,hkv,d", [(FP32, 8, 2, 32), (FP32, 8, 2, 64), (INT8, 16, 1, 64), (BF16, 32, 2, 128), (FP32, 8, 2, 128),
                                         (INT8, 8, 2, 128), (FP32, 8, 2, 256), (BF16, 16, 2, 256), (INT8, 16, 1, 256)])
def test_sparse_decode_splits_of_other_shapes(kv, hq, hkv, d, n, budget):
    """Workgroups of four and of eight waves, one or two to a CU: cut rows, whole ones, several whole ones."""
    lens = [16 * (budget + 2) - 3 * (i % 40) for i in range(n)]
    p = ref.Pool(46, lens, hq, hkv, d, kv, FP32)
    qs, g = p.queries(n), gpu_pool(p)
    sel = random_lists(p, range(n), lens, budget, p.rng)
    want, tol = ref.attend(p, qs, range(n), lens, sel)
    close(run_sparse(p, g, qs, None, lens, sel), want, tol)


@pytest.mark.parametrize("kv", [FP32, BF16, INT8])
def test_sparse_decode_lists_of_the_callers(kv):
    """Entries in any order, holes, blocks past the context, the same block twice, nothing at all, bad pages."""
    p = ref.Pool(46, [200, 200, 77, 200, 40], 8, 2, 128, kv, BF16)
    sel = np.full((5, 2, 40), -1, np.int32)
    sel[0, 0, :6] = [9, 2, 12, 0, 7, 3]
    sel[0, 1, 30:40:3] = [11, -5, 13, 4]
    sel[1, 0, :4] = [5, 5, 5, 6]
    sel[1, 1] = [1000000, 2 ** 31 - 1, -2 ** 31] + [-1] * 37
    sel[2, :, :8] = np.arange(8)
    sel[3, :, ::2] = 3
    p.tables[2, 1], p.tables[2, 2], p.tables[3, 3] = -1, p.nb, p.nb + 7
    qs, g, lens = p.queries(5), gpu_pool(p), [200, 200, 77, 200, 40]
    want, tol = ref.attend(p, qs, range(5), lens, sel)
    got = run_sparse(p, g, qs, None, lens, sel)
    close(got, want, tol)
    assert (got[1, 4:] == 0).all() and (got[4] == 0).all() and (got[3] == 0).all()


@pytest.mark.parametrize("kv", [FP32, BF16])
def test_sparse_decode_unused_slots_may_hold_anything(kv):
    lens = [1, 6, 19, 30, 47]
    p = ref.Pool(47, lens, 8, 2, 64, kv, BF16)
    inf, nan = (ref.of_type(np.float32(x).reshape(1), kv)[0] for x in (np.inf, np.nan))
    sel = np.tile(np.arange(4, dtype=np.int32), (5, 2, 1))
    qs = p.queries(5)
    want, tol = ref.attend(p, qs, range(5), lens, sel)  # before the slots are spoilt
    for s, t in enumerate(lens):
        b = p.tables[s, (t - 1) // 16]
        p.k[b, :, (t - 1) % 16 + 1:], p.v[b, :, :, (t - 1) % 16 + 1:] = nan, inf
    close(run_sparse(p, gpu_pool(p), qs, None, lens, sel), want, tol)


def test_sparse_decode_infinite_keys():
    """Scores of -inf count nothing beside finite ones; a row with nothing else, and one with +inf or NaN, is not a number."""
    p = ref.Pool(48, [16 * 20] * 4, 2, 2, 64, FP32, FP32)
    qs = np.abs(p.queries(4)) + np.float32(0.1)
    sel = np.tile(np.arange(20, dtype=np.int32), (4, 2, 1))
    want, tol = ref.attend(p, qs, [0], [320], np.sort(sel[:1, :, 3:]))
    p.k[p.tables[0, :3]] = -np.inf
    p.k[p.tables[1]] = -np.inf
    p.k[p.tables[2, 4], :, 2, 0] = np.inf
    p.k[p.tables[3, 4], :, 2, 0] = np.nan
    got = run_sparse(p, gpu_pool(p), qs, None, [320] * 4, sel)
    close(got[:1], want, tol)
    assert np.isnan(got[1:]).all()


@pytest.mark.parametrize("kv", [FP32, BF16])
@pytest.mark.parametrize("budget", [20, 600])
def test_sparse_decode_nan_in_a_block_of_its_own(kv, budget):
    """A single token with a NaN key, alone in its block, and so alone with the wave or the part that has the block: its query's
    outputs are NaN whatever the others are; beside it the rows stay as they were."""
    lens = [16 * (budget - 1) + 1] * 3
    p = ref.Pool(54, lens, 4, 2, 64, kv, BF16)
    qs = p.queries(3)
    sel = np.tile(np.arange(budget, dtype=np.int32), (3, 2, 1))
    clean = run_sparse(p, gpu_pool(p), qs, None, lens, sel)
    p.k[p.tables[1, budget - 1], 0, 0] = ref.of_type(np.full(1, np.nan, np.float32), kv)[0]
    got = run_sparse(p, gpu_pool(p), qs, None, lens, sel)
    assert np.isnan(got[1, :2]).all()
    np.testing.assert_array_equal(got[[0, 2]], clean[[0, 2]])
    np.testing.assert_array_equal(got[1, 2:], clean[1, 2:])


def test_sparse_decode_large_scores_and_scale():
    lens = [400, 77, 640]
    p = ref.Pool(49, lens, 8, 2, 64, BF16, FP32)
    p.cfg.scale = 3.0
    qs, g = p.queries(3) * np.float32(4), gpu_pool(p)
    sel = random_lists(p, range(3), lens, 30, p.rng)
    want, tol = ref.attend(p, qs, range(3), lens, sel)
    close(run_sparse(p, g, qs, None, lens, sel), want, tol)


def test_sparse_decode_several_queries_of_a_sequence():
    p = ref.Pool(50, [16 * 70, 16 * 33 + 4, 16 * 9], 8, 2, 128, BF16, BF16)
    rows = [0, 0, 0, 1, 1, 2, 2, -1, 3, 1]
    lens = [16 * 70 - 2, 16 * 70 - 1, 16 * 70, 16 * 33 + 3, 16 * 33 + 4, 1, 144, 500, 500, 0]
    qs, g = p.queries(len(rows)), gpu_pool(p)
    sel = random_lists(p, rows, lens, 20, p.rng)
    sel[7:9] = np.arange(20)
    want, tol = ref.attend(p, qs, rows, lens, sel)
    close(run_sparse(p, g, qs, rows, lens, sel), want, tol)
    want, tol = ref.attend(p, qs, rows, [10 ** 6] * 10, sel, max_len=555)
    close(run_sparse(p, g, qs, rows, [10 ** 6] * 10, sel, max_len=555), want, tol)


@pytest.mark.parametrize("kv", [BF16, INT8])
def test_no_sequences_and_empty_contexts(kv):
    """Queries whose sequence does not exist (none does, or theirs does not): nothing selected, zeros attended."""
    p = ref.Pool(52, [16 * 30], 8, 2, 64, kv)
    qs, g = p.queries(3), gpu_pool(p)
    for seqs, rows in ((0, [0, 0, 0]), (1, [1, -1, 7])):
        q, p.tables = p.tables, p.tables[:seqs] if seqs else p.tables[:0]
        sel = run_select(p, g, qs, rows, [480, 480, 480], 1, 2, 9)
        out = run_sparse(p, g, qs, rows, [480, 480, 480], np.tile(np.arange(9, dtype=np.int32), (3, 2, 1)))
        p.tables = q
        assert (sel == -1).all() and (out == 0).all()


@pytest.mark.parametrize("kv,hkv,d,nb", [(BF16, 8, 128, 150000), (FP32, 8, 256, 36000), (INT8, 8, 256, 140000)])
def test_blocks_past_four_gigabytes(kv, hkv, d, nb):
    """The same blocks at the far end of a pool whose keys pass 4 GiB (and whose bounds, for fp32, do not): the same bits."""
    import torch
    lens = [16 * 20 + 3, 16 * 9]
    p = ref.Pool(53, lens, hkv, hkv, d, kv, BF16)
    qs, g = p.queries(2), gpu_pool(p)
    near = [run_bounds(p, g, [0, 0], lens), run_select(p, g, qs, None, lens, 1, 2, 8)]
    near.append(run_sparse(p, g, qs, None, lens, near[1]))
    dt = {FP32: torch.float32, BF16: torch.int16, INT8: torch.int8}[kv]
    far = {"k": torch.empty(nb, hkv, 16, d, dtype=dt, device="cuda:0"), "v": torch.empty(nb, hkv, d, 16, dtype=dt, device="cuda:0"),
           "bounds": torch.empty(nb, hkv, 2, d, dtype=dt, device="cuda:0")}
    assert far["k"].numel() * far["k"].element_size() > 1 << 32
    shift = nb - p.nb
    for name in ("k", "v", "bounds"):
        far[name][shift - 100:shift - 100 + p.nb] = g[name]  # (bounds are as key_bounds_update left them)
    far["stats"] = [torch.zeros(nb, hkv, device="cuda:0") if s is not None else None for s in g["stats"]]
    for a, b in zip(far["stats"], g["stats"]):
        if a is not None:
            a[shift - 100:shift - 100 + p.nb] = b
    # copied page by page to the very end, then everything done there
    small, p.cfg.num_blocks = p.nb, nb
    pairs = to_gpu(np.stack([np.arange(small) + shift - 100, np.arange(small) + shift], 1).astype(np.int32))
    pa.copy_pages(None, p.cfg, far["k"], far["v"], *far["stats"], far["bounds"], pairs, small)
    p.tables = np.where(p.tables >= 0, p.tables + shift, -1).astype(np.int32)
    far["tables"] = to_gpu(p.tables)
    far["bounds"][shift:] = 0
    pa.key_bounds_update(None, p.cfg, far["k"], far["tables"], p.width, to_gpu(np.zeros(2, np.int32)), to_gpu(p.lens), 2, max(lens),
                         far["bounds"])
    torch.cuda.synchronize()
    moved = to_np(far["bounds"][shift:], ref.NP_DTYPE[kv])
    used = np.unique(p.tables[p.tables >= 0]) - shift
    np.testing.assert_array_equal(moved[used], near[0][used])
    np.testing.assert_array_equal(run_select(p, far, qs, None, lens, 1, 2, 8), near[1])
    np.testing.assert_array_equal(run_sparse(p, far, qs, None, lens, near[1]), near[2])


def test_all_blocks_selected_is_the_dense_decode():
    import torch
    lens = [5, 300, 1024, 77]
    p = ref.Pool(51, lens, 32, 8, 128, BF16, BF16)
    qs, g = p.queries(4), gpu_pool(p)
    sel = run_select(p, g, qs, None, lens, 1, 2, 64)
    got = run_sparse(p, g, qs, None, lens, sel)
    out = empty_gpu((4, 32, 128), np.float32)
    size = pa.decode_workspace_size(p.cfg, 4, 1024)
    ws = empty_gpu((size,), np.uint8)
    pa.paged_decode(None, p.cfg, out, to_gpu(qs), g["k"], g["v"], None, None, g["tables"], to_gpu(p.lens), 4, p.width, 1024, ws, size)
    torch.cuda.synchronize()
    # the dense decode keeps 16 bits of a probability: 2^-16 of it, over values of 4 at most
    np.testing.assert_allclose(to_np(out), got, atol=2.0 ** -16 * 4, rtol=0)


@pytest.mark.parametrize("kv", [FP32, BF16, INT8])
def test_decode_steps_append_bounds_select_attend(kv):
    """Steps of a batch as a program runs them, captured once and replayed: the new token is appended, its block's bounds
    brought up to date, blocks selected and attended; every replay against the 64-bit forms and against an eager run."""
    import torch
    S, hq, hkv, d, budget, steps = 5, 8, 2, 64, 7, 4
    begin = [14, 100, 16 * 20 - 1, 16 * 31, 250]
    p = ref.Pool(60 + kv, [t + steps for t in begin], hq, hkv, d, kv, FP32)
    g = gpu_pool(p)
    dev = pa.Device(0)
    st = pa.Stream(dev)
    run_bounds(p, g, [0] * S, begin)
    most = int(p.lens.max())
    bufs = dict(q=empty_gpu((S, hq, d), np.float32), kn=empty_gpu((S, hkv, d), np.float32), vn=empty_gpu((S, hkv, d), np.float32),
                start=empty_gpu((S,), np.int32), lens=empty_gpu((S,), np.int32), one=to_gpu(np.ones(S, np.int32)),
                off=to_gpu(np.arange(S, dtype=np.int32)), slots=empty_gpu((S,), np.int64))
    n1, n2 = pa.select_workspace_size(p.cfg, S, most), pa.sparse_workspace_size(p.cfg, S, budget)
    ws1, ws2 = empty_gpu((max(8, n1),), np.uint8), empty_gpu((max(8, n2),), np.uint8)
    sel, out = empty_gpu((S, hkv, budget), np.int32), empty_gpu((S, hq, d), np.float32)

    def step(stream):
        b = bufs
        pa.build_slot_mapping(stream, p.cfg, g["tables"], p.width, b["start"], b["one"], b["off"], S, 1, b["slots"])
        pa.kv_append(stream, p.cfg, b["kn"], b["vn"], b["slots"], S, g["k"], g["v"], *g["stats"])
        pa.key_bounds_update(stream, p.cfg, g["k"], g["tables"], p.width, b["start"], b["one"], S, 1, g["bounds"])
        pa.select_blocks(stream, p.cfg, b["q"], g["bounds"], g["stats"][0], g["tables"], S, p.width, None, b["lens"], S, most, 1, 2,
                         budget, sel, ws1, n1)
        pa.sparse_decode(stream, p.cfg, out, b["q"], g["k"], g["v"], g["stats"][0], g["stats"][1], g["tables"], S, p.width, None,
                         b["lens"], S, most, sel, budget, ws2, n2)

    torch.cuda.synchronize()
    graph = pa.Graph().capture(st)
    step(st)
    graph.end()
    assert graph.node_count() >= 5
    for k in range(steps):
        pos = np.array(begin, np.int32) + k
        x = [p.rng.standard_normal(s, np.float32) for s in ((S, hq, d), (S, hkv, d), (S, hkv, d))]
        for name, a in zip(("q", "kn", "vn"), x):
            bufs[name].copy_(to_gpu(a))
        bufs["start"].copy_(to_gpu(pos))
        bufs["lens"].copy_(to_gpu(pos + 1))
        sel.fill_(-9)
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.launch(st)
        st.synchronize()
        got_sel, got_out = to_np(sel).copy(), to_np(out).copy()
        # what the replay left in the cache is where the 64-bit forms start from
        p.k, p.v = to_np(g["k"], ref.NP_DTYPE[kv]).copy(), to_np(g["v"], ref.NP_DTYPE[kv]).copy()
        if p.stats:
            p.stats = [to_np(s).copy() for s in g["stats"]]
        p.bounds = ref.key_bounds(p, [0] * S, pos + 1)
        np.testing.assert_array_equal(got_sel, ref.select(p, x[0], range(S), pos + 1, 1, 2, budget))
        want, tol = ref.attend(p, x[0], range(S), pos + 1, got_sel)
        close(got_out, want, tol, f"step {k}")
        junk = torch.randn(1 << 20, device="cuda:0").sum()  # the program's own work between replays
        torch.cuda.synchronize()
        del junk
    graph.destroy()
    st.destroy()
    dev.close()


def test_two_streams_at_once():
    """Two decode steps on two streams, each with its own workspaces: what they give alone."""
    import torch
    lens = [16 * 150 + 3] * 6
    p = ref.Pool(70, lens, 8, 2, 128, BF16, BF16)
    g = gpu_pool(p)
    run_bounds(p, g, [0] * 6, lens)
    dev = pa.Device(0)
    streams = [pa.Stream(dev), pa.Stream(dev)]
    qs = [p.queries(6), p.queries(6)]
    alone = []
    for q in qs:
        sel = run_select(p, g, q, None, lens, 1, 2, 48)
        alone.append((sel, run_sparse(p, g, q, None, lens, sel)))
    gq, glens = [to_gpu(q) for q in qs], to_gpu(p.lens)
    n1, n2 = pa.select_workspace_size(p.cfg, 6, lens[0]), pa.sparse_workspace_size(p.cfg, 6, 48)
    mem = [(empty_gpu((6, 2, 48), np.int32), empty_gpu((6, 8, 128), np.float32), empty_gpu((n1,), np.uint8),
            empty_gpu((max(8, n2),), np.uint8)) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, q, (sel, out, w1, w2) in zip(streams, gq, mem):
            pa.select_blocks(s, p.cfg, q, g["bounds"], None, g["tables"], 6, p.width, None, glens, 6, lens[0], 1, 2, 48, sel, w1, n1)
            pa.sparse_decode(s, p.cfg, out, q, g["k"], g["v"], None, None, g["tables"], 6, p.width, None, glens, 6, lens[0], sel,
                             48, w2, n2)
    for s, (sel, out, _, _), (want_sel, want) in zip(streams, mem, alone):
        s.synchronize()
        np.testing.assert_array_equal(to_np(sel), want_sel)
        np.testing.assert_array_equal(to_np(out), want)
        s.destroy()
    dev.close()
