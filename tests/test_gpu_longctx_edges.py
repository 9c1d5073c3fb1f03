"""Calls at the edges of what the long-context operators and the page books accept, on the GPU against their 64-bit forms
(longctx_ref.py)."""
import numpy as np
import pytest

import longctx_ref as ref
import paged_attention as pa
from helpers import empty_gpu, to_gpu, to_np
from test_gpu_pages import run_compact
from test_gpu_sparse import close, gpu_pool, random_lists, run_select, run_sparse

pytestmark = pytest.mark.gpu

INT8, FP32 = 2, 0


def select_pool(p):
    return {"bounds": to_gpu(p.bounds), "tables": to_gpu(p.tables), "stats": [to_gpu(s) for s in p.stats] if p.stats else [None] * 4}


@pytest.mark.parametrize("queries", [1, 3])
def test_select_int8_codes_of_minus_128(queries):
    """Codes of -128 in all 512 places of a block's bounds at head_dim 256, against weights whose fourth digit (of base 256) is -128 in
    every place: the digit's sum over the places is 2^23, and a digit pair's 2^31. The weights are a = 1/2 - 2^-14 of the maxima and -b
    = -(1 + 2^-14) of the minima, so such a block has 128 * 256 (b - a), the best score, and a block with -127 for n of its channels
    n (b - a) less, all of them exact in 64 bits."""
    blocks = 120
    p = ref.Pool(71, [16 * blocks] * 2, 2, 1, 256, INT8, FP32, values=False)
    p.stats[0][:] = 0.03125
    p.bounds[:] = -128
    for i in range(2 * blocks):
        if i % 3:
            p.bounds[p.tables.ravel()[i], 0, :, :1 + (7 * i) % 15] = -127
    rows = [0, 1] * queries
    qs = np.empty((len(rows), 2, 256), np.float32)
    qs[:, 0], qs[:, 1] = 0.5 - 2.0 ** -14, -(1 + 2.0 ** -14)
    lens = [16 * blocks] * len(rows)
    want = ref.select(p, qs, rows, lens, 1, 2, 30)
    got = run_select(p, select_pool(p), qs, rows if queries > 1 else None, lens, 1, 2, 30)
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("kv", [FP32, 1, INT8])
def test_select_group_sums_past_the_largest_fp32(kv):
    """Finite queries whose sums over the heads of a group pass the largest fp32 value: ordinary scores in 64 bits."""
    p = ref.Pool(72 + kv, [16 * 90] * 3, 32, 2, 64, kv, FP32, values=False)
    qs = p.queries(3)
    qs[1] = np.clip(qs[1], -2, 2) * np.float32(1.5e38)
    qs[2, :16] = np.float32(3.4e38) * np.sign(qs[2, :16])
    with np.errstate(over="ignore"):
        assert np.isinf(np.maximum(qs[1], 0).reshape(2, 16, 64).sum(1, dtype=np.float32)).any() and np.isfinite(qs).all()
    got = run_select(p, select_pool(p), qs, None, p.lens, 1, 2, 20)
    np.testing.assert_array_equal(got, ref.select(p, qs, range(3), p.lens, 1, 2, 20))


@pytest.mark.parametrize("width,most", [(9, 1), (9, 1000), (9, 0), (0, 5)])
@pytest.mark.parametrize("null", [True, False])
def test_reserve_for_no_rows(null, width, most):
    """An empty batch, whose arrays may all be null: nothing taken, nothing missing, the books not looked at."""
    import torch
    cfg = pa.make_config(num_q_heads=2, num_kv_heads=2, head_dim=64, kv_dtype=1, num_blocks=100)
    refs, some, status = to_gpu(np.arange(100, dtype=np.int32) % 3), empty_gpu((8,), np.int32), empty_gpu((2,), np.int32)
    status.fill_(77)
    size = pa.pages_workspace_size(cfg, 0, width)
    ws = empty_gpu((size,), np.uint8)
    given = (None,) * 5 if null else (some, some, some, refs, some)
    pa.pages_reserve(None, cfg, *given[:3], 0, width, most, *given[3:], status, ws, size)
    torch.cuda.synchronize()
    assert to_np(status).tolist() == [0, 0]
    np.testing.assert_array_equal(to_np(refs), np.arange(100) % 3)


@pytest.mark.parametrize("live", [262144, 262145, 262144 + 64 * 100 + 17, 2 * 262144 - 1, 2 * 262144, 2 * 262144 + 4095])
def test_compact_where_the_rounds_words_differ(live):
    """Pools of several rounds of 262144 blocks whose words around the live count are full in one round and empty in the other, so
    that a word of the wrong round would give another number of moves."""
    config = pa.make_config(num_q_heads=2, num_kv_heads=2, head_dim=64, kv_dtype=1, num_blocks=3 * 262144 + 5)
    nb = config.num_blocks
    held = np.ones(nb, bool)
    at = live % 262144  # the word that is read, and the same one of every other round
    for r in range(4):
        lo = max(0, r * 262144 + at - 200)
        held[lo:r * 262144 + at + 200] = r != live // 262144
    spare = np.nonzero(held)[0]
    held[spare[spare > live + 300][::-1][:held.sum() - live]] = False
    extra = np.nonzero(held)[0][::7][:held.sum() - live]
    held[extra] = False
    assert held.sum() == live
    refs = held.astype(np.int32) * 2
    ids = np.nonzero(held)[0].astype(np.int32)
    tables = np.full((1, live + 3), -1, np.int32)
    tables[0, :live] = ids
    t, r, pairs, st = run_compact(config, tables, refs, nb)
    up, down = ids[ids >= live][::-1], np.nonzero(~held[:live])[0]
    assert len(up) == len(down)
    name = np.arange(nb, dtype=np.int32)
    name[up] = down
    np.testing.assert_array_equal(pairs[:len(up)], np.stack([up, down], 1))
    assert (pairs[len(up):] == -1).all()
    np.testing.assert_array_equal(r, (np.arange(nb) < live) * 2)
    np.testing.assert_array_equal(t[0, :live], name[ids])
    assert (t[0, live:] == -1).all() and st.tolist() == [len(up), live]


@pytest.mark.parametrize("kv", [1, INT8])
def test_step_in_a_graph_whose_reservation_fails(kv):
    """Fork, reservation, copies and append in one graph. Where too few blocks are free the step's slots are -1 (its start positions are
    made negative by status) and its lengths stay, so no byte of the cache, no count and no length changes behind the fork;
    the next replay, which forks every row to itself, repeats the reservation alone, and succeeds once a block is free."""
    import torch
    B, hkv, d, width, nb = 4, 2, 64, 4, 12
    rng = np.random.default_rng(80 + kv)
    cfg = pa.make_config(num_q_heads=hkv, num_kv_heads=hkv, head_dim=d, kv_dtype=kv, q_dtype=FP32, num_blocks=nb)
    k, v, bounds = (to_gpu(ref.of_type(rng.standard_normal(s, np.float32), kv)) for s in ((nb, hkv, 16, d), (nb, hkv, d, 16), (nb, hkv, 2, d)))
    stats = [to_gpu(np.full((nb, hkv), x, np.float32)) for x in (0.03, 0.04, 0.03 * 127, 0.04 * 127)] if kv == INT8 else [None] * 4
    first = np.full((B, width), -1, np.int32)
    first[0, :2], first[1, :2], first[2, 0] = (7, 3), (1, 9), 5  # 20, 32 and 5 tokens
    tables = [to_gpu(first), empty_gpu((B, width), np.int32)]
    lens = [to_gpu(np.array([20, 32, 5, 0], np.int32)), empty_gpu((B,), np.int32)]
    held = np.ones(nb, np.int32)
    held[11] = 0  # one block is free, the others that no row holds are a prefix cache's
    refs, src = to_gpu(held), to_gpu(np.array([0, 0, 1, 2], np.int32))
    one, off = to_gpu(np.ones(B, np.int32)), to_gpu(np.arange(B, dtype=np.int32))
    pairs, status, slots = empty_gpu((B, 2), np.int32), empty_gpu((2,), np.int32), empty_gpu((B,), np.int64)
    size = pa.pages_workspace_size(cfg, B, width)
    ws, start, granted = empty_gpu((size,), np.uint8), empty_gpu((B,), np.int32), empty_gpu((B,), np.int32)
    none, ok = to_gpu(np.full(B, -2 ** 31, np.int32)), torch.zeros(1, dtype=torch.bool, device="cuda:0")
    kn, vn = empty_gpu((B, hkv, d), np.float32), empty_gpu((B, hkv, d), np.float32)
    dev = pa.Device(0)
    ts = pa.Stream(dev)
    tstream = torch.cuda.ExternalStream(ts.native(), device="cuda:0")

    def gate(b):
        with torch.cuda.stream(tstream):
            torch.eq(status[1:], 0, out=ok)
            torch.where(ok, lens[b], none, out=start)
            torch.mul(one, ok, out=granted)

    def step(a, b):
        pa.pages_fork(ts, cfg, tables[a], lens[a], B, src, tables[b], lens[b], B, width, refs)
        pa.pages_reserve(ts, cfg, tables[b], lens[b], one, B, width, 1, refs, pairs, status, ws, size)
        pa.copy_pages(ts, cfg, k, v, *stats, bounds, pairs, B)
        gate(b)
        pa.build_slot_mapping(ts, cfg, tables[b], width, start, one, off, B, 1, slots)
        pa.kv_append(ts, cfg, kn, vn, slots, B, k, v, *stats)
        pa.key_bounds_update(ts, cfg, k, tables[b], width, start, one, B, 1, bounds)
        with torch.cuda.stream(tstream):
            lens[b].add_(granted)

    torch.cuda.synchronize()
    gate(1)
    lens[1].add_(granted)  # (loaded before a capture)
    torch.cuda.synchronize()
    graphs = []
    for a, b in ((0, 1), (1, 0)):
        gr = pa.Graph().capture(ts)
        step(a, b)
        graphs.append(gr.end())
    data = [t for t in (k, v, bounds, *stats) if t is not None]
    short = np.array([[7, 3, -1, -1], [7, 3, -1, -1], [1, 9, -1, -1], [5, -1, -1, -1]], np.int32)  # behind the fork
    held[[7, 3]] = 2
    for n in range(5):
        x = [rng.standard_normal((B, hkv, d), np.float32) for _ in range(2)]
        kn.copy_(to_gpu(x[0]))
        vn.copy_(to_gpu(x[1]))
        if n == 1:
            src.copy_(off)  # every row to itself
        if n == 3:
            refs[10] = 0  # the prefix cache gives a block back
            held[10] = 0
        before = [to_np(t).copy() for t in data]
        torch.cuda.synchronize()
        graphs[n % 2].launch(ts)
        ts.synchronize()
        now = (n + 1) % 2
        if n < 3:  # rows 0 (a copy of the tail it shares) and 2 (a new block) ask for one each
            assert to_np(status).tolist() == [0, 1] and (to_np(pairs) == -1).all() and (to_np(slots) == -1).all()
            for t, was in zip(data, before):
                np.testing.assert_array_equal(to_np(t), was)
            np.testing.assert_array_equal(to_np(tables[now]), short)
            np.testing.assert_array_equal(to_np(refs), held)
            assert to_np(lens[now]).tolist() == [20, 20, 32, 5]
        junk = torch.randn(1 << 20, device="cuda:0").sum()  # the program's own work between replays
        torch.cuda.synchronize()
        del junk
        if n < 3:
            continue
        at = [20 + n - 3, 20 + n - 3, 32 + n - 3, 5 + n - 3]
        if n == 3:
            assert to_np(status).tolist() == [2, 0] and to_np(pairs).tolist() == [[3, 10]] + [[-1, -1]] * 3
            short[0, 1], short[2, 2] = 10, 11
            held[[3, 10, 11]] = 1
            if kv == 1:  # the tail's four tokens went along
                np.testing.assert_array_equal(to_np(k)[10, :, :4], before[0][3, :, :4])
                np.testing.assert_array_equal(to_np(v)[10, :, :, :4], before[1][3, :, :, :4])
        np.testing.assert_array_equal(to_np(tables[now]), short)
        np.testing.assert_array_equal(to_np(refs), held)
        assert to_np(lens[now]).tolist() == [t + 1 for t in at]
        for i, t in enumerate(at):
            b = short[i, t // 16]
            for which, (cache, new) in enumerate(((k, x[0][i]), (v, x[1][i]))):
                got = to_np(cache, ref.NP_DTYPE[kv])[b]
                got = got[:, t % 16] if which == 0 else got[:, :, t % 16]
                if kv == 1:  # the upper 16 bits, as pa_kv_append stores them
                    np.testing.assert_array_equal(got, ref.bf16_of(new))
                else:  # a code is off by half a step, its product with the scale and the division by 2^-22 of the value
                    sc = to_np(stats[which])[b][:, None].astype(np.float64)
                    assert (np.abs(ref.f64(got) * sc - new) <= 0.5 * sc + np.abs(new) * 2.0 ** -22).all()
    for gr in graphs:
        gr.destroy()
    ts.destroy()
    dev.close()


@pytest.mark.parametrize("far", [4, 16, 20, 24])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (32, 8, 128), (8, 1, 128), (16, 1, 256)])
def test_sparse_decode_int8_queries_far_apart(hq, hkv, d, far):
    """One channel of a query 2^far times the others, and its codes zero: the others decide.

    Tolerance: that of the exact products, and the queries' rounding: 2^-30 of the largest value in every channel, all of one
    sign at worst, makes e = 2^-30 max|q| sum_d |k_d| scale of a score and twice that of a probability."""
    lens = [100, 16 * 30 + 7, 16 * 12]
    p = ref.Pool(90 + far, lens, hq, hkv, d, INT8, FP32)
    p.k[:, :, :, 5] = 0
    qs = p.queries(3)
    qs[:, :, 5] = 2.0 ** far
    sel = random_lists(p, range(3), lens, 24, p.rng)
    want, tol = ref.attend(p, qs, range(3), lens, sel)
    k = np.abs(ref.f64(p.k)).sum(3).max() * p.stats[0].max()
    v = np.abs(ref.f64(p.v)).max() * p.stats[1].max()
    tol = tol + 2 * 2.0 ** -30 * np.abs(qs).max(2, keepdims=True) * k / np.sqrt(d) * v
    close(run_sparse(p, gpu_pool(p), qs, None, lens, sel), want, tol)
