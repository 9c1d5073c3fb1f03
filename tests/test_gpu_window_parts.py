"""What fp32 operands in bf16 parts leave out of a product, in the attention of chunks and the masses of prompts over fp32 caches with fp32
queries: less than 2^-22 of it."""
import numpy as np
import pytest

import bounded_ref as bref
import longctx_ref as ref
from test_gpu_window import gpu_pool, run_mass, run_prefill

pytestmark = pytest.mark.gpu

# Just below a multiple of 2^-7 (2^-8, 2^-9) above 1: parts that are cut off leave two full lower ones, of whose products 2^-21 (2^-23,
# 2^-25) would be missing. With one factor's parts rounded (1 + 2^-7, -2^-23, 0 for the first, 1, 2^-8, -2^-23 for the second, and so on)
# what is left out is at most 2^-8 (2^-15 - 2^-23) + 2^-23 2^-7, less than 2^-23 + 2^-29 of the product.
LOW = [1 + 2.0 ** -7 - 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -23, 1 + 2.0 ** -9 - 2.0 ** -23, 1.5 + 2.0 ** -7 - 2.0 ** -23]
PAIRS = [(sx * x, y) for x in LOW for y in LOW for sx in (1, -1)]


def pool(d, at, grow):
    """A sequence of one token a pair, whose query and key are 0 but for one dimension."""
    p = ref.Pool(800, [1] * len(PAIRS), 1, 1, d, 0, 0)
    p.cfg.scale = float(np.float32(np.log(2.0)))
    qs = np.zeros((len(PAIRS), 1, d), np.float32)
    p.k[:] = 0
    for s, (x, y) in enumerate(PAIRS):
        qs[s, 0, at] = grow * x
        p.k[p.tables[s, 0], 0, 0, at] = y
        assert float(qs[s, 0, at]) == grow * x and float(p.k[p.tables[s, 0], 0, 0, at]) == y
    return p, qs


@pytest.mark.parametrize("d,at", [(32, 0), (64, 21), (128, 127), (256, 200)])
@pytest.mark.parametrize("bound", [1, 20000])
def test_scores_of_chunks(d, at, bound):
    """One token's lse is its score. Off it is by what is left out of its product (2 2^-24, see LOW), by the additions of the parts' products,
    of which the last three have bits below 2^-23 (the second parts', the third ones' of either factor), and by the way back from log2 units
    (the scale times log2 e is 1): 6 2^-24. (bound: waves that share columns, that own them.)"""
    p, qs = pool(d, at, 1)
    n = len(PAIRS)
    _, lse = run_prefill(p, gpu_pool(p), qs, [1] * n, [1] * n, 0, 0, max_chunk=bound)
    want = np.array([p.cfg.scale * x * y for x, y in PAIRS])
    off = np.abs(lse[:, 0] - want) / np.abs(want)
    assert off.max() <= (6 + 2.0 ** -4) * bref.EPS, f"off by {off.max() / bref.EPS:.2f} 2^-24"


@pytest.mark.parametrize("d,at", [(32, 0), (64, 21), (128, 127), (256, 200)])
def test_masses_of_prompts(d, at):
    """Scores of 2^5 times the products, which are off by 5 2^-24 of their size (as above); exp makes that relative. The given logarithm is
    multiplied by a rounded log2 e and rounded again (1.5 2^-24 of its size in log2 units); the difference, exp2 and the sum add 4 2^-24."""
    p, qs = pool(d, at, 32)
    n = len(PAIRS)
    score = np.array([p.cfg.scale * 32 * x * y for x, y in PAIRS])
    lse = np.ascontiguousarray(score[:, None] - 0.25, np.float32)
    zero = np.zeros(p.tables.shape, np.float32)
    got = run_mass(p, gpu_pool(p), qs, lse, [1] * n, [1] * n, 1, 0, 0, zero)[:, 0]
    want = np.exp(score - lse[:, 0].astype(np.float64))
    rel = np.abs(got - want) / want
    tol = (np.abs(score) * (1.5 + 5) + 4) * bref.EPS
    assert (rel <= tol).all(), f"off by {(rel / bref.EPS).max():.1f} 2^-24"


@pytest.mark.parametrize("q", [0, 1])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("bound", [40, 9000])
def test_queries_that_see_one_token_give_its_value(q, d, bound):
    """A window of one token: its weight p is 1 but for the rounding of its score, and out = p v / p: the six products of their parts are
    added up, divided and multiplied, 2^-24 each. (A part that is lost would show as 2^-8 or 2^-16.)"""
    lens, chunks = [200, 70, 33, 7], [40, 40, 33, 7]
    p = ref.Pool(810 + d, lens, 4, 2, d, 0, q)
    rows, at = bref.chunk_rows(lens, chunks)
    got, _ = run_prefill(p, gpu_pool(p), p.queries(len(rows)), lens, chunks, 0, 1, max_chunk=bound)
    want = np.stack([p.v[p.tables[s, t // 16], :, :, t % 16] for s, t in zip(rows, at)])
    want = np.repeat(want[:, :, None], 2, 2).astype(np.float64)
    off = np.abs(got.reshape(len(rows), 2, 2, d) - want) / np.abs(want)
    assert off.max() <= 8 * bref.EPS, f"off by {off.max() / bref.EPS:.1f} 2^-24"
