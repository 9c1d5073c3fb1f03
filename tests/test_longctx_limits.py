"""Calls of the long-context operators and the page books that no launch can hold: refused on the host before anything is launched.
(HIP takes fewer than 2^32 threads along a grid's dimension.)"""
import pytest

import paged_attention as pa
from test_longctx_refusals import UNSUP, bounds, cfg, copy, fork, refused, select, sparse

FAKE, FAR = 0x1000, 1 << 40  # never dereferenced


def test_key_bounds():
    # 2^23 blocks of 8 heads, 4 to a workgroup of 256 threads
    refused(UNSUP, "too many", lambda: bounds(width=1 << 23, most=(1 << 27) + 16))


@pytest.mark.parametrize("kw", [
    dict(n=1 << 19, width=1025, most=1025 * 16),  # 2^22 rows of 1024 threads
    dict(n=1 << 20, width=1024, most=1024 * 16),  # 2^23 of 512
    dict(n=1 << 20, width=8, most=1024 * 16),
    # as many sequences as queries: the scores go by query
    dict(n=1 << 12, seqs=1 << 12, width=1 << 17, most=1 << 21),  # scores: 2^27 waves
    dict(n=1 << 13, seqs=1 << 13, width=1 << 17, most=1 << 21, c=cfg(kv_dtype=pa.PA_DTYPE_INT8), ks=FAKE),  # 2^26 waves
    dict(n=1 << 13, seqs=1 << 13, width=1 << 17, most=1 << 21, c=cfg(kv_dtype=pa.PA_DTYPE_FP32)),
])
def test_select(kw):
    refused(UNSUP, "too many", lambda: select(rows=FAKE, size=1 << 60, **kw))


def test_select_of_several_queries_a_sequence():
    # more queries than sequences: the scores go by sequence, 2^13 of them
    refused(UNSUP, "too many", lambda: select(n=(1 << 13) + 1, seqs=1 << 13, rows=FAKE, width=1 << 17, most=1 << 21, size=1 << 60,
                                              c=cfg(kv_dtype=pa.PA_DTYPE_INT8), ks=FAKE))


def test_sparse_decode():
    # the rows that are cut are joined by a wave per (row, query head)
    refused(UNSUP, "too many", lambda: sparse(c=cfg(num_q_heads=16, num_kv_heads=1), n=(1 << 22) + 1, seqs=1, rows=FAKE, budget=500))


@pytest.mark.parametrize("n_in,n_out", [((1 << 24) - 4, 4), (4, (1 << 24) - 4), (1 << 23, 1 << 23)])
def test_fork(n_in, n_out):
    refused(UNSUP, "too many", lambda: fork(n_in=n_in, n_out=n_out, width=0, lin=FAR, src=2 * FAR, lout=3 * FAR))


def test_empty_calls():
    """No query, no pair, no row, no new token: nothing to do, whatever the arrays are."""
    bounds(seqs=0, k=None, tables=None, start=None, new=None, out=None)
    bounds(most=0)
    bounds(width=0)
    select(n=0, q=None, b=None, tables=None, lens=None, out=None)
    sparse(n=0, out=None, q=None, k=None, v=None, tables=None, lens=None, sel=None)
    fork(n_in=0, n_out=0, tin=None, lin=None, src=None, tout=None, lout=None, refs=None)
    copy(most=0, pairs=None)
