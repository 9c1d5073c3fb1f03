"""What the long-context operators refuse, on the host: no call here launches anything."""
import pytest

import paged_attention as pa

FAKE = 0x1000  # never dereferenced


def cfg(**kw):
    base = dict(num_q_heads=32, num_kv_heads=8, head_dim=128, kv_dtype=pa.PA_DTYPE_BF16, q_dtype=pa.PA_DTYPE_BF16,
                num_blocks=100)
    base.update(kw)
    return pa.make_config(**base)


ARG, CONFIG, UNSUP, SMALL = (pa.PA_ERROR_INVALID_ARGUMENT, pa.PA_ERROR_INVALID_CONFIG, pa.PA_ERROR_UNSUPPORTED,
                             pa.PA_ERROR_WORKSPACE_TOO_SMALL)


def refused(status, text, f):
    with pytest.raises(pa.PagedAttentionError) as e:
        f()
    assert e.value.status == status and text in str(e.value), str(e.value)


def bounds(c=None, k=FAKE, tables=FAKE, width=9, start=FAKE, new=FAKE, seqs=4, most=5, out=FAKE):
    pa.key_bounds_update(None, c or cfg(), k, tables, width, start, new, seqs, most, out)


@pytest.mark.parametrize("status,text,kw", [
    (UNSUP, "block_size", dict(c=cfg(block_size=8))),
    (ARG, "negative", dict(seqs=-1)), (ARG, "negative", dict(most=-1)), (ARG, "negative", dict(width=-1)),
    (UNSUP, "65535", dict(seqs=65536)),
    (UNSUP, "too many", dict(c=cfg(num_q_heads=1 << 20, num_kv_heads=1 << 20), most=1 << 30, width=1 << 27)),
    (ARG, "null", dict(k=None)), (ARG, "null", dict(tables=None)), (ARG, "null", dict(start=None)),
    (ARG, "null", dict(new=None)), (ARG, "null", dict(out=None)),
    (ARG, "aligned", dict(k=FAKE + 8)), (ARG, "aligned", dict(out=FAKE + 2)),
])
def test_key_bounds(status, text, kw):
    refused(status, text, lambda: bounds(**kw))


def select(c=None, q=FAKE, b=FAKE, ks=None, tables=FAKE, seqs=4, width=300, rows=None, lens=FAKE, n=4, most=4096, sink=1,
           recent=2, budget=32, out=FAKE, ws=FAKE, size=1 << 40):
    pa.select_blocks(None, c or cfg(), q, b, ks, tables, seqs, width, rows, lens, n, most, sink, recent, budget, out, ws, size)


@pytest.mark.parametrize("status,text,kw", [
    (UNSUP, "head_dim", dict(c=cfg(head_dim=96))),
    (ARG, "negative", dict(seqs=-1)), (ARG, "negative", dict(n=-1)), (ARG, "negative", dict(most=-1)),
    (UNSUP, "max_context_len", dict(most=2097153)), (UNSUP, "too many", dict(n=1 << 22, rows=FAKE)),
    (ARG, "sink_blocks", dict(sink=-1)), (ARG, "recent_blocks", dict(recent=0)),
    (ARG, "budget", dict(budget=0)), (ARG, "budget", dict(sink=30, recent=3)),
    (ARG, "budget", dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1)),
    (ARG, "null", dict(q=None)), (ARG, "null", dict(b=None)), (ARG, "null", dict(tables=None)),
    (ARG, "null", dict(lens=None)), (ARG, "null", dict(out=None)), (ARG, "query_seqs", dict(n=5)),
    (ARG, "k_scale", dict(c=cfg(kv_dtype=2))), (ARG, "aligned", dict(b=FAKE + 8)),
    (ARG, "aligned", dict(q=FAKE + 8)), (CONFIG, "num_blocks", dict(c=cfg(num_blocks=0))),
    (SMALL, "workspace", dict(size=4 * 8 * 256 * 8 - 1)), (SMALL, "workspace", dict(ws=None)), (ARG, "aligned", dict(ws=FAKE + 4)),
])
def test_select(status, text, kw):
    refused(status, text, lambda: select(**kw))


def sparse(c=None, out=FAKE, q=FAKE, k=FAKE, v=FAKE, ks=None, vs=None, tables=FAKE, seqs=4, width=300, rows=None, lens=FAKE, n=4,
           most=4096, sel=FAKE, budget=64, ws=FAKE, size=1 << 40):
    pa.sparse_decode(None, c or cfg(), out, q, k, v, ks, vs, tables, seqs, width, rows, lens, n, most, sel, budget, ws, size)


@pytest.mark.parametrize("status,text,kw", [
    (CONFIG, "multiple", dict(c=cfg(num_q_heads=12))), (UNSUP, "num_q_heads", dict(c=cfg(num_q_heads=24))),
    (UNSUP, "num_q_heads", dict(c=cfg(num_q_heads=256))),
    (ARG, "negative", dict(n=-1)), (ARG, "negative", dict(budget=-1)), (ARG, "negative", dict(most=-1)),
    (ARG, "negative", dict(seqs=-1)), (ARG, "negative", dict(width=-1)),
    (UNSUP, "32 bits", dict(width=1 << 28)), (UNSUP, "too many", dict(n=1 << 24, rows=FAKE)),
    (ARG, "budget", dict(budget=0)), (ARG, "null", dict(out=None)), (ARG, "null", dict(q=None)), (ARG, "null", dict(k=None)),
    (ARG, "null", dict(v=None)), (ARG, "null", dict(tables=None)), (ARG, "null", dict(lens=None)), (ARG, "null", dict(sel=None)),
    (ARG, "query_seqs", dict(n=5)), (ARG, "v_scale", dict(c=cfg(kv_dtype=2), ks=FAKE)), (ARG, "aligned", dict(v=FAKE + 8)),
    (ARG, "aligned", dict(q=FAKE + 4)),
    (SMALL, "workspace", dict(size=0)), (SMALL, "workspace", dict(ws=None)), (ARG, "aligned", dict(ws=FAKE + 2)),
])
def test_sparse_decode(status, text, kw):
    refused(status, text, lambda: sparse(**kw))


def fork(c=None, tin=0x10000, lin=0x20000, n_in=4, src=0x30000, tout=0x40000, lout=0x50000, n_out=4, width=9, refs=FAKE):
    pa.pages_fork(None, c or cfg(), tin, lin, n_in, src, tout, lout, n_out, width, refs)


@pytest.mark.parametrize("status,text,kw", [
    (ARG, "negative", dict(n_in=-1)), (ARG, "negative", dict(n_out=-1)), (ARG, "negative", dict(width=-1)),
    (UNSUP, "too many", dict(n_in=2 ** 31 - 1)), (ARG, "null", dict(refs=None)), (ARG, "null", dict(src=None)),
    (ARG, "null", dict(tin=None)), (ARG, "null", dict(tout=None)), (ARG, "null", dict(lin=None)), (ARG, "null", dict(lout=None)),
    (ARG, "overlap", dict(tout=0x10000)), (ARG, "overlap", dict(tout=0x10000 + 4 * 4 * 9 - 4)),
    (ARG, "overlap", dict(lout=0x20000)), (ARG, "overlap", dict(src=0x50000)), (ARG, "overlap", dict(src=0x40004)),
])
def test_fork(status, text, kw):
    refused(status, text, lambda: fork(**kw))


def reserve(c=None, t=FAKE, lens=FAKE, new=FAKE, rows=4, width=9, most=1, refs=FAKE, pairs=FAKE, st=FAKE, ws=FAKE, size=1 << 30):
    pa.pages_reserve(None, c or cfg(), t, lens, new, rows, width, most, refs, pairs, st, ws, size)


@pytest.mark.parametrize("status,text,kw", [
    (ARG, "negative", dict(rows=-1)), (ARG, "negative", dict(width=-1)), (ARG, "negative", dict(most=-1)),
    (ARG, "status", dict(st=None)), (ARG, "null", dict(t=None)), (ARG, "null", dict(lens=None)), (ARG, "null", dict(new=None)),
    (ARG, "null", dict(refs=None)), (ARG, "null", dict(pairs=None)),
    (UNSUP, "too many", dict(rows=1 << 20, width=1 << 20, most=1 << 20)),
    (SMALL, "workspace", dict(size=99)), (SMALL, "workspace", dict(ws=None)), (ARG, "aligned", dict(ws=FAKE + 2)),
])
def test_reserve(status, text, kw):
    refused(status, text, lambda: reserve(**kw))


def compact(c=None, t=FAKE, rows=4, width=9, refs=FAKE, most=5, pairs=FAKE, st=FAKE, ws=FAKE, size=1 << 30):
    pa.pages_compact(None, c or cfg(), t, rows, width, refs, most, pairs, st, ws, size)


@pytest.mark.parametrize("status,text,kw", [
    (ARG, "negative", dict(rows=-1)), (ARG, "negative", dict(width=-1)), (ARG, "negative", dict(most=-1)),
    (ARG, "null", dict(st=None)), (ARG, "null", dict(refs=None)), (ARG, "null", dict(pairs=None)), (ARG, "null", dict(t=None)),
    (SMALL, "workspace", dict(size=99)), (SMALL, "workspace", dict(ws=None)), (ARG, "aligned", dict(ws=FAKE + 2)),
])
def test_compact(status, text, kw):
    refused(status, text, lambda: compact(**kw))


def copy(c=None, k=FAKE, v=FAKE, stats=(None,) * 4, b=None, pairs=FAKE, most=3, num=None):
    pa.copy_pages(None, c or cfg(), k, v, *stats, b, pairs, most, num)


@pytest.mark.parametrize("status,text,kw", [
    (ARG, "max_pairs", dict(most=-1)), (ARG, "null", dict(k=None)), (ARG, "null", dict(v=None)), (ARG, "pairs", dict(pairs=None)),
    (ARG, "aligned", dict(k=FAKE + 8)), (ARG, "aligned", dict(b=FAKE + 8)), (ARG, "int8", dict(c=cfg(kv_dtype=2))),
    (ARG, "int8", dict(c=cfg(kv_dtype=2), stats=(FAKE, FAKE, FAKE, None))),
])
def test_copy(status, text, kw):
    refused(status, text, lambda: copy(**kw))


def test_sizes_and_empty_calls():
    assert pa.key_bounds_bytes(cfg()) == 100 * 8 * 2 * 128 * 2
    assert pa.key_bounds_bytes(cfg(kv_dtype=2)) == 100 * 8 * 2 * 128
    assert pa.select_workspace_size(cfg(), 3, 100) == 3 * 8 * 7 * 8
    assert pa.select_workspace_size(cfg(), 0, 100) == 0
    assert pa.sparse_workspace_size(cfg(), 0, 100) == 0
    assert pa.sparse_workspace_size(cfg(), 1, 512) > 0


@pytest.mark.parametrize("c", [cfg(), cfg(num_q_heads=16, num_kv_heads=1, head_dim=256), cfg(head_dim=64), cfg(head_dim=64, kv_dtype=2),
                               cfg(head_dim=256, kv_dtype=0)])
def test_sparse_workspace_serves_smaller_calls(c):
    """One workspace of the largest call's size is enough for every smaller call: a call reports what it needs itself."""
    for n, budget in ((512, 64), (40, 130), (7, 300)):
        size = pa.sparse_workspace_size(c, n, budget)
        assert size <= 16 << 20
        for m in (1, 2, 3, 5, 7, 16, 17, 31, 40, 64, 65, 100, 129, 200, 257, 300, 511, 512):
            for b in (1, 2, 9, 16, 17, 33, 63, 64, 90, 129, 130, 299, 300):
                if m <= n and b <= budget:
                    assert pa.sparse_workspace_size(c, m, b) <= size
                    # (the alignment is checked behind the size)
                    refused(ARG, "aligned", lambda: sparse(c=c, ks=FAKE, vs=FAKE, n=m, rows=FAKE, budget=b, ws=FAKE + 2, size=size))
    bounds(seqs=0, k=None, tables=None, start=None, new=None, out=None)
    bounds(most=0)
    select(n=0, q=None, b=None, tables=None, lens=None, out=None)
    sparse(n=0, out=None, q=None, k=None, v=None, tables=None, lens=None, sel=None)
    fork(n_in=0, n_out=0, tin=None, lin=None, src=None, tout=None, lout=None, refs=None)
    copy(most=0, pairs=None)
