"""Calls of the operators for bounded caches that are refused on the host, before anything is launched; sizes of their
workspaces. No GPU."""
import re

import pytest

import paged_attention as pa

FAKE = 0x1000  # 16-byte aligned, never dereferenced: every call below is refused
INVALID, CONFIG, UNSUPPORTED, WORKSPACE = 1, 2, 5, 6


def cfg(**kw):
    base = dict(num_q_heads=8, num_kv_heads=2, head_dim=64, kv_dtype=pa.PA_DTYPE_BF16, q_dtype=pa.PA_DTYPE_BF16, num_blocks=100)
    return pa.make_config(**{**base, **kw})


def refused(fn, status, text, *args):
    with pytest.raises(pa.PagedAttentionError) as e:
        fn(None, *args)
    assert e.value.status == status and text in str(e.value), str(e.value)


def decode(c=None, out=FAKE, q=FAKE, k=FAKE, v=FAKE, ks=None, vs=None, tables=FAKE, lens=FAKE, n=3, width=8, most=100, sink=4,
           window=32, mass=None, ws=FAKE, size=1 << 30):
    return (c or cfg(), out, q, k, v, ks, vs, tables, lens, n, width, most, sink, window, mass, ws, size)


@pytest.mark.parametrize("status,text,kw", [
    (INVALID, "null", dict(out=None)), (INVALID, "null", dict(q=None)), (INVALID, "null", dict(k=None)),
    (INVALID, "null", dict(v=None)), (INVALID, "null", dict(tables=None)), (INVALID, "null", dict(lens=None)),
    (INVALID, "negative size", dict(n=-1)), (INVALID, "negative size", dict(width=-1)), (INVALID, "negative size", dict(most=-1)),
    (INVALID, "must not be negative", dict(sink=-1)), (INVALID, "must not be negative", dict(window=-1)),
    (INVALID, "aligned", dict(q=FAKE + 8)), (INVALID, "aligned", dict(k=FAKE + 4)), (INVALID, "aligned", dict(v=FAKE + 2)),
    (INVALID, "8-byte", dict(ws=FAKE + 4)), (INVALID, "k_scale", dict(c=cfg(kv_dtype=2))), (WORKSPACE, "needs", dict(size=8)),
    (WORKSPACE, "needs", dict(ws=None)), (UNSUPPORTED, "1, 2, 4, 8 or 16", dict(c=cfg(num_q_heads=6))),
    (UNSUPPORTED, "1, 2, 4, 8 or 16", dict(c=cfg(num_q_heads=64))), (UNSUPPORTED, "32 bits", dict(width=1 << 27)),
    (UNSUPPORTED, "too many blocks", dict(n=2000, most=2 ** 31 - 1, window=0)), (CONFIG, "multiple", dict(c=cfg(num_q_heads=7))),
    (UNSUPPORTED, "head_dim", dict(c=cfg(head_dim=96))), (UNSUPPORTED, "int8", dict(c=cfg(head_dim=32, kv_dtype=2)))])
def test_window_decode(status, text, kw):
    refused(pa.window_decode, status, text, *decode(**kw))


def prefill(c=None, out=FAKE, q=FAKE, start=FAKE, prefix=FAKE, k=FAKE, v=FAKE, ks=None, vs=None, tables=FAKE, n=1, width=80, chunk=4,
            most=1000, sink=4, window=0, lse=None, ws=FAKE, size=1 << 30):
    return (c or cfg(), out, q, start, prefix, k, v, ks, vs, tables, n, width, chunk, most, sink, window, lse, ws, size)


@pytest.mark.parametrize("status,text,kw", [
    (INVALID, "null", dict(out=None)), (INVALID, "null", dict(q=None)), (INVALID, "null", dict(start=None)),
    (INVALID, "null", dict(prefix=None)), (INVALID, "null", dict(k=None)), (INVALID, "null", dict(v=None)),
    (INVALID, "null", dict(tables=None)), (INVALID, "negative size", dict(n=-1)), (INVALID, "negative size", dict(width=-1)),
    (INVALID, "negative size", dict(chunk=-1)), (INVALID, "negative size", dict(most=-1)),
    (INVALID, "must not be negative", dict(sink=-1)), (INVALID, "must not be negative", dict(window=-5)),
    (INVALID, "aligned", dict(out=FAKE + 4)), (INVALID, "aligned", dict(q=FAKE + 8)), (INVALID, "aligned", dict(k=FAKE + 8)),
    (INVALID, "k_scale", dict(c=cfg(kv_dtype=2))), (INVALID, "16-byte", dict(ws=FAKE + 8)), (WORKSPACE, "needs", dict(size=8)),
    (WORKSPACE, "needs", dict(ws=None)), (UNSUPPORTED, "65535", dict(n=40000)), (UNSUPPORTED, "32 bits", dict(chunk=2 ** 30)),
    (UNSUPPORTED, "32 bits", dict(width=1 << 27)), (UNSUPPORTED, "too many", dict(n=30000, chunk=2 ** 20))])
def test_window_prefill(status, text, kw):
    refused(pa.window_prefill, status, text, *prefill(**kw))


def mass(c=None, q=FAKE, lse=FAKE, start=FAKE, prefix=FAKE, k=FAKE, ks=None, tables=FAKE, n=1, width=80, most=1000, last=8, sink=4,
         window=0, out=FAKE):
    return (c or cfg(), q, lse, start, prefix, k, ks, tables, n, width, most, last, sink, window, out)


@pytest.mark.parametrize("status,text,kw", [
    (INVALID, "null", dict(q=None)), (INVALID, "null", dict(lse=None)), (INVALID, "null", dict(start=None)),
    (INVALID, "null", dict(prefix=None)), (INVALID, "null", dict(k=None)), (INVALID, "null", dict(tables=None)),
    (INVALID, "null", dict(out=None)), (INVALID, "negative size", dict(n=-1)), (INVALID, "negative size", dict(last=-1)),
    (INVALID, "negative size", dict(width=-1)), (INVALID, "negative size", dict(most=-1)),
    (INVALID, "must not be negative", dict(sink=-1)), (INVALID, "must not be negative", dict(window=-1)),
    (INVALID, "k_scale", dict(c=cfg(kv_dtype=2))), (INVALID, "aligned", dict(q=FAKE + 8)), (INVALID, "aligned", dict(k=FAKE + 8)),
    (UNSUPPORTED, "65535", dict(n=65536)), (UNSUPPORTED, "32 bits", dict(width=1 << 27)),
    (UNSUPPORTED, "30 bits", dict(last=2 ** 27)),
    (UNSUPPORTED, "2^20", dict(c=cfg(num_q_heads=2 ** 22, num_kv_heads=2))), (UNSUPPORTED, "too many blocks", dict(most=2 ** 31 - 1, width=2 ** 27 - 1))])
def test_prefill_mass(status, text, kw):
    refused(pa.prefill_mass, status, text, *mass(**kw))


def evict(c=None, tables=FAKE, lens=FAKE, out=FAKE, n=3, width=8, sink=1, recent=1, budget=4, refs=FAKE, gone=None):
    return (c or cfg(), tables, lens, out, n, width, sink, recent, budget, refs, gone)


@pytest.mark.parametrize("status,text,kw", [
    (INVALID, "null", dict(tables=None)), (INVALID, "null", dict(lens=None)), (INVALID, "null", dict(refs=None)),
    (INVALID, "negative size", dict(n=-1)), (INVALID, "negative size", dict(width=-1)), (INVALID, "recent_blocks >= 1", dict(recent=0)),
    (INVALID, "sink_blocks", dict(sink=-1)), (INVALID, "<= budget", dict(budget=1)),
    (INVALID, "<= budget", dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1)), (UNSUPPORTED, "32 bits", dict(width=1 << 27)),
    (UNSUPPORTED, "too many rows", dict(n=2 ** 22))])
def test_evict_blocks(status, text, kw):
    refused(pa.evict_blocks, status, text, *evict(**kw))


def test_nothing_to_do_is_no_error():
    pa.window_decode(None, *decode(n=0, out=None, q=None, k=None, v=None, tables=None, lens=None, ws=None, size=0))
    pa.window_prefill(None, *prefill(n=0, out=None, ws=None, size=0))
    pa.window_prefill(None, *prefill(chunk=0, out=None, ws=None, size=0))
    pa.prefill_mass(None, *mass(n=0, q=None))
    pa.prefill_mass(None, *mass(last=0, q=None))
    pa.evict_blocks(None, *evict(n=0, tables=None))


@pytest.mark.parametrize("kv,d", [(0, 32), (1, 64), (1, 128), (2, 128), (0, 256), (1, 256)])
@pytest.mark.parametrize("with_mass", [False, True])
def test_a_decode_workspace_serves_smaller_calls(kv, d, with_mass):
    c = cfg(kv_dtype=kv, head_dim=d, q_dtype=0)
    for sink, window in ((0, 0), (4, 100), (100, 1), (0, 2 ** 31 - 1), (2 ** 31 - 1, 7)):
        last = 0
        for n, t in ((0, 0), (1, 1), (1, 17), (2, 300), (5, 300), (64, 4000), (300, 4000), (3000, 4000), (5000, 9000)):
            size = pa.window_decode_workspace_size(c, n, t, sink, window, with_mass)
            assert size >= last
            last = size
            if n:  # a byte less is refused
                refused(pa.window_decode, WORKSPACE, "needs",
                        *decode(c, ks=FAKE, vs=FAKE, n=n, width=1000, most=t, sink=sink, window=window,
                                mass=FAKE if with_mass else None, size=size - 1))


def test_a_prefill_workspace_serves_smaller_calls():
    for kv, d in ((0, 32), (1, 64), (2, 128), (0, 128), (1, 256), (0, 256)):
        for hq, hkv in ((8, 2), (3, 3), (32, 2), (20, 4)):
            c = cfg(kv_dtype=kv, head_dim=d, num_q_heads=hq, num_kv_heads=hkv)
            size = pa.window_prefill_workspace_size(c, 1, 1, 17, 0, 0)
            assert size == pa.window_prefill_workspace_size(c, 5, 4000, 100000, 3, 0) > 0
            # what a call whose keys are cut asks for is within it
            for n, chunk, most, window in ((1, 1, 100000, 0), (1, 30, 100000, 0), (2, 5, 20000, 4000), (1, 4, 100000, 0)):
                with pytest.raises(pa.PagedAttentionError) as e:
                    pa.window_prefill(None, *prefill(c, ks=FAKE, vs=FAKE, n=n, width=8000, chunk=chunk, most=most, window=window, ws=None,
                                                     size=0, lse=FAKE))
                assert e.value.status == WORKSPACE
                assert 0 < int(re.search(r"needs (\d+) bytes", str(e.value)).group(1)) <= size
