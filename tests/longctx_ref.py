"""Plain 64-bit forms of the long-context operators (key bounds, block selection, attention over selected blocks) and
of the page books, written from their definitions in include/paged_attn.h, and the inputs their tests share. numpy only."""
import numpy as np

import paged_attention as pa

BLOCK = 16
NP_DTYPE = {0: np.float32, 1: np.uint16, 2: np.int8}


def bf16_of(x):
    """fp32 -> bf16 bits, truncated."""
    return (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def f64_of_bf16(b):
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def f64(a):
    """An array of a cache or activation type as the values it holds (int8: codes)."""
    return f64_of_bf16(a) if a.dtype == np.uint16 else a.astype(np.float64)


def of_type(x, dtype):
    """fp32 values in a cache or activation type; int8: codes of 24 a unit."""
    if dtype == 1:
        return bf16_of(x)
    if dtype == 2:
        return np.clip(np.rint(x * 24), -127, 127).astype(np.int8)
    return np.ascontiguousarray(x, np.float32)


class Pool:
    """A pool of random blocks and the block tables of sequences of the given lengths over it."""

    def __init__(self, seed, lens, hq=8, hkv=2, d=64, kv=1, q=1, extra=3, width=None, values=True):
        rng = self.rng = np.random.default_rng(seed)
        self.lens = np.array(lens, np.int32)
        need = [max(0, (int(t) + 15) // 16) for t in lens]
        self.nb = sum(need) + extra
        self.width = width or max(need + [1])
        self.hq, self.hkv, self.d, self.kv, self.q = hq, hkv, d, kv, q
        self.cfg = pa.make_config(num_q_heads=hq, num_kv_heads=hkv, head_dim=d, kv_dtype=kv, q_dtype=q, num_blocks=self.nb)
        ids = rng.permutation(self.nb).astype(np.int32)
        self.tables = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.tables[s, :n] = ids[at:at + n]
            at += n
        self.stats = None
        if kv == 2:
            sc = (rng.random((2, self.nb, hkv)) * 0.03 + 0.02).astype(np.float32)
            self.stats = [sc[0], sc[1], sc[0] * 127, sc[1] * 127]
        if values:
            self.k = of_type(rng.standard_normal((self.nb, hkv, BLOCK, d), np.float32), kv)
            self.v = of_type(rng.standard_normal((self.nb, hkv, d, BLOCK), np.float32), kv)
        self.bounds = of_type(np.sort(rng.standard_normal((self.nb, hkv, 2, d), np.float32), axis=2), kv)

    def queries(self, n):
        return of_type(self.rng.standard_normal((n, self.hq, self.d), np.float32), self.q)

    def scale_of(self, which):
        return self.stats[which].astype(np.float64) if self.stats else np.ones((self.nb, self.hkv))


def blocks_of(p, seq, length, max_len=None):
    """(blocks, tokens) of a context, cut at the table's width and at max_len."""
    if seq < 0 or seq >= len(p.tables):
        return 0, 0
    t = min(int(length), p.width * BLOCK, int(max_len) if max_len is not None else int(length))
    return ((t + 15) // 16, t) if t > 0 else (0, 0)


def key_bounds(p, start, num_new):
    """The bounds after key_bounds_update, in the cache's type."""
    out = p.bounds.copy()
    for s, (a, n) in enumerate(zip(start, num_new)):
        if a < 0 or n <= 0:
            continue
        for lb in range(a // 16, (a + n + 15) // 16):
            if lb >= p.width or not 0 <= p.tables[s, lb] < p.nb:
                continue
            b, held = p.tables[s, lb], min(16, a + n - lb * 16)
            k = p.k[b, :, :held]
            val = f64(k)
            nan = np.isnan(val).any(1)
            lo = np.take_along_axis(k, val.argmin(1)[:, None], 1)[:, 0]
            hi = np.take_along_axis(k, val.argmax(1)[:, None], 1)[:, 0]
            out[b, :, 0], out[b, :, 1] = lo, hi
            if nan.any():
                out[b, :, 0][nan] = out[b, :, 1][nan] = np.array(np.nan, np.float32) if p.kv == 0 else 0x7fc0
    return out


def select(p, q, seqs, lens, sink, recent, budget, max_len=None):
    got = np.full((len(lens), p.hkv, budget), -1, np.int32)
    bounds, ks, qv, g = f64(p.bounds), p.scale_of(0), f64(q), p.hq // p.hkv
    for r, (s, t) in enumerate(zip(seqs, lens)):
        n, _ = blocks_of(p, s, t, max_len)
        for h in range(p.hkv):
            if n <= budget:
                got[r, h, :n] = np.arange(n)
                continue
            score = np.zeros(n)
            for b in range(n):
                i = p.tables[s, b]
                if 0 <= i < p.nb:
                    x = qv[r, h * g:(h + 1) * g]
                    with np.errstate(invalid="ignore"):
                        up = np.where(np.isnan(x), np.nan, np.maximum(x, 0)).sum(0)
                        down = np.where(np.isnan(x), np.nan, np.minimum(x, 0)).sum(0)
                        score[b] = ks[i, h] * (up * bounds[i, h, 1] + down * bounds[i, h, 0]).sum()
            score[np.isnan(score)] = np.inf
            forced = list(range(sink)) + list(range(n - recent, n))
            rest = sorted(range(sink, n - recent), key=lambda b: (-score[b], b))
            got[r, h] = sorted(forced + rest[:budget - sink - recent])
    return got


def attend(p, q, seqs, lens, selected, max_len=None):
    """(output in 64 bits, tolerance for each value).

    Tolerance, from fp32 sums of exact products. A score is a sum of D products whose magnitudes add to at most S
    (scaled): each addition rounds by at most 2^-24 of a partial sum no larger than S, the roundings have no common
    sign, so their sum is taken as 4 sqrt(D) 2^-24 S. exp of it adds 2^-22 (its argument's rounding near the
    maximum, and its own). A probability is off by twice that with its normalisation, and the T additions of P V and of
    the sum by 4 sqrt(T) 2^-24, each relative to the largest |v|."""
    g = p.hq // p.hkv
    out = np.zeros((len(lens), p.hq, p.d))
    tol = np.zeros((len(lens), p.hq, 1))
    kall, vall, qv = f64(p.k), f64(p.v), f64(q)
    ks, vs = p.scale_of(0), p.scale_of(1)
    scale = p.cfg.scale if p.cfg.scale > 0 else 1 / np.sqrt(p.d)
    for r, (s, t) in enumerate(zip(seqs, lens)):
        n, t = blocks_of(p, s, t, max_len)
        for h in range(p.hkv):
            kk, vv = [], []
            for b in selected[r, h]:
                if b < 0 or b >= n:
                    continue
                i, m = p.tables[s, b], min(16, t - b * 16)
                ok = 0 <= i < p.nb
                kk.append(kall[i, h, :m] * ks[i, h] if ok else np.zeros((m, p.d)))
                vv.append(vall[i, h, :, :m].T * vs[i, h] if ok else np.zeros((m, p.d)))
            if not kk:
                continue
            k, v = np.concatenate(kk), np.concatenate(vv)
            for j in range(h * g, (h + 1) * g):
                x = k @ qv[r, j] * scale
                w = np.exp(x - x.max())
                out[r, j] = w @ v / w.sum()
                S = (np.abs(k) @ np.abs(qv[r, j])).max() * scale
                e = 4 * np.sqrt(p.d) * 2.0 ** -24 * S + 2.0 ** -22
                tol[r, j] = (2 * e + 4 * np.sqrt(len(k)) * 2.0 ** -24) * np.abs(v).max()
    return out, tol


# ---- the page books: one row, one block at a time -----------------------------------------------------
def fork(tables, lens, src, refs):
    refs = refs.copy()
    nb, width = len(refs), tables.shape[1]
    out, out_lens = np.full((len(src), width), -1, np.int32), np.zeros(len(src), np.int32)
    for row in tables:
        for b in row:
            if 0 <= b < nb:
                refs[b] -= 1
    for i, s in enumerate(src):
        if 0 <= s < len(tables):
            out[i], out_lens[i] = tables[s], lens[s]
            for b in tables[s]:
                if 0 <= b < nb:
                    refs[b] += 1
    return out, out_lens, refs


def reserve(tables, lens, num_new, refs):
    """(tables, refcounts, pairs, status)"""
    t, f = tables.copy(), refs.copy()
    nb, width = len(refs), tables.shape[1]
    pairs = np.full((len(lens), 2), -1, np.int32)
    taken = 0
    free = [b for b in range(nb) if refs[b] == 0]
    for i, (n, new) in enumerate(zip(lens, num_new)):
        if n < 0 or new <= 0:
            continue
        for lb in range(n // 16, (int(n) + int(new) - 1) // 16 + 1):
            if lb >= width:
                break
            b = t[i, lb]
            held = 0 <= b < nb
            if held and f[b] <= 1:
                continue
            taken += 1
            if taken > len(free):
                # only counted from here on
                if held:
                    f[b] -= 1
                continue
            new_b = free[taken - 1]
            if held:
                f[b] -= 1
                if lb * 16 < n:
                    pairs[i] = (b, new_b)
            f[new_b] = 1
            t[i, lb] = new_b
    if taken > len(free):
        return tables.copy(), refs.copy(), np.full((len(lens), 2), -1, np.int32), np.array([0, taken - len(free)], np.int32)
    return t, f, pairs, np.array([taken, 0], np.int32)


def compact(tables, refs, max_moves):
    """(tables, refcounts, pairs, status)"""
    t, f = tables.copy(), refs.copy()
    pairs = np.full((max_moves, 2), -1, np.int32)
    n = 0
    while n < max_moves:
        live, free = np.nonzero(f > 0)[0], np.nonzero(f == 0)[0]
        if not len(live) or not len(free) or free[0] > live[-1]:
            break
        a, b = live[-1], free[0]
        f[b], f[a] = f[a], 0
        t[t == a] = b
        pairs[n] = (a, b)
        n += 1
    live = np.nonzero(f > 0)[0]
    return t, f, pairs, np.array([n, live[-1] + 1 if len(live) else 0], np.int32)
