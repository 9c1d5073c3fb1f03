"""Plain 64-bit forms of the operators for caches of bounded size (attention over a window and sinks, block masses, eviction),
written from their definitions in include/paged_attn.h. numpy only; inputs are longctx_ref's pools.

Tolerances, from fp32 sums of products. A score is a sum of D products whose magnitudes add to at most S (scaled): each
addition rounds by at most 2^-24 of a partial sum no larger than S, the roundings have no common sign, so their sum is taken
as 4 sqrt(D) 2^-24 S. Where an operand is fp32, products are formed of bf16 parts and those of parts below 2^-24 are left out,
at most four of them a product: 2^-22 S. exp of the score adds 2^-22 (its argument's rounding near the maximum, and its own).
That is `e`. A probability is off by twice that with its normalisation; the T additions of P V and of the sum add 4 sqrt(T) 2^-24, each relative to the largest |v|."""
import numpy as np

from longctx_ref import BLOCK, f64

EPS = 2.0 ** -24


def seen(pos, t, sink, window):
    """Which of the tokens t the query at position pos sees."""
    t = np.asarray(t)
    return (t <= pos) & ((t > pos - window) | (t < sink) if window else True)


def context(p, s, length, max_len=None):
    """(keys, values) [hkv, T, d] of a row's tokens; zeros for blocks that are none."""
    t = max(0, min(int(length), p.width * BLOCK, int(length) if max_len is None else int(max_len)))
    n = (t + BLOCK - 1) // BLOCK
    ids = p.tables[s, :n]
    ok = (ids >= 0) & (ids < p.nb)
    at = np.where(ok, ids, 0)
    k = f64(p.k[at]) * p.scale_of(0)[at][:, :, None, None] * ok[:, None, None, None]
    v = f64(p.v[at]) * p.scale_of(1)[at][:, :, None, None] * ok[:, None, None, None]
    k = np.where(ok[:, None, None, None], k, 0).transpose(1, 0, 2, 3).reshape(p.hkv, n * BLOCK, p.d)
    v = np.where(ok[:, None, None, None], v, 0).transpose(1, 0, 3, 2).reshape(p.hkv, n * BLOCK, p.d)
    return k[:, :t], v[:, :t]


def attend(p, q, rows, positions, sink, window, lens, max_len=None):
    """Query r of row rows[r] at position positions[r], in a context of lens[r] tokens. (out, tolerance, lse, its
    tolerance, weights per row and block [len(tables), width], their tolerance)"""
    n, g = len(rows), p.hq // p.hkv
    scale = p.cfg.scale if p.cfg.scale > 0 else 1 / np.sqrt(p.d)
    out, tol = np.zeros((n, p.hq, p.d)), np.zeros((n, p.hq, 1))
    lse, lse_tol = np.full((n, p.hq), -np.inf), np.zeros((n, p.hq))
    mass, mass_tol = np.zeros(p.tables.shape), np.zeros(p.tables.shape)
    qv, kept = f64(q), {}
    for r, (s, pos) in enumerate(zip(rows, positions)):
        key = (s, lens[r])
        if key not in kept:
            kept[key] = context(p, s, lens[r], max_len)
        k, v = kept[key]
        vis = np.nonzero(seen(pos, np.arange(k.shape[1]), sink, window))[0]
        if not len(vis):
            continue
        for h in range(p.hq):
            kk, vv = k[h // g][vis], v[h // g][vis]
            x = kk @ qv[r, h] * scale
            with np.errstate(invalid="ignore", over="ignore"):
                w = np.exp(x - x.max())
                total = w.sum()
                out[r, h], lse[r, h] = w @ vv / total, x.max() + np.log(total)
            S = (np.abs(kk) @ np.abs(qv[r, h])).max() * scale
            e = (4 * np.sqrt(p.d) * EPS + (4 * EPS if p.kv == 0 or p.q == 0 else 0)) * S + 4 * EPS
            t = 2 * e + 4 * np.sqrt(len(vis)) * EPS
            tol[r, h] = t * np.abs(vv).max()
            # in log2 units and back: three roundings of a value of that size
            lse_tol[r, h] = e + 4 * np.sqrt(len(vis)) * EPS + 4 * EPS * (1 + abs(lse[r, h]) + np.abs(x).max())
            b = np.bincount(vis // BLOCK, w / total, minlength=p.width)
            mass[s] += b
            mass_tol[s] += b * (t + 4 * EPS * (1 + np.abs(x).max()))
    # a row's sum over n queries and their heads: as many additions again
    mass_tol += mass * 4 * np.sqrt(n * p.hq) * EPS
    return out, tol, lse, lse_tol, mass, mass_tol


def decode(p, q, lens, sink, window, max_len=None):
    cut = [max(0, min(int(t), p.width * BLOCK, int(t) if max_len is None else max_len)) for t in lens]
    return attend(p, q, range(len(lens)), [t - 1 for t in cut], sink, window, cut)


def chunk_rows(lens, chunks):
    rows = [s for s, n in enumerate(chunks) for _ in range(n)]
    return rows, [t - n + i for t, n in zip(lens, chunks) for i in range(n)]


def prompt_mass(p, q, lse, lens, chunks, last, sink, window, max_len=None):
    """(what is added to the masses [rows, width], tolerance): weights by a given lse."""
    rows, positions = chunk_rows(lens, chunks)
    start = np.concatenate([[0], np.cumsum(chunks)])
    g = p.hq // p.hkv
    scale = p.cfg.scale if p.cfg.scale > 0 else 1 / np.sqrt(p.d)
    mass, tol = np.zeros(p.tables.shape), np.zeros(p.tables.shape)
    qv, n = f64(q), 0
    for s in range(len(lens)):
        k, _ = context(p, s, lens[s], max_len)
        for r in range(start[s + 1] - min(last, chunks[s]), start[s + 1]):
            vis = np.nonzero(seen(positions[r], np.arange(k.shape[1]), sink, window))[0]
            n += 1
            for h in range(p.hq if len(vis) else 0):
                x = k[h // g][vis] @ qv[r, h] * scale
                b = np.bincount(vis // BLOCK, np.exp(x - float(lse[r, h])), minlength=p.width)
                S = (np.abs(k[h // g][vis]) @ np.abs(qv[r, h])).max() * scale
                e = (4 * np.sqrt(p.d) * EPS + (4 * EPS if p.kv == 0 or p.q == 0 else 0)) * S + 4 * EPS
                mass[s] += b
                tol[s] += b * (e + 4 * EPS * (1 + abs(float(lse[r, h])) + np.abs(x).max()))
    return mass, tol + mass * 4 * np.sqrt(16 * max(1, n) * p.hq) * EPS


def evict(tables, lens, mass, sink, recent, budget, refs):
    """(tables, lens, masses, reference counts, evicted), one row and one block at a time."""
    tables, lens, refs = tables.copy(), lens.copy(), refs.copy()
    mass = None if mass is None else mass.copy()
    width, gone = tables.shape[1], np.zeros(len(lens), np.int32)
    for i in range(len(lens)):
        n = min((int(lens[i]) + BLOCK - 1) // BLOCK, width) if lens[i] > 0 else 0
        if n <= budget:
            continue
        may = list(range(sink, n - recent))
        if mass is None:
            may.sort(key=lambda b: -b)
        else:
            may.sort(key=lambda b: (0, 0, b) if np.isnan(mass[i, b]) else (1, -mass[i, b], b))
        out = set(may[budget - sink - recent:])
        stay = [b for b in range(width) if b not in out]
        for b in out:
            if 0 <= tables[i, b] < len(refs):
                refs[tables[i, b]] -= 1
        tables[i] = np.concatenate([tables[i, stay], np.full(len(out), -1)])
        if mass is not None:
            mass[i] = np.concatenate([mass[i, stay], np.zeros(len(out))])
        lens[i] -= BLOCK * len(out)
        gone[i] = len(out)
    return tables, lens, mass, refs, gone
