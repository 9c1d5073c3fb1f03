"""A model with a sliding window served from rows whose expired blocks have left: what its tokens see, against attention over the whole
text with the positions of the text. (A wrong window or budget over the row as it stands would agree with itself.)"""
import numpy as np
import pytest

import bounded_ref as bref
import longctx_ref as ref
import paged_attention as pa
from helpers import empty_gpu, to_gpu, to_np
from test_gpu_window import BF16, FP32, I32, close

pytestmark = pytest.mark.gpu

HQ, HKV, D = 8, 2, 64


class Text:
    """The queries, keys and values of a batch's tokens, in the types of the cache."""

    def __init__(self, seed, lens, kv):
        rng = np.random.default_rng(seed)
        most = max(lens)
        self.q, self.k, self.v = (ref.of_type(rng.standard_normal((len(lens), most, h, D), np.float32), kv) for h in (HQ, HKV, HKV))
        self.k64, self.v64, self.q64 = ref.f64(self.k), ref.f64(self.v), ref.f64(self.q)

    def attend(self, s, pos, sink, window, fp32):
        """(outputs [HQ, D], tolerance [HQ, 1]) of the token at pos; tolerances as bounded_ref derives them."""
        out, tol = np.zeros((HQ, D)), np.zeros((HQ, 1))
        vis = np.nonzero(bref.seen(pos, np.arange(pos + 1), sink, window))[0]
        for h in range(HQ):
            k, v = self.k64[s, vis, h // (HQ // HKV)], self.v64[s, vis, h // (HQ // HKV)]
            x = k @ self.q64[s, pos, h] / np.sqrt(D)
            w = np.exp(x - x.max())
            out[h] = w @ v / w.sum()
            size = (np.abs(k) @ np.abs(self.q64[s, pos, h])).max() / np.sqrt(D)
            e = (4 * np.sqrt(D) + 4 * fp32) * bref.EPS * size + 4 * bref.EPS
            tol[h] = (2 * e + 4 * np.sqrt(len(vis)) * bref.EPS) * np.abs(v).max()
        return out, tol


@pytest.mark.parametrize("kv", [BF16, FP32])
@pytest.mark.parametrize("sink,window", [(0, 5), (4, 17), (16, 64), (20, 100), (33, 16), (1, 1)])
@pytest.mark.parametrize("draft", [1, 5])
def test_rows_that_lost_their_expired_blocks(kv, sink, window, draft):
    """Prompts, then steps of one token or of several, every one behind an eviction to the budget that the window needs."""
    prompts, steps = [7, 150, 64, 301], 24
    B = len(prompts)
    lens = [t + steps * draft for t in prompts]
    text = Text(900 + kv, lens, kv)
    nb, width = sum((t + 15) // 16 for t in prompts) + 8 * B + 40, (max(prompts) + 15) // 16 + 16
    cfg = pa.make_config(num_q_heads=HQ, num_kv_heads=HKV, head_dim=D, kv_dtype=kv, q_dtype=kv, num_blocks=nb)
    kc, vc = (empty_gpu((nb, HKV, 16, D), np.float32 if kv == FP32 else np.uint16) for _ in range(2))
    kc.fill_(-1 if kv == BF16 else float("nan"))  # NaN in every place that no token has
    vc.fill_(-1 if kv == BF16 else float("nan"))
    tables, refs, held = to_gpu(np.full((B, width), -1, I32)), to_gpu(np.zeros(nb, I32)), to_gpu(np.zeros(B, I32))
    most_new = max(prompts)
    pairs, status = empty_gpu((B * (most_new // 16 + 2), 2), I32), empty_gpu((2,), I32)
    rs_b = pa.pages_workspace_size(cfg, B, width)
    rs = empty_gpu((max(rs_b, 16),), np.uint8)
    gone = empty_gpu((B,), I32)
    sink_blocks = (sink + 15) // 16
    budget = sink_blocks + window // 16 + 2

    at = np.zeros(B, int)  # tokens of the text so far
    left = 0
    for step in range(steps + 1):
        new = np.array(prompts if step == 0 else [draft] * B, I32)
        total = int(new.sum())
        off = np.concatenate([[0], np.cumsum(new)]).astype(I32)
        tokens = [(s, at[s] + i) for s in range(B) for i in range(new[s])]
        q, k, v = (np.stack([a[s, i] for s, i in tokens]) for a in (text.q, text.k, text.v))
        gnew, goff = to_gpu(new), to_gpu(off[:-1])
        pa.pages_reserve(None, cfg, tables, held, gnew, B, width, most_new if step == 0 else draft, refs, pairs, status, rs, rs_b)
        slots = empty_gpu((total,), np.int64)
        pa.build_slot_mapping(None, cfg, tables, width, held, gnew, goff, B, int(new.max()), slots)
        pa.kv_append(None, cfg, to_gpu(k), to_gpu(v), slots, total, kc, vc, None, None, None, None)
        prefix = held.clone()
        held += gnew
        most = width * 16
        out = empty_gpu((total, HQ, D), np.float32)
        if step and draft == 1:
            size = pa.window_decode_workspace_size(cfg, B, most, sink, window)
            ws = empty_gpu((size,), np.uint8)
            pa.window_decode(None, cfg, out, to_gpu(q), kc, vc, None, None, tables, held, B, width, most, sink, window, None, ws, size)
        else:
            size = pa.window_prefill_workspace_size(cfg, B, int(new.max()), most, sink, window)
            ws = empty_gpu((max(size, 16),), np.uint8)
            pa.window_prefill(None, cfg, out, to_gpu(q), to_gpu(off), prefix, kc, vc, None, None, tables, B, width, int(new.max()), most,
                              sink, window, None, ws, size)
        pa.evict_blocks(None, cfg, tables, held, None, B, width, sink_blocks, budget - sink_blocks, budget, refs, gone)
        got = to_np(out)
        assert to_np(status)[1] == 0
        left += to_np(gone).sum()
        # a prompt's rows in part
        check = range(total) if step else sorted(set(range(0, total, 13)) | {int(o) - 1 for o in off[1:]})
        for r in check:
            want, tol = text.attend(*tokens[r], sink, window, kv == FP32)
            close(got[r], want, tol, f"step {step}, sequence {tokens[r][0]}, position {tokens[r][1]}")
        at += new
    assert left > B and (to_np(held) <= 16 * budget).all()
    assert to_np(refs).sum() == sum((int(t) + 15) // 16 for t in to_np(held))
