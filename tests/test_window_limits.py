"""Bounds that include/paged_attn.h gives the operators for bounded caches, met from both sides on the host. Every call is
refused: one within its bound for the argument that is checked last. No GPU."""
import pytest

import paged_attention as pa
from test_window_refusals import INVALID, UNSUPPORTED, cfg, mass, refused

TYPES = [(kv, q) for kv in (0, 1, 2) for q in (0, 1)]


@pytest.mark.parametrize("kv,q", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_contexts_of_prompt_masses(kv, q, d):
    if kv == 2 and d == 32:
        return  # refused whatever the context is
    c = cfg(kv_dtype=kv, q_dtype=q, head_dim=d)
    within, beyond = dict(width=2 ** 27 - 1, most=5 * 10 ** 8), dict(width=2 ** 27 - 1, most=2 ** 31 - 1)
    for more in (dict(), dict(window=2 ** 31 - 1)):
        refused(pa.prefill_mass, INVALID, "null", *mass(c, q=None, **within, **more))
        refused(pa.prefill_mass, UNSUPPORTED, "too many blocks", *mass(c, q=None, **beyond, **more))
    # a window bounds what is read; a narrow table too
    refused(pa.prefill_mass, INVALID, "null", *mass(c, q=None, **beyond | dict(window=10 ** 6)))
    refused(pa.prefill_mass, INVALID, "null", *mass(c, q=None, **beyond | dict(width=5 * 10 ** 8 // 16)))
