"""Barriers between a workgroup's reads of LDS and the writes that reuse it, followed along the branches of the compiled kernels
(no GPU needed): a wave that runs ahead into a missing one shows in results only now and then."""
import os
import re

import pytest

from test_code_objects import HIPCC, kernels


def unguarded(text, reads, writes):
    """The instructions matching `writes` that a path reaches from one matching `reads` with no barrier on it."""
    code, labels = [], {}
    for line in text.splitlines():
        m = re.match(r"(\.LBB\w+):", line)
        if m:
            labels[m[1]] = len(code)
        elif re.match(r"\s+[a-z]", line):
            code.append(line.split(";")[0].strip())
    found, seen = set(), set()
    todo = [(0, False)]  # (instruction, a read without a barrier behind it)
    while todo:
        at, open_read = todo.pop()
        while at < len(code) and (at, open_read) not in seen:
            seen.add((at, open_read))
            op = code[at]
            if op.startswith("s_barrier"):
                open_read = False
            elif re.match(reads, op):
                open_read = True
            elif open_read and re.match(writes, op):
                found.add((at, op))
            m = re.match(r"s_(c?)branch\w*\s+(\.LBB\w+)", op)
            if m:
                todo.append((labels[m[2]], open_read))
            if op.startswith("s_endpgm") or (m and not m[1]):
                break
            at += 1
    return sorted(found)


def test_the_walk_sees_a_missing_barrier():
    loop = "\n.LBB0_1:\n\tds_write_b64 v1, v[2:3]\n\ts_barrier\n\tds_read_b64 v[2:3], v1\n%s\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm\n"
    assert len(unguarded(loop % "", "ds_read", "ds_write")) == 1
    assert unguarded(loop % "\ts_barrier\n", "ds_read", "ds_write") == []


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_compaction_rewrites_no_word_that_is_still_read():
    """The compaction keeps 64 blocks a word in LDS, a round of the pool at a time: every round's words are read before the next
    round's overwrite them. (The words are its only 64-bit writes.)"""
    text = [v for k, v in kernels("pages.hip").items() if "pages_compact_kernel" in k]
    assert len(text) == 1
    assert re.search(r"ds_write\w*_b64", text[0]) and re.search(r"ds_read\w*_b64", text[0])
    assert unguarded(text[0], r"ds_read\w*_b64", r"ds_write\w*_b64") == []
