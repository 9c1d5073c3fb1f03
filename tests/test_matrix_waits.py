"""Waits that hipcc puts into the assembly of the kernels, and what it cannot see to.

Reads of a matrix instruction's result, in the assembly that hipcc writes for every kernel: along every way through the branches, as many
wait states as the instruction needs lie between it and the first vector instruction that reads or overwrites its result (the
hardware does not wait by itself; hipcc counts too few where a block can be reached on several ways). No GPU needed."""
import concurrent.futures
import glob
import os
import re

import pytest

from test_code_objects import HIPCC, PKG, kernels

# What hipcc keeps to in straight code: the passes of an instruction, and three or four more (fp32 operands: two).
WAITS = {"v_mfma_f32_16x16x16_bf16": 8, "v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_i32_16x16x64_i8": 8,
         "v_mfma_f32_32x32x16_bf16": 12, "v_mfma_f32_16x16x4_f32": 10, "v_mfma_f32_4x4x1_16b_f32": 4}


def registers(operand):
    m = re.match(r"-?\|?([av])(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    first, last = (m[2], m[2]) if m[2] else (m[3], m[4])
    return {(m[1], i) for i in range(int(first), int(last) + 1)}


def instructions(text):
    """[(name, operands)], labels as (label, None)."""
    out = []
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        label = re.match(r"(\.LBB\w+):", line)
        if label:
            out.append((label[1], None))
        elif line and not line.startswith(".") and not line.endswith(":"):
            name, _, rest = line.partition(" ")
            out.append((name.strip(), [x.strip() for x in rest.split(",")] if rest.strip() else []))
    return out


def touches(name, operands, result):
    """Whether a vector instruction reads or overwrites registers of a result."""
    used = set().union(*(registers(x.split(" ")[0]) for x in operands)) if operands else set()
    return bool(used & result)


def too_early(code):
    """[(wait states, matrix instruction, the one that comes too early)]"""
    at = {name: i for i, (name, operands) in enumerate(code) if operands is None}
    found = []
    for i, (name, operands) in enumerate(code):
        if operands is None or not name.startswith("v_mfma"):
            continue
        need, result = WAITS[name], registers(operands[0])
        todo, best = [(i + 1, 0)], {}
        while todo:
            j, waits = todo.pop()
            while j < len(code) and waits < need and best.get(j, need) > waits:
                best[j] = waits
                other, ops = code[j]
                j += 1
                if ops is None:
                    continue
                if other == "s_endpgm":
                    break
                if other == "s_nop":
                    waits += int(ops[0], 0) + 1
                    continue
                if other.startswith("v_mfma"):
                    if any(registers(x) & result for x in ops[1:3]):
                        found.append((waits, f"{name} {operands}", f"{other} {ops}"))
                        break
                    if registers(ops[0]) & result:
                        break  # its own result is looked at for itself
                elif not other.startswith("s_") and touches(other, ops, result):
                    found.append((waits, f"{name} {operands}", f"{other} {ops}"))
                    break
                waits += 1
                if other == "s_branch":
                    j = at[ops[0]]
                elif other.startswith("s_cbranch"):
                    todo.append((at[ops[0]], waits))
    return found


def test_the_search_itself():
    """A way of 7 and one of 8 wait states to the same read: the shorter one is found, whichever comes first."""
    text = """
    v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]
    s_cbranch_scc1 .LBB0_2
    s_nop 0
.LBB0_2:
    s_nop {}
    v_accvgpr_read_b32 v9, a3
    s_endpgm
    """
    assert [x[0] for x in too_early(instructions(text.format(5)))] == [7]
    assert too_early(instructions(text.format(6))) == []
    assert too_early(instructions(text.format(0).replace("a3", "a4"))) == []
    assert len(too_early(instructions(text.format(0).replace("v_accvgpr_read_b32 v9, a3", "ds_write_b32 v1, a2 offset:8")))) > 0


@pytest.fixture(scope="module")
def assembly():
    """[(source, kernel, its assembly)] of every kernel."""
    if not os.path.exists(HIPCC):
        pytest.skip("needs hipcc")
    sources = sorted(os.path.basename(f) for f in glob.glob(os.path.join(PKG, "csrc", "*.hip")))
    flags = {"chunked_prefill.hip": ["-fno-honor-nans"]}  # as in the Makefile
    with concurrent.futures.ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
        built = list(pool.map(lambda s: kernels(s, *flags.get(s, [])), sources))
    return [(source, name, text) for source, texts in zip(sources, built) for name, text in texts.items()]


def test_results_are_waited_for(assembly):
    products, found = 0, []
    for source, name, text in assembly:
        code = instructions(text)
        products += sum(n.startswith("v_mfma") for n, _ in code)
        found += [(source, name, *x) for x in too_early(code)]
    assert products > 1000
    assert not found, "\n".join(str(x) for x in found)


def test_inline_asm_forms_no_values(assembly):
    """hipcc knows no instruction of inline asm by what it reads and writes, so it leaves out the waits between one and the vector instructions
    around it: inline asm holds waits, barriers and loads alone."""
    blocks = 0
    for source, name, text in assembly:
        for block in re.findall(r";;#ASMSTART(.*?);;#ASMEND", text, flags=re.S):
            names = [line.split(";")[0].split()[0] for line in block.splitlines() if line.split(";")[0].strip()]
            assert not [x for x in names if x.startswith("v_")], (source, name, block)
            blocks += len(names) > 0
    assert blocks > 100
