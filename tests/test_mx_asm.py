"""Compiled MXFP4 kernels (CPU: compiles them to gfx950 assembly and reads it).

  - Inline-assembly DMAs keep their wait states and read no address register written just before them
    (the checks of tests/test_asm_hazards.py, on mx_gemm.hip).
  - No instruction touches the result of a matrix instruction before it is written.  The matrix unit does not
    hold such an instruction up; the compiler inserts the wait states, but was seen to count too few of them where a
    branch around an inline-assembly DMA lay between, and an element of an accumulator was read stale.  The
    kernels settle their accumulators with wait states of their own; here every path is counted.
"""
import os
import re

import pytest

from test_asm_hazards import CSRC, device_asm, instructions, sgprs

# wait states between a scaled fp4 matrix instruction and a read or write of its result by another unit: passes (of
# four cycles) + 3
WAIT = {"v_mfma_scale_f32_32x32x64_f8f6f4": 8 + 3, "v_mfma_scale_f32_16x16x128_f8f6f4": 4 + 3}


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    return device_asm(os.path.join(CSRC, "mx_gemm.hip"), tmp_path_factory.mktemp("asm"))


def vgprs(text):
    out = set()
    for m in re.finditer(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        out |= set(range(int(m.group(1)), int(m.group(2)) + 1)) if m.group(1) else {int(m.group(3))}
    return out


def functions(lines):
    """Name -> [(label or None, instruction or None)] of every kernel."""
    out, cur = {}, None
    for l in lines:
        m = re.match(r"^(_Z\w+):", l)
        if m:
            cur = out.setdefault(m.group(1), [])
            continue
        if cur is None or l.startswith(";"):
            continue
        m = re.match(r"^(\.LBB\w+):", l)
        if m:
            cur.append((m.group(1), None))
        elif l.startswith(".Lfunc_end"):
            cur = None
        elif l and not l.startswith(".") and not l.endswith(":"):
            cur.append((None, l.split(";")[0].strip()))
    return out


def early_touches(code):
    """(matrix instruction, instruction that touches its result too early) over every path."""
    at = {lab: i for i, (lab, _) in enumerate(code) if lab}
    bad = []
    for i, (_, ins) in enumerate(code):
        op = ins.split()[0] if ins else ""
        if op not in WAIT:
            continue
        dst = vgprs(ins.split(None, 1)[1].split(",")[0])
        todo, seen = [(i + 1, WAIT[op])], {}
        while todo:
            p, left = todo.pop()
            while p < len(code) and left > 0:
                if seen.get(p, 0) >= left:
                    break
                seen[p] = left
                t = code[p][1]
                if t is None:
                    p += 1
                    continue
                o = t.split()[0]
                if o == "s_nop":
                    left -= int(t.split()[1]) + 1
                    p += 1
                    continue
                if o in WAIT:                            # as the addend it is forwarded; as a factor it would not be
                    args = t.split(None, 1)[1].split(",")
                    if vgprs(",".join(args[1:3])) & dst:
                        bad.append((ins, t))
                    if vgprs(args[0]) & dst:             # a new result in its place: counted from there
                        break
                elif o[0] in "vdgb" and len(t.split()) > 1 and vgprs(t.split(None, 1)[1]) & dst:
                    bad.append((ins, t))
                left -= 1
                if o.startswith("s_cbranch"):
                    todo.append((at[t.split()[1]], left))
                elif o == "s_branch":
                    p = at[t.split()[1]]
                    continue
                elif o == "s_endpgm":
                    break
                p += 1
    return bad


def test_matrix_results_are_not_touched_early(lines):
    fns = functions(lines)
    kernels = {n: c for n, c in fns.items() if any(t and t.split()[0] in WAIT for _, t in c)}
    assert len(kernels) >= 8, list(fns)
    for name, code in kernels.items():
        bad = early_touches(code)
        assert not bad, (name, len(bad), bad[:5])


def test_the_check_sees_an_early_read():
    """The check itself, on a sequence as it was once compiled: a branch, three wait states, then a read."""
    code = [(None, "v_mfma_scale_f32_32x32x64_f8f6f4 v[2:17], v[34:37], v[38:41], v[2:17], v77, v42"), (None, "s_mov_b32 s38, 1"),
            (None, "s_cbranch_vccnz .LBB1_1"), (None, "s_nop 15"), (".LBB1_1", None), (None, "s_nop 2"), (None, "v_mov_b32_e32 v49, v17"), (None, "s_endpgm")]
    assert early_touches(code)
    code[5] = (None, "s_nop 9")
    assert not early_touches(code)


def test_dma_guard_and_addresses(lines):
    ins = instructions(lines)
    dma = [i for i, (t, inasm) in enumerate(ins) if t.startswith("global_load_lds") and inasm]
    assert len(dma) > 20
    for i in dma:
        assert ins[i - 1][0] == "s_nop 4", ins[i - 2:i + 1]
    vmem = re.compile(r"(global|buffer|flat)_")
    for i, (text, _) in enumerate(ins):
        if not vmem.match(text):
            continue
        reads = {r for op in text.split(None, 1)[1].split(",") for r in sgprs(op.split()[0] if op.split() else "")}
        states, j = 0, i - 1
        while reads and j >= 0 and states < 5:
            t = ins[j][0]
            if t.startswith("s_nop"):
                states += int(t.split()[1]) + 1
            else:
                states += 1
                if t.startswith("v_") and len(t.split()) > 1:
                    assert not (sgprs(t.split(None, 1)[1].split(",")[0]) & reads), (t, text)
            j -= 1
