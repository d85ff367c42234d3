"""Results of matrix instructions in the compiled MXFP4 kernels, in both register files (CPU: compiles mx_gemm.hip to gfx950
assembly and reads it).

A matrix instruction writes its result some cycles after it was issued, to vector registers (v) or to accumulation
registers (a, where a wave is alone on its SIMD and has 512).  Along every path from it, another unit that reads or
writes the result, or another matrix instruction that takes it as a factor, has to lie as many wait states behind as the
instruction takes passes, and four: the compiler itself puts twelve between one of 8 passes and a vector instruction
(test_the_compilers_own_distance).  As the addend of a later matrix instruction it is forwarded."""
import os
import re
import subprocess

import pytest

from test_asm_hazards import CSRC, HIPCC, device_asm
from test_mx_asm import functions

# wait states: passes + 4
WAIT = {"v_mfma_scale_f32_32x32x64_f8f6f4": 8 + 4, "v_mfma_scale_f32_16x16x128_f8f6f4": 4 + 4}


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not installed")
    fns = functions(device_asm(os.path.join(CSRC, "mx_gemm.hip"), tmp_path_factory.mktemp("asm")))
    return {n: c for n, c in fns.items() if any(t and t.split()[0] in WAIT for _, t in c)}


def registers(text):
    """{"v3", "a17", ..}: the vector and accumulation registers that a text names."""
    out = set()
    for f, lo, hi, one in re.findall(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        out |= {f + str(i) for i in (range(int(lo), int(hi) + 1) if lo else [int(one)])}
    return out


def operands(ins):
    """The operands of an instruction, as texts."""
    return [o.strip() for o in ins.split(None, 1)[1].split(",")] if " " in ins else []


def early(code):
    """(matrix instruction, instruction, wait states too few) of every touch of a result that is not there yet."""
    at = {lab: i for i, (lab, _) in enumerate(code) if lab}
    bad = []
    for i, (_, ins) in enumerate(code):
        if not ins or ins.split()[0] not in WAIT:
            continue
        dst = registers(operands(ins)[0])
        assert len(dst) in (4, 16), ins
        todo, seen = [(i + 1, WAIT[ins.split()[0]])], {}
        while todo:
            p, left = todo.pop()
            while p < len(code) and left > 0 and seen.get(p, 0) < left:
                seen[p] = left
                t = code[p][1]
                p += 1
                if t is None:
                    continue
                o, args = t.split()[0], operands(t)
                if o == "s_nop":
                    left -= int(args[0]) + 1
                    continue
                if o in WAIT:
                    if registers(",".join(args[1:3])) & dst:
                        bad.append((ins, t, left))
                    if registers(args[0]) & dst:         # a new result in its place: counted from there
                        break
                elif not o.startswith("s_") and registers(" ".join(args)) & dst:
                    bad.append((ins, t, left))
                left -= 1
                if o.startswith("s_cbranch"):
                    todo.append((at[args[0]], left))
                elif o == "s_branch":
                    p = at[args[0]]
                elif o == "s_endpgm":
                    break
    return bad


def test_no_result_is_touched_early(kernels):
    assert len(kernels) >= 8, list(kernels)
    for name, code in kernels.items():
        bad = early(code)
        assert not bad, (name, len(bad), bad[:5])


def test_both_register_files_occur(kernels):
    """The kernels with accumulators in a[..] are among those that are checked."""
    files = {f: {n for n, c in kernels.items() for _, t in c if t and t.split()[0] in WAIT and operands(t)[0].startswith(f)} for f in "va"}
    assert len(files["a"]) >= 4 and len(files["v"]) >= 8, {f: sorted(n) for f, n in files.items()}


M32 = "v_mfma_scale_f32_32x32x64_f8f6f4 {0}[2:17], v[34:37], v[38:41], {0}[2:17], v77, v42 op_sel_hi:[0,0,0]"


@pytest.mark.parametrize("f,touch", [("v", "v_mov_b32_e32 v49, v17"), ("v", "v_mov_b32_e32 v2, 0"), ("v", "ds_write_b128 v60, v[14:17]"),
                                     ("a", "v_accvgpr_read_b32 v49, a17"), ("a", "v_accvgpr_write_b32 a2, v1"), ("a", "ds_write_b128 v60, a[14:17]"),
                                     ("a", "global_store_dwordx4 v[60:61], a[2:5], off"),
                                     ("v", "v_mfma_scale_f32_32x32x64_f8f6f4 v[80:95], v[14:17], v[38:41], v[80:95], v77, v42")])
def test_the_check_counts_to_twelve(f, touch):
    """Eleven wait states are one too few, on the straight way and over a branch around a longer one."""
    nops = lambda n: [(None, "s_nop 7"), (None, f"s_nop {n - 9}")]       # noqa: E731
    for n, ok in ((11, False), (12, True)):
        straight = [(None, M32.format(f)), *nops(n), (None, touch), (None, "s_endpgm")]
        around = [(None, M32.format(f)), (None, "s_cbranch_vccnz .LBB1_1"), (None, "s_nop 15"), (".LBB1_1", None), *nops(n - 1), (None, touch), (None, "s_endpgm")]
        assert (not early(straight)) == ok and (not early(around)) == ok, (n, touch)
    chain = [(None, M32.format(f)), (None, M32.format(f)), (None, "s_endpgm")]           # the sum itself goes on
    assert not early(chain)


def test_the_compilers_own_distance(tmp_path):
    """Where no branch is in its way the compiler waits as long as is asked for here."""
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not installed")
    src = tmp_path / "one.hip"
    src.write_text("""#include <hip/hip_runtime.h>
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
__global__ void k(const v8i* a, v16f* d) {
    v16f c = d[threadIdx.x];
    c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[0], a[threadIdx.x], c, 4, 4, 0, 127, 0, 127);
    for (int i = 0; i < 16; ++i) c[i] = c[i] * c[i];
    d[threadIdx.x] = c;
}
""")
    out = tmp_path / "one.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "--cuda-device-only", "-S", "-o", str(out), str(src)], check=True, capture_output=True)
    code = functions([l.strip() for l in out.read_text().splitlines()])
    code = next(c for n, c in code.items() if "1k" in n)
    at = next(i for i, (_, t) in enumerate(code) if t and t.split()[0] in WAIT)
    dst, states = registers(operands(code[at][1])[0]), 0
    for _, t in code[at + 1:]:
        if not t:
            continue
        if not t.startswith("s_") and registers(" ".join(operands(t))) & dst:
            break
        states += int(operands(t)[0]) + 1 if t.startswith("s_nop") else 1
    assert states >= WAIT[code[at][1].split()[0]], states
    assert not early(code)
