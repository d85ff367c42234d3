"""Compiled kernels of attention (CPU: compiles them to gfx950 assembly and LLVM IR and reads it).

  - Inline-assembly DMAs keep their wait states and read no register written just before them.
  - No instruction touches the result of a matrix instruction before it is written: the compiler inserts the wait states, but was seen
    to count too few where a branch around an inline-assembly DMA lay between.
  - Exchanges between a wave's lanes through LDS without a barrier are ordered by fences.
"""
import os
import re
import subprocess

import pytest

import test_mx_asm
import test_mx_lds_order
import test_mx_results_asm as results
from test_asm_hazards import CSRC, HIPCC, device_asm

FILES = ["attn_prompt.hip", "attn_kv.hip"]
# passes (of four cycles) + 4, as the compiler waits where no branch is in its way
WAIT = {"v_mfma_f32_32x32x16_bf16": 8 + 4, "v_mfma_f32_16x16x32_bf16": 4 + 4}


@pytest.fixture(scope="module", params=FILES)
def asm(request, tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not installed")
    return request.param, device_asm(os.path.join(CSRC, request.param), tmp_path_factory.mktemp("asm"))


def test_no_result_is_touched_early(asm, monkeypatch):
    monkeypatch.setattr(results, "WAIT", WAIT)
    name, lines = asm
    kernels = {n: c for n, c in test_mx_asm.functions(lines).items() if any(t and t.split()[0] in WAIT for _, t in c)}
    assert len(kernels) >= {"attn_prompt.hip": 3, "attn_kv.hip": 11}[name], list(kernels)
    for n, code in kernels.items():
        bad = results.early(code)
        assert not bad, (n, len(bad), bad[:5])


def test_the_check_sees_an_early_read(monkeypatch):
    monkeypatch.setattr(results, "WAIT", WAIT)
    m = "v_mfma_f32_32x32x16_bf16 v[2:17], v[34:37], v[38:41], v[2:17]"
    for n, ok in ((11, False), (12, True)):
        code = [(None, m), (None, "s_cbranch_vccnz .LBB1_1"), (None, "s_nop 15"), (".LBB1_1", None), (None, "s_nop 7"), (None, f"s_nop {n - 10}"),
                (None, "v_mov_b32_e32 v49, v17"), (None, "s_endpgm")]
        assert (not results.early(code)) == ok


def test_dma_guard_and_addresses(asm):
    name, lines = asm
    if name == "attn_prompt.hip":
        test_mx_asm.test_dma_guard_and_addresses(lines)
    else:
        assert not [l for l in lines if l.startswith(("global_load_lds", "buffer_load")) and "lds" in l]


def test_lds_exchanges_are_ordered(tmp_path):
    """Between a lane's writes and reads of the cache kernel's LDS there is a fence or a barrier; the transposing reads are reads."""
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not installed")
    out = tmp_path / "k.ll"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only",
                    "-S", "-emit-llvm", "-o", str(out), os.path.join(CSRC, "attn_kv.hip")], check=True, capture_output=True)
    fns, name = {}, None
    for l in out.read_text().splitlines():
        m = re.match(r"define .*@(\w+)\(", l)
        if m:
            name = m.group(1)
            fns[name] = []
        elif l == "}":
            name = None
        elif name:
            fns[name].append(re.sub(r"= (tail )?call <4 x i16> @llvm\.amdgcn\.ds\.read\.tr16", "= load <4 x i16>, tr16", l.strip()))
    fns = {n: c for n, c in fns.items() if "k_attn" in n}
    assert len(fns) == 26, list(fns)                                     # 23 of the attention, three joins
    for n, code in fns.items():
        assert sum("ptr addrspace(3)" in l for l in code) > 3, n
        assert not test_mx_lds_order.unordered(code), (n, test_mx_lds_order.unordered(code)[:4])


def test_no_scratch(asm):
    """The kernels that carry the load keep their state in registers: at most 64 bytes a thread go to memory (some address arithmetic
    of the narrowest register budgets)."""
    name, lines = asm
    sizes = [int(l.split(":")[1]) for l in lines if l.startswith(".private_segment_fixed_size:")]
    assert sizes and max(sizes) <= 64, sizes


def test_all_state_is_in_registers(asm):
    """No kernel has a private segment, nor a spilled register."""
    name, lines = asm
    sizes, spills = ([int(l.split(":")[1]) for l in lines if l.startswith(x)] for x in (".private_segment_fixed_size:", ".vgpr_spill_count:"))
    assert len(sizes) == len(spills) == {"attn_prompt.hip": 6, "attn_kv.hip": 26}[name]
    assert max(sizes) == 0 and max(spills) == 0, (sizes, spills)
