"""The MXFP4 GEMV turns activation rows into operands through LDS of the wave, without a barrier: a lane reads what others
wrote.  The hardware carries out a wave's LDS accesses in order, the compiler keeps the order of a lane's accesses only where
it is told to (CPU: compiles mx_gemm.hip to LLVM IR for gfx950 and reads it)."""
import os
import re
import subprocess

import pytest

from test_asm_hazards import CSRC, HIPCC


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not installed")
    out = tmp_path_factory.mktemp("ir") / "mx_gemm.ll"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only",
                    "-S", "-emit-llvm", "-o", str(out), os.path.join(CSRC, "mx_gemm.hip")], check=True, capture_output=True)
    fns, name = {}, None
    for l in out.read_text().splitlines():
        m = re.match(r"define .*@(\w+)\(", l)
        if m:
            name = m.group(1)
            fns[name] = []
        elif l == "}":
            name = None
        elif name:
            fns[name].append(l.strip())
    return {n: c for n, c in fns.items() if "k_gemv_mxfp4" in n}


def unordered(code):
    """LDS reads right after writes, and writes right after reads, of a block with nothing that orders them."""
    bad, last = [], None
    for l in code:
        if re.match(r"\d+:|[\w.]+:", l) or "fence syncscope" in l or "amdgcn.s.barrier" in l:
            last = None
        elif re.search(r"\bload .*ptr addrspace\(3\)", l) or re.match(r"store .*, ptr addrspace\(3\)", l):
            kind = "load" if " load " in l else "store"
            if last not in (None, kind):
                bad.append(l)
            last = kind
    return bad


def test_lds_exchanges_are_ordered(kernels):
    assert len(kernels) == 6, list(kernels)
    for name, code in kernels.items():
        lds = [l for l in code if "ptr addrspace(3)" in l and (" load " in l or l.startswith("store"))]
        assert len(lds) > 20, (name, len(lds))
        assert not unordered(code), (name, unordered(code)[:4])


def test_the_check_sees_a_missing_fence():
    w, r = "store <4 x i32> %1, ptr addrspace(3) %2, align 16", "%3 = load <4 x i32>, ptr addrspace(3) %4, align 16"
    assert unordered([w, r]) and unordered([r, w]) and not unordered([w, w]) and not unordered([w, 'fence syncscope("wavefront") acq_rel', r])
