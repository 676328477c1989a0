"""Wait states in front of the LDS DMAs that are written as inline assembly, whose
operands the compiler's own hazard pass does not look at (no GPU).  Between a vector
instruction that writes a scalar register and a vector memory instruction that reads
it there have to be five wait states, between any write of M0 and an LDS DMA one;
s_nop n makes n + 1, every other instruction one."""
import glob
import os
import re
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "chat-wgpu_amd", "csrc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-I", CSRC, "-I", os.path.join(ROOT, "include"), "-S", "--cuda-device-only"]

# A base straight from a vector instruction, as any caller may have it
FRESH = """
#include "prompt_device.hpp"
using namespace cwi;
__device__ const char *fresh(const char *p) {{
    const uint64_t v = (uint64_t)(uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    return reinterpret_cast<const char *>((uintptr_t)((uint64_t)hi << 32 | lo));
}}
__global__ void k(const char *const *p, float *y) {{
    __shared__ __attribute__((aligned(1024))) unsigned char lds[4096];
    const char *mine = p[threadIdx.x];
    const uint32_t off = threadIdx.x * 16;
    unsigned char *to = lds + (threadIdx.x >> 6) * 1024;
    {call};
    wait_vm<0>();
    __syncthreads();
    y[threadIdx.x] = reinterpret_cast<float *>(lds)[threadIdx.x];
}}
"""


def assembly(source, out):
    r = subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *FLAGS, source, "-o", out],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return open(out).read()


def registers(op):
    """The scalar registers that an operand names."""
    m = re.fullmatch(r"s\[(\d+):(\d+)\]|s(\d+)", op)
    if not m:
        return {op} & {"m0", "vcc"}
    lo, hi = (m.group(1), m.group(2)) if m.group(1) else (m.group(3), m.group(3))
    return {f"s{i}" for i in range(int(lo), int(hi) + 1)}


def short_waits(text):
    """(DMAs, those behind too few wait states) in the order of the code; a jump, which
    takes longer than five wait states, ends a run."""
    code, found, bad = [], 0, []
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        m = re.match(r"([a-z]\w+)\s*(.*)", line)
        if not m or line.startswith("."):
            continue
        name, ops = m.group(1), [o.strip() for o in m.group(2).split(",")]
        if name.startswith("global_load_lds"):
            found += 1
            base, waits = registers(ops[1].split()[0]), 0
            for n, o in reversed(code):
                second = re.match(r"v_(add|sub|subrev|addc|subb|subbrev)_co|v_div_scale|v_mad_[ui]64", n)
                written = set().union(*(registers(x) for x in o[:2 if second else 1]))
                if (n.startswith("v_") and waits < 5 and written & base) or (waits < 1 and "m0" in written):
                    bad.append((line, n, o, waits))
                waits += int(o[0], 0) + 1 if n == "s_nop" else 1
                if waits >= 5:
                    break
        code = [] if name in ("s_branch", "s_endpgm", "s_setpc_b64") else code[-5:] + [(name, ops)]
    return found, bad


def test_the_check_itself():
    dma = "global_load_lds_dwordx4 v1, s[2:3]"
    for before, ok in (("v_readfirstlane_b32 s3, v0\ns_nop 3", False), ("v_readfirstlane_b32 s3, v0\ns_nop 4", True),
                       ("v_readfirstlane_b32 s4, v0", True), ("v_add_co_u32 v0, s[2:3], v1, v2", False), ("s_mov_b32 s3, s9", True),
                       ("s_mov_b32 m0, s9", False), ("s_mov_b32 m0, s9\ns_nop 0", True),
                       ("v_readlane_b32 s2, v0, 3\n" + 4 * "v_mov_b32 v2, v3\n", False),
                       ("v_readlane_b32 s2, v0, 3\n" + 5 * "v_mov_b32 v2, v3\n", True)):
        found, bad = short_waits(before + "\n" + dma)
        assert found == 1 and (not bad) == ok, before


@pytest.mark.parametrize("call,ok", [("dma16(fresh(mine), off, to)", False),
                                     ("dma16u(mine, off, lds_off(to))", True),
                                     ("dma4u(mine, off, lds_off(to))", True)])
def test_a_base_from_a_vector_instruction(tmp_path, call, ok):
    """What the helpers for any base are for, and that it shows where another is taken."""
    source = tmp_path / "fresh.hip"
    source.write_text(FRESH.format(call=call))
    text = assembly(str(source), str(tmp_path / "fresh.s"))
    found, bad = short_waits(text)
    assert found == 1 and "v_readfirstlane_b32" in text
    assert (not bad) == ok, bad


def with_dmas():
    files = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    return [os.path.basename(f) for f in files if re.search(r"\bdma\w*\(|global_load_lds", open(f).read())]


@pytest.mark.parametrize("source", with_dmas())
def test_the_kernels(tmp_path, source):
    found, bad = short_waits(assembly(os.path.join(CSRC, source), str(tmp_path / "k.s")))
    assert found > 0 and not bad, bad[:5]
