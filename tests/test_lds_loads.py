"""The loads that go straight to LDS (csrc/attn_common.h) take their LDS address
from M0, which a scalar instruction has just written: gfx950 needs a wait state
between the two, which the compiler puts behind its own writes of M0 and not into
inline assembly.  Read from the assembly that the compiler makes of each of them,
and from the source of every kernel.  No GPU is used.
"""
import glob
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "pku-aiprogramming_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

KERNELS = """
#include "attn_common.h"
__global__ void sixteen(const char* p, uint32_t lds) { tt::glds16(p, 16u * threadIdx.x, lds); }
__global__ void sixteen_at(const char* p, uint32_t lds) { tt::glds16_at(p + 16u * threadIdx.x, lds); }
__global__ void four(const char* p, uint32_t lds) { tt::glds4(p, 4u * threadIdx.x, lds); }
__global__ void builtin(const char* p, uint32_t lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(p + 16u * threadIdx.x),
                                   (__attribute__((address_space(3))) void*)(uintptr_t)(lds + 16u), 16, 0, 0);
}
"""


def _waits(lines):
    """For each load to LDS, the wait states between the last write of M0 and it."""
    found, since = [], None
    for line in lines:
        op = line.split(";")[0].split()
        if not op or op[0].startswith(".") or op[0].endswith(":"):
            continue
        if "_lds_" in op[0] and op[0].startswith(("global_load", "buffer_load")):
            found.append(since)
        if since is not None:
            since += int(op[1], 0) + 1 if op[0] == "s_nop" else 1
        if op[0].startswith("s_") and len(op) > 1 and op[1].rstrip(",") == "m0":
            since = 0
    return found


def test_the_counting():
    assert _waits(["s_mov_b32 m0, s1", "global_load_lds_dword v0, off"]) == [0]
    assert _waits(["s_add_i32 m0, s1, 4 ; x", "s_nop 0", "global_load_lds_dword v0, off", "global_load_lds_dword v0, off"]) == [1, 2]
    assert _waits(["global_load_lds_dwordx4 v0, s[0:1]", "global_load_dwordx4 v[0:3], v0, s[0:1]"]) == [None]


@pytest.mark.skipif(not (os.path.exists(HIPCC) or shutil.which("hipcc")), reason="hipcc not available")
def test_a_wait_state_between_m0_and_the_load(tmp_path):
    src, out = tmp_path / "loads.hip", tmp_path / "loads.s"
    src.write_text(KERNELS)
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-S", "--offload-device-only", "-I", CSRC, "-I",
                        os.path.join(ROOT, "include"), str(src), "-o", str(out)],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
    waits = _waits(out.read_text().splitlines())
    assert len(waits) >= 4 and all(w is not None and w >= 1 for w in waits), waits


def test_no_source_writes_m0_right_before_a_load():
    bad = []
    for path in glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip")):
        with open(path) as f:
            for m in re.finditer(r'asm volatile\(\s*((?:"[^"]*"\s*)+)', f.read()):
                text = "".join(re.findall(r'"([^"]*)"', m.group(1)))
                if any(w is not None and w < 1 for w in _waits(re.split(r"\\n(?:\\t)?", text))):
                    bad.append((os.path.basename(path), text))
    assert not bad, bad
