"""CPU checks of workspaces that a launcher gives up: where the work that clears a new
one cannot be queued, no later call may take it for cleared (tests/native/
workspace_checks.cpp over csrc/device_cache.h, under sanitizers)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "pku-aiprogramming_amd", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_buffers_given_up(tmp_path):
    exe = str(tmp_path / "workspace_checks")
    src = os.path.join(ROOT, "tests", "native", "workspace_checks.cpp")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-pthread",
                        "-I", CSRC, src, "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=1"))
    assert r.returncode == 0 and "workspace checks passed" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("name", ["attn_decode_paged.hip", "norm_rope.hip"])
def test_launchers_of_cleared_buffers(name):
    """The launch that clears a fresh buffer is followed by the check that gives it up."""
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    blocks = re.findall(r"if \(fresh\) \{(.*?)\n\s*\}", text, re.S)
    assert len(blocks) == 1 and "lease->cleared(" in blocks[0] and "TT_LAUNCHED" not in blocks[0]
