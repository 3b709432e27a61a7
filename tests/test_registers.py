"""The kernels of norms, rotation and the paged cache keep their values in registers:
read from the resource usage that the compiler wrote into the built library."""
import os
import re
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
READELF = "/opt/rocm/llvm/bin/llvm-readelf"
KERNELS = ("qkv_norm_rope_kernel", "qkv_norm_rope_bwd_kernel", "kv_append_kernel", "kv_append_e4m3_kernel", "kv_gather_kernel",
           "attn_decode_paged_kernel")


def code_objects(path):
    """The gfx950 code objects bundled in a shared library."""
    with open(path, "rb") as f:
        data = f.read()
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    for m in re.finditer(magic, data):
        at = m.start()
        (n,) = struct.unpack_from("<Q", data, at + len(magic))
        pos = at + len(magic) + 8
        for _ in range(n if n < 16 else 0):
            off, size, k = struct.unpack_from("<QQQ", data, pos)
            name = data[pos + 24:pos + 24 + k]
            pos += 24 + k
            if name.endswith(b"gfx950") and size:
                yield data[at + off:at + off + size]


@pytest.mark.skipif(not os.path.exists(READELF), reason="llvm-readelf not available")
def test_no_kernel_spills(tmp_path):
    import tt_capi

    found = {}
    for i, blob in enumerate(code_objects(tt_capi.LIB_PATH)):
        obj = tmp_path / f"{i}.co"
        obj.write_bytes(blob)
        text = subprocess.run([READELF, "--notes", str(obj)], capture_output=True, text=True, check=True, timeout=60).stdout
        for kernel in re.split(r"- \.agpr_count", text)[1:]:
            get = lambda key: re.search(r"\.%s:\s+(\S+)" % key, kernel).group(1)  # noqa: E731
            found[get("name")] = int(get("private_segment_fixed_size")), int(get("vgpr_spill_count"))
    mine = {n: v for n, v in found.items() if any(re.search(r"\d%sI" % k, n) for k in KERNELS)}
    assert all(any(k in n for n in mine) for k in KERNELS)
    bad = {n: v for n, v in mine.items() if any(v)}
    assert not bad, bad
