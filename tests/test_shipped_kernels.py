"""The code objects inside the built module, as they ship: no kernel uses scratch memory or spills a vector register.

Compiling the sources again would check what other flags make of them; this reads the metadata that the build's own
compiler wrote into the module (CPU-only)."""
import os
import re
import struct
import subprocess

import pytest

from crack_detection_federatedlearning_grpc_amd import _build

READELF = "/opt/rocm/llvm/bin/llvm-readelf"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(blob):
    """The device code objects of every translation unit's offload bundle."""
    at = blob.find(MAGIC)
    while at >= 0:
        (n,) = struct.unpack_from("<Q", blob, at + len(MAGIC))
        pos = at + len(MAGIC) + 8
        for _ in range(n):
            off, size, idlen = struct.unpack_from("<QQQ", blob, pos)
            name = blob[pos + 24:pos + 24 + idlen].decode()
            pos += 24 + idlen
            if name.startswith("hip") and _build.ARCH in name and size:
                yield blob[at + off:at + off + size]
        at = blob.find(MAGIC, at + 1)


@pytest.mark.skipif(not os.path.exists(READELF) or not os.path.exists(_build.hip_path()), reason="no module or no readelf")
def test_no_shipped_kernel_uses_scratch(tmp_path):
    with open(_build.hip_path(), "rb") as f:
        blob = f.read()
    bad, names = [], []
    for n, code in enumerate(code_objects(blob)):
        path = tmp_path / f"{n}.co"
        path.write_bytes(code)
        text = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True, check=True).stdout
        for kernel in re.split(r"\n  - \.agpr_count:", text)[1:]:
            get = {k: v for k, v in re.findall(r"\.(name|private_segment_fixed_size|vgpr_spill_count):\s+(\S+)", kernel)
                   if k != "name" or v.startswith("_Z")}
            names.append(get["name"])
            if int(get["private_segment_fixed_size"]) or int(get["vgpr_spill_count"]):
                bad.append(get)
    assert len(names) > 200 and any("attn_dkv_kernel" in n for n in names)
    assert not bad, bad
