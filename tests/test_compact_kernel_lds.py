"""The built compaction kernel: all of its LDS is in the launch's size, which the host holds against
64 KB (LDS of the kernel's own would come on top, past it for pools just below 2^18 pages)."""
import os
import re
import struct
import subprocess

import pytest

from test_kernel_wait_states import AMDGPU, LIB

READELF = "/opt/rocm/llvm/bin/llvm-readelf"


def test_no_lds_beside_the_launchs_size(tmp_path):
    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    with open(LIB, "rb") as f:
        data = f.read()
    at, sizes = data.find(b"\x7fELF", 1), []
    while at > 0:
        if struct.unpack_from("<H", data, at + 18)[0] == AMDGPU:
            path = tmp_path / "code.elf"
            path.write_bytes(data[at:])
            notes = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True).stdout
            for kernel in notes.split(".agpr_count:")[1:]:
                field = lambda name: re.search(rf"\.{name}:\s+(\S+)", kernel).group(1)
                if "compact_kernel" in field("name"):
                    sizes.append(int(field("group_segment_fixed_size")))
        at = data.find(b"\x7fELF", at + 4)
    assert sizes == [0]
