"""The built attention over cached pages: registers that keep three workgroups on a CU with nothing
spilled to memory, and its loads to LDS, which are written in assembly.  On gfx9 a vector
instruction that writes a scalar register must lie five wait states before a load that reads it,
and m0 must be one wait state old; the compiler keeps no distances to assembly."""
import os
import re
import struct
import subprocess

import pytest

from test_kernel_wait_states import AMDGPU, LIB, OBJDUMP, parse, states, violations

READELF = "/opt/rocm/llvm/bin/llvm-readelf"


@pytest.fixture(scope="module")
def code_object(tmp_path_factory):
    if not os.path.exists(OBJDUMP) or not os.path.exists(READELF):
        pytest.skip("no llvm-objdump or llvm-readelf")
    assert os.path.exists(LIB), "build first"
    with open(LIB, "rb") as f:
        data = f.read()
    starts, at = [], data.find(b"\x7fELF", 1)
    while at > 0:
        if struct.unpack_from("<H", data, at + 18)[0] == AMDGPU:
            starts.append(at)
        at = data.find(b"\x7fELF", at + 4)
    for s, e in zip(starts, starts[1:] + [len(data)]):
        if b"chunk_kernel" in data[s:e]:
            path = tmp_path_factory.mktemp("co") / "code.elf"
            path.write_bytes(data[s:e])
            return str(path)
    raise AssertionError("no chunk_kernel in the library")


@pytest.fixture(scope="module")
def kernels(code_object):
    out = subprocess.run([OBJDUMP, "-d", code_object], capture_output=True, text=True, check=True).stdout
    found = {n: c for n, c in parse(out).items() if "chunk_kernel" in n and c}
    assert len(found) == 2, sorted(found)
    return found


def test_registers_and_lds_of_three_workgroups_a_cu(code_object):
    notes = subprocess.run([READELF, "--notes", code_object], capture_output=True, text=True, check=True).stdout
    seen = 0
    for kernel in notes.split(".agpr_count:")[1:]:
        field = lambda name: re.search(rf"\.{name}:\s+(\S+)", kernel).group(1)
        if "chunk_kernel" in field("name"):
            seen += 1
            assert int(field("vgpr_count")) <= 168 and int(field("private_segment_fixed_size")) == 0
            assert 3 * int(field("group_segment_fixed_size")) <= 160 * 1024
    assert seen == 2


def test_scalars_are_written_five_wait_states_before_a_load_reads_them(kernels):
    for name, code in kernels.items():
        bad = [(code[j][1:3], code[i][1:3]) for j, i in violations(code)]
        assert not bad, (name, bad)


def test_loads_to_lds_carry_their_own_wait(kernels):
    for name, code in kernels.items():
        loads = [i for i, ins in enumerate(code) if ins[1].startswith("global_load_lds")]
        assert len(loads) >= 16, name
        for i in loads:
            setup, wait = code[i - 2], code[i - 1]
            assert setup[1] == "s_mov_b32" and setup[2][0] == "m0" and wait[1] == "s_nop", (name, code[i - 2:i + 1])
            based = code[i][2][-1] != "off"  # a scalar base
            assert states(*setup[1:3]) + states(*wait[1:3]) >= (5 if based else 2), (name, code[i - 2:i + 1])


def test_nothing_else_uses_m0(kernels):
    for name, code in kernels.items():
        for i, (_, opcode, operands, _) in enumerate(code):
            if "m0" in operands:
                assert opcode == "s_mov_b32" and operands.index("m0") == 0 and code[i + 2][1].startswith("global_load_lds"), (name, code[i])
