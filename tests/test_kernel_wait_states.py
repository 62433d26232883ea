"""Wait states in the built prompt attention.  On gfx9 a vector instruction that writes a scalar
register (v_readlane and v_readfirstlane among them, which also bring back spilled scalars) must
lie five wait states before a buffer load that reads it.  The compiler keeps the distance for its
own loads, but does not look into assembly, so the loads to LDS, which are written in it, carry
the wait themselves.  Read from the kernels in the built library: the loads' text, and every path of
the last five wait states before each memory instruction."""
import os
import re
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "persistentkv-attention_amd", "libpkv.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
AMDGPU = 224  # e_machine of the code objects inside the library
WAIT = 5
MEMORY = ("buffer_", "global_", "scratch_", "flat_")


def scalars(operand):
    """The scalar registers of one operand: s6, s[4:7], vcc."""
    if operand.startswith("vcc"):
        return {"vcc"}
    m = re.fullmatch(r"s(\d+)|s\[(\d+):(\d+)\]", operand)
    if not m:
        return set()
    first, last = (m[1], m[1]) if m[1] else (m[2], m[3])
    return set(range(int(first), int(last) + 1))


def parse(text):
    """{kernel: [(address, opcode, operands, branch target or None)]} of a listing."""
    kernels, code = {}, None
    for line in text.splitlines():
        head = re.match(r"([0-9a-f]+) <(\S+)>:", line)
        if head:
            base, code = int(head[1], 16), kernels.setdefault(head[2], [])
            continue
        m = re.match(r"\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):", line)
        if not m or code is None:
            continue
        operands = [x for x in re.split(r"[,\s]+", m[2]) if x]
        target = re.search(r"<\S+?(?:\+0x([0-9a-f]+))?>$", line) if "branch" in m[1] else None
        code.append((int(m[3], 16), m[1], operands, base + int(target[1] or "0", 16) if target else None))
    return kernels


def states(opcode, operands):
    return int(operands[0], 0) + 1 if opcode == "s_nop" else 1


def violations(code):
    """(writer, reader) pairs less than WAIT wait states apart on some path."""
    at = {ins[0]: i for i, ins in enumerate(code)}
    before = [[] for _ in code]
    for i, (_, opcode, _, target) in enumerate(code):
        if i + 1 < len(code) and opcode not in ("s_branch", "s_endpgm"):
            before[i + 1].append(i)
        if target is not None:
            before[at[target]].append(i)
    found = set()
    for i, (_, opcode, operands, _) in enumerate(code):
        if not opcode.startswith(MEMORY):
            continue
        reads = set().union(*map(scalars, operands)) if operands else set()
        todo = [(p, 0) for p in before[i]]
        while todo and reads:
            j, waited = todo.pop()
            if waited >= WAIT:
                continue
            _, op, args, _ = code[j]
            writes = set().union(*map(scalars, args[:2])) if op.startswith("v_cmp") or "_co_" in op else \
                scalars(args[0]) if op.startswith("v_") and args else set()
            if writes & reads:
                found.add((j, i))
            todo += [(p, waited + states(op, args)) for p in before[j]]
    return sorted(found)


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    assert os.path.exists(LIB), "build first"
    with open(LIB, "rb") as f:
        data = f.read()
    starts, at = [], data.find(b"\x7fELF", 1)
    while at > 0:
        if struct.unpack_from("<H", data, at + 18)[0] == AMDGPU:
            starts.append(at)
        at = data.find(b"\x7fELF", at + 4)
    found = {}
    for s, e in zip(starts, starts[1:] + [len(data)]):
        if b"prefill_kernel" in data[s:e]:
            path = tmp_path_factory.mktemp("co") / "code.elf"
            path.write_bytes(data[s:e])
            out = subprocess.run([OBJDUMP, "-d", str(path)], capture_output=True, text=True, check=True).stdout
            found.update({n: c for n, c in parse(out).items() if "prefill_kernel" in n and c})
    assert len(found) == 4, sorted(found)
    return found


def test_the_search_finds_what_it_looks_for():
    def listing(*lines):
        return "0000000000000000 <k>:\n" + "".join(f"\t{x} // {4 * i:012X}: 0\n" for i, x in enumerate(lines))

    load = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    for wait, bad in (("s_nop 3", True), ("s_nop 4", False)):
        for write in ("v_readlane_b32 s6, v205, 47", "v_readfirstlane_b32 s7, v1", "v_cmp_lt_u32_e64 s[4:5], v1, v2"):
            assert bool(violations(parse(listing(write, wait, load))["k"])) == bad, (write, wait)
    assert not violations(parse(listing("v_readlane_b32 s8, v205, 47", load))["k"])
    assert not violations(parse(listing("s_mov_b32 s6, s9", load))["k"])
    jump = "\ts_branch 1 // 000000000004: 0 <k+0xc>\n"
    code = listing("v_readlane_b32 s6, v205, 47", "s_nop 0", "s_nop 7", load).splitlines(keepends=True)
    code[2] = jump  # over the wait
    assert violations(parse("".join(code))["k"]) == [(0, 3)]


def test_scalars_are_written_five_wait_states_before_a_load_reads_them(kernels):
    for name, code in kernels.items():
        bad = [(code[j][1:3], code[i][1:3]) for j, i in violations(code)]
        assert not bad, (name, bad)


def test_loads_to_lds_carry_their_own_wait(kernels):
    """Whatever stands before: m0 is set and four wait states pass, with nothing between."""
    for name, code in kernels.items():
        loads = [i for i, ins in enumerate(code) if ins[2] and ins[2][-1] == "lds"]
        assert len(loads) >= 8, name
        for i in loads:
            setup, wait = code[i - 2], code[i - 1]
            assert setup[1] == "s_mov_b32" and setup[2][0] == "m0" and wait[1] == "s_nop", (name, code[i - 2:i + 1])
            assert states(*setup[1:3]) + states(*wait[1:3]) >= WAIT, (name, code[i - 2:i + 1])


def test_nothing_else_uses_m0(kernels):
    """The assembly sets m0, and the compiler takes no clobber of it."""
    for name, code in kernels.items():
        for i, (_, opcode, operands, _) in enumerate(code):
            if "m0" in operands:
                assert opcode.startswith("s_") and operands.index("m0") == 0 and code[i + 2][2][-1] == "lds", (name, code[i])
