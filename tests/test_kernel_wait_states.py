"""Wait states in front of the library's vector-memory instructions, from its own gfx950 code.

A vector instruction that writes a scalar register has to be five wait states ahead of a
vector-memory instruction that reads it (descriptor or offset): the register's old value may be
read otherwise. The compiler keeps that distance for the instructions it makes itself, but not
for those written in assembly. Every way that leads to such a load is followed backwards here
for five wait states, over labels and branches.
"""
from __future__ import annotations

import os
import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]
LIBRARY = REPO / "raggedroute_amd" / "libraggedroute_amd.so"
OBJDUMP = Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "llvm" / "bin" / "llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
STATES = 5

LINE = re.compile(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):")
LABEL = re.compile(r"^([0-9a-f]+) <(.+)>:")
TARGET = re.compile(r"// [0-9A-F]+:.*<(.+?)(?:\+0x([0-9a-f]+))?>\s*$")
VMEM = re.compile(r"^(buffer|tbuffer|global|flat|scratch)_")
SCALARS = re.compile(r"\b(vcc\b|s\[(\d+):(\d+)\]|s(\d+)\b)")
# vector instructions whose second operand is a scalar result
CARRY = re.compile(r"^v_(add|sub|subrev|addc|subb|subbrev)_co_|^v_div_scale|^v_mad_[ui]64_")


def code_objects(library: bytes):
    """The gfx950 code objects in a library's offload bundles."""
    at = library.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", library, at + len(MAGIC))
        entry = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", library, entry)
            name = library[entry + 24:entry + 24 + length].decode()
            entry += 24 + length
            if "gfx950" in name and size:
                yield library[at + offset:at + offset + size]
        at = library.find(MAGIC, at + len(MAGIC))


def scalars(text: str) -> set:
    found = set()
    for name, low, high, one in SCALARS.findall(text):
        found |= {"vcc"} if name == "vcc" else {int(one)} if one else set(range(int(low), int(high) + 1))
    return found


def written(mnemonic: str, operands: str) -> set:
    """Scalar registers that a vector instruction writes."""
    if not mnemonic.startswith("v_"):
        return set()
    parts = re.split(r",\s*", operands)
    return scalars(", ".join(parts[:2] if CARRY.match(mnemonic) else parts[:1]))


def parse(text: str):
    """[(mnemonic, operands)], predecessors of every instruction, the function it lies in."""
    instructions, functions, where, branches, labels = [], [], {}, [], {}
    function = None
    for line in text.splitlines():
        label = LABEL.match(line)
        if label:
            function = label.group(2)
            labels[function] = int(label.group(1), 16)
            continue
        m = LINE.match(line)
        if not m:
            continue
        index = len(instructions)
        where[int(m.group(3), 16)] = index
        instructions.append((m.group(1), m.group(2)))
        functions.append(function)
        if m.group(1).startswith(("s_branch", "s_cbranch")):
            branches.append((index, TARGET.search(line)))
    before = [[] for _ in instructions]
    for i, (mnemonic, _) in enumerate(instructions[:-1]):
        if not mnemonic.startswith(("s_branch", "s_endpgm", "s_setpc")):
            before[i + 1].append(i)
    for i, target in branches:
        assert target, instructions[i]
        before[where[labels[target.group(1)] + int(target.group(2) or "0", 16)]].append(i)
    return instructions, before, functions


def too_early(instructions, before, functions):
    """(function, writer, reader) of every scalar register that is read too early."""
    found = []
    for i, (mnemonic, operands) in enumerate(instructions):
        if not VMEM.match(mnemonic):
            continue
        wanted = scalars(operands)
        if not wanted:
            continue
        ways = [(p, 0) for p in before[i]]
        seen = set()
        while ways:
            at, states = ways.pop()
            if (at, states) in seen:
                continue
            seen.add((at, states))
            name, args = instructions[at]
            if written(name, args) & wanted:
                found.append((functions[i], f"{name} {args}", f"{mnemonic} {operands}", states))
                continue
            states += int(args, 0) + 1 if name == "s_nop" else 1
            if states < STATES:
                ways += [(p, states) for p in before[at]]
    return found


def test_the_reader_sees_a_short_distance():
    """The scan itself, on instructions written here."""
    near = [("v_readfirstlane_b32", "s7, v1"), ("s_mov_b32", "m0, s2"), ("s_nop", "0"),
            ("buffer_load_dwordx4", "v1, s[4:7], 0 offen lds"), ("s_endpgm", "")]
    line = [[], [0], [1], [2], [3]]
    assert len(too_early(near, line, ["f"] * 5)) == 1
    assert not too_early(near[:2] + [("s_nop", "3")] + near[3:], line, ["f"] * 5)
    assert not too_early([("v_readfirstlane_b32", "s8, v1")] + near[1:], line, ["f"] * 5)
    assert not too_early([("s_add_u32", "s7, s8, s9")] + near[1:], line, ["f"] * 5)
    assert too_early([("v_add_co_u32", "v2, s[6:7], v1, v2")] + near[1:], line, ["f"] * 5)
    # over a branch back
    assert too_early(near, [[], [], [1], [2, 0], [3]], ["f"] * 5)


def test_assembly_names_m0_where_it_writes_it():
    """m0 is the compiler's, too (LDS loads of its own, lane and register indexes): an
    assembly statement that writes it lists it among its clobbers."""
    writers = 0
    for source in sorted((REPO / "raggedroute_amd" / "csrc").glob("*")):
        for statement in re.findall(r"\basm\b.*?;", source.read_text(), re.S):
            if re.search(r"s_mov\w*\s+m0", statement):
                writers += 1
                assert re.search(r":[^:]*\"m0\"[^:]*\)\s*;$", statement), f"{source.name}: {statement}"
    assert writers > 0


@pytest.mark.skipif(not LIBRARY.exists() or not OBJDUMP.exists(), reason="needs the built library and llvm-objdump")
def test_scalar_registers_of_loads_and_stores(tmp_path):
    objects = list(code_objects(LIBRARY.read_bytes()))
    assert objects
    loads, found = 0, []
    for n, image in enumerate(objects):
        path = tmp_path / f"{n}.o"
        path.write_bytes(image)
        text = subprocess.run([str(OBJDUMP), "-d", "--no-show-raw-insn", str(path)], capture_output=True, text=True,
                              check=True).stdout
        code = parse(text)
        loads += sum(VMEM.match(m) is not None and " lds" in args for m, args in code[0])
        found += too_early(*code)
    assert loads > 0  # (the loads into LDS are written in assembly)
    assert not found, f"{len(found)} read too early, as {found[:3]}"
