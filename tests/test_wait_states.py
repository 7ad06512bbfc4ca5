"""Direct-to-LDS copies in the built library, from its assembly. The copies are inline asm, which the
compiler's hazard pass does not look into, so the wait states the hardware wants between a
scalar register's write and a copy that reads it have to be in the asm:

* m0, which holds a copy's LDS address: one, after a scalar instruction;
* the scalar base: five, after a vector instruction (v_readfirstlane_b32).
"""

import os
import re
import shutil
import struct
import subprocess

import pytest

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
M0_STATES, BASE_STATES = 1, 5


def _objdump():
    for cand in ("/opt/rocm/llvm/bin/llvm-objdump", shutil.which("llvm-objdump")):
        if cand and os.path.exists(cand):
            return cand
    pytest.skip("no llvm-objdump")


def _code_objects(data: bytes):
    """The gfx950 code objects of a library's offload bundles."""
    at = data.find(MAGIC)
    while at >= 0:
        pos = at + len(MAGIC)
        (n,) = struct.unpack_from("<Q", data, pos)
        pos += 8
        for _ in range(n):
            offset, size, name_len = struct.unpack_from("<QQQ", data, pos)
            name = data[pos + 24:pos + 24 + name_len]
            pos += 24 + name_len
            if size and b"gfx950" in name:
                yield data[at + offset:at + offset + size]
        at = data.find(MAGIC, pos)


def _registers(operand: str) -> set:
    """m0, or the scalar registers of an operand: s5, s[4:5]."""
    got = set()
    if re.fullmatch(r"m0", operand):
        got.add("m0")
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        got |= {f"s{i}" for i in range(int(m[1]), int(m[2]) + 1)}
    elif re.fullmatch(r"s\d+", operand):
        got.add(operand)
    return got


def _operands(line: str) -> list:
    head, _, rest = line.partition(" ")
    return [o.strip() for o in re.split(r",\s*|\s+(?=off|offset|lds)", rest) if o.strip()]


def too_early(lines: list) -> list:
    """The copies that come too soon after a write of what they read, each with that write."""
    bad = []
    for i, line in enumerate(lines):
        if not line.startswith("global_load_lds"):
            continue
        base = set().union(*(_registers(o) for o in _operands(line))) - {"m0"}
        states, j = 0, i - 1
        while j >= 0 and states < BASE_STATES:
            prev = lines[j]
            name = prev.split(" ")[0]
            if name == "s_nop":
                states += int(prev.split()[1], 0) + 1
            else:
                dst = _registers(_operands(prev)[0]) if _operands(prev) else set()
                if "m0" in dst and states < M0_STATES:
                    bad.append((prev, line))
                if name.startswith("v_") and dst & base:
                    bad.append((prev, line))
                states += 1
            j -= 1
    return bad


def _clean(text: str) -> list:
    lines = [l.split("//")[0].strip() for l in text.splitlines()]
    return [re.sub(r"\s+", " ", l) for l in lines if l and not l.endswith(":") and not l.startswith("<")]


def test_the_rule():
    ok = ["s_add_i32 m0, s4, 16", "s_nop 0", "global_load_lds_dwordx4 v[2:3], off"]
    assert not too_early(ok) and too_early(ok[:1] + ok[2:]) == [(ok[0], ok[2])]
    read = ["v_readfirstlane_b32 s22, v1", "s_mov_b32 m0, s3", "s_nop 4", "global_load_lds_dword v2, s[22:23]"]
    assert not too_early(read) and len(too_early(read[:2] + ["s_nop 2"] + read[3:])) == 1
    assert not too_early(["v_readfirstlane_b32 s21, v1", "s_nop 0", read[3]])


def test_copies_wait(tmp_path):
    from torchtitan_amd import _lib

    objdump = _objdump()
    if not os.path.exists(_lib.library_path()):
        from torchtitan_amd import build

        build.build()
    with open(_lib.library_path(), "rb") as f:
        objects = list(_code_objects(f.read()))
    assert objects
    copies, bad = 0, []
    for i, code in enumerate(objects):
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], check=True,
                              capture_output=True, text=True).stdout
        lines = _clean(text)
        copies += sum(l.startswith("global_load_lds") for l in lines)
        bad += too_early(lines)
    assert copies > 0
    assert not bad, f"{len(bad)} of {copies} copies, the first: {bad[0]}"
