"""Matrix instructions of the built library, read from its disassembly: on every path, also over
branches, eight wait states lie between one and whatever reads or overwrites its result.

The hardware does not hold such an access back; the compiler counts. It has been seen to miss the
first instruction of a block that two others lead to, and the result read there was an old one."""
from __future__ import annotations

import re
import struct
import subprocess
from pathlib import Path

import pytest

from vllm_expert_cache import _lib

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
WAIT = 8  # v_mfma_f32_16x16x32 (four passes of four clocks) on gfx950
MATRIX = {"v_mfma_f32_16x16x32_bf16", "v_mfma_f32_16x16x32_f16"}


def _code_object(so: bytes) -> bytes:
    """The gfx950 entry of the offload bundle in a library."""
    at = so.index(b"__CLANG_OFFLOAD_BUNDLE__")
    count, = struct.unpack_from("<Q", so, at + 24)
    p = at + 32
    for _ in range(count):
        offset, size, length = struct.unpack_from("<QQQ", so, p)
        name = so[p + 24:p + 24 + length].decode()
        p += 24 + length
        if name.endswith("gfx950"):
            return so[at + offset:at + offset + size]
    raise AssertionError("no code for gfx950")


def _registers(text: str) -> set:
    out = set()
    for kind, a, b in re.findall(r"\b([va])\[(\d+):(\d+)\]", text):
        out.update((kind, i) for i in range(int(a), int(b) + 1))
    out.update((kind, int(a)) for kind, a in re.findall(r"\b([va])(\d+)\b", text))
    return out


def _kernels(listing: str):
    """(name, [(address, operation, operands)]) of every function."""
    name, code = None, []
    for line in listing.splitlines():
        head = re.match(r"^[0-9a-f]+ <(.+)>:$", line)
        if head:
            if code:
                yield name, code
            name, code = head.group(1), []
            continue
        m = re.match(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):", line)
        if m:
            code.append((int(m.group(3), 16), m.group(1), m.group(2)))
    if code:
        yield name, code


def _target(address: int, operands: str) -> int:
    words = int(operands.split()[0])
    return address + 4 + 4 * (words - 65536 if words >= 32768 else words)


def _too_early(code) -> list:
    """(address of a matrix instruction, address that touches its result, wait states between)."""
    at = {address: i for i, (address, _, _) in enumerate(code)}
    found = []
    for i, (address, op, operands) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        assert op in MATRIX, op
        result = _registers(operands.split(", ")[0])
        todo, seen = [(i + 1, 0)], {}
        while todo:
            p, waited = todo.pop()
            while p < len(code) and waited < WAIT and seen.get(p, WAIT) > waited:
                seen[p] = waited
                here, op, operands = code[p]
                if op == "s_endpgm":
                    break
                if op == "s_nop":
                    waited += int(operands) + 1
                elif op == "s_branch":
                    p, waited = at[_target(here, operands)], waited + 1
                    continue
                else:
                    if op.startswith("v_mfma"):
                        # adding to the same registers, or writing them anew, is held back
                        parts = operands.split(", ")
                        touched = _registers(parts[1] + " " + parts[2])
                    else:
                        touched = _registers(operands) if not op.startswith("s_") else set()
                    if touched & result:
                        found.append((hex(address), hex(here), waited))
                        break
                    if op.startswith("s_cbranch"):
                        todo.append((at[_target(here, operands)], waited + 1))
                    waited += 1
                p += 1
    return found


def test_the_reading_of_a_listing():
    listing = """
0000000000000000 <k>:
	v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[0:3]  // 000000000000: D3B50000 0
	s_cbranch_vccnz 2                                          // 000000000008: BF870002 <k+0x14>
	s_nop 7                                                    // 00000000000C: BF800007
	s_nop 0                                                    // 000000000010: BF800000
	v_mov_b32_e32 v4, v2                                       // 000000000014: 7E080302
	s_endpgm                                                   // 000000000018: BF810000
"""
    (name, code), = _kernels(listing)
    assert name == "k" and len(code) == 6
    assert _too_early(code) == [("0x0", "0x14", 1)]
    assert not _too_early(list(_kernels(listing.replace("cbranch_vccnz 2", "cbranch_vccnz 0")))[0][1])
    assert _target(0x18, "65534") == 0x14


def test_no_matrix_result_is_touched_too_early(tmp_path):
    if not OBJDUMP.exists():
        pytest.skip(f"no {OBJDUMP}")
    obj = tmp_path / "kernels.o"
    obj.write_bytes(_code_object(Path(_lib.library_path()).read_bytes()))
    listing = subprocess.run([str(OBJDUMP), "-d", "--mcpu=gfx950", str(obj)], check=True,
                             capture_output=True, text=True).stdout
    products, bad = 0, {}
    for name, code in _kernels(listing):
        products += sum(op.startswith("v_mfma") for _, op, _ in code)
        early = _too_early(code)
        if early:
            bad[name] = early
    assert products > 1000
    assert not bad, bad
