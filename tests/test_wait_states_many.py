"""The same reading of matrix results as in test_wait_states.py for every device code of the
library: also that of the operators for many tokens, whose products are in 8-bit integers."""
from __future__ import annotations

import struct
import subprocess
from pathlib import Path

import pytest

import test_wait_states as one
from vllm_expert_cache import _lib

INT8 = "v_mfma_i32_16x16x64_i8"  # four passes of four clocks, like the others


def _code_objects(so: bytes) -> list:
    """The gfx950 entries of all offload bundles in a library."""
    found, at = [], so.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        count, = struct.unpack_from("<Q", so, at + 24)
        p = at + 32
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", so, p)
            name = so[p + 24:p + 24 + length].decode()
            p += 24 + length
            if name.endswith("gfx950"):
                found.append(so[at + offset:at + offset + size])
        at = so.find(b"__CLANG_OFFLOAD_BUNDLE__", p)
    return found


def test_no_matrix_result_is_touched_too_early_in_any_code(tmp_path, monkeypatch):
    if not one.OBJDUMP.exists():
        pytest.skip(f"no {one.OBJDUMP}")
    monkeypatch.setattr(one, "MATRIX", one.MATRIX | {INT8})
    objects = _code_objects(Path(_lib.library_path()).read_bytes())
    assert len(objects) == 2
    products, bad = {}, {}
    for i, data in enumerate(objects):
        obj = tmp_path / f"kernels{i}.o"
        obj.write_bytes(data)
        listing = subprocess.run([str(one.OBJDUMP), "-d", "--mcpu=gfx950", str(obj)], check=True,
                                 capture_output=True, text=True).stdout
        for name, code in one._kernels(listing):
            for _, op, _ in code:
                if op.startswith("v_mfma"):
                    products[op] = products.get(op, 0) + 1
            early = one._too_early(code)
            if early:
                bad[name] = early
    assert set(products) == one.MATRIX and products[INT8] > 100
    assert not bad, bad
