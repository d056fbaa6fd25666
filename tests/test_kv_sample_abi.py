"""The C layouts of styx_kv_cache and styx_sample_params (printed by a gcc
build of the header) against their ctypes and Rust mirrors.  No GPU needed."""
from __future__ import annotations

import ctypes as C
import json
import shutil
import subprocess

import pytest

from test_abi_drift import HDR, rust_layout, rust_structs

STRUCTS = {"styx_kv_cache": ("KvCache", {"type_": "type"}), "styx_sample_params": ("SampleParams", {})}


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_mirrors_have_the_header_layout(name, tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc not available")
    from styx_amd import _lib
    mirror, renamed = STRUCTS[name]
    cls = getattr(_lib, mirror)
    fields = [f for f, _ in cls._fields_]
    src = "\n".join(["#include <stdio.h>", "#include <stddef.h>", f'#include "{HDR}"', "int main(void) {",
                     f'printf("[%zu", sizeof({name}));',
                     *[f'printf(", %zu", offsetof({name}, {f}));' for f in fields], 'printf("]"); return 0; }'])
    (tmp_path / "lay.c").write_text(src)
    subprocess.run([gcc, "-std=c11", "-o", str(tmp_path / "lay"), str(tmp_path / "lay.c")], check=True)
    size, *offs = json.loads(subprocess.run([str(tmp_path / "lay")], capture_output=True, text=True, check=True).stdout)
    assert C.sizeof(cls) == size and [getattr(cls, f).offset for f in fields] == offs
    rust = rust_structs()[name]
    assert [renamed.get(f, f) for f, _ in rust] == fields
    assert rust_layout(rust, {}) == (offs, size)
