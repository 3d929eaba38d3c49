"""The built kernels' own instructions (disassembled, without a GPU).

A kernel that joined statistics with several interleaved divisions gave wrong values now
and then; in its code a ``v_div_fmas`` had its condition from a scalar write of VCC right
before it.  No kernel here has such code, and the group norm's divide nothing.
"""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from piecewiselinearembeddings_optimized_amd import capi

_OBJDUMP = shutil.which("llvm-objdump") or os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")


def _code_objects(library: bytes):
    """The gfx950 code objects of a library's offload bundles."""
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    number = lambda at: int.from_bytes(library[at:at + 8], "little")  # noqa: E731
    for found in re.finditer(magic, library):
        begin = found.start()
        at = begin + len(magic) + 8
        for _ in range(number(begin + len(magic))):
            offset, size, name = number(at), number(at + 8), number(at + 16)
            target = library[at + 24:at + 24 + name].decode()
            at += 24 + name
            if size > 0 and target.endswith("gfx950"):
                yield library[begin + offset:begin + offset + size]


@pytest.fixture(scope="module")
def divisions(tmp_path_factory):
    """Of every kernel: its name, and for each ``v_div_fmas`` the six instructions before it."""
    if not os.path.exists(_OBJDUMP):
        pytest.skip("llvm-objdump not found")
    capi.lib()
    with open(os.path.join(os.path.dirname(capi.__file__), "libple_hip.so"), "rb") as f:
        library = f.read()
    kernels = {}
    for i, code in enumerate(_code_objects(library)):
        path = tmp_path_factory.mktemp("code") / f"{i}.o"
        path.write_bytes(code)
        text = subprocess.run([_OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], capture_output=True, text=True,
                              check=True).stdout
        name, before = "", []
        for line in text.splitlines():
            if line.endswith(">:"):
                name, before = line[line.index("<") + 1:-2], []
                kernels[name] = []
            elif line.strip():
                instruction = line.split("//")[0].strip()
                if instruction.startswith("v_div_fmas"):
                    kernels[name].append(list(before))
                before = [*before[-5:], instruction]
    assert any("ple_group_forward_kernel" in k for k in kernels) and any("ple_bwd" in k for k in kernels)
    return kernels


def test_group_norm_divides_nothing(divisions):
    assert [k for k, found in divisions.items() if "ple_group" in k and found] == []


def test_no_scalar_condition_right_before_a_division(divisions):
    scalar = re.compile(r"s_\w+\s+vcc")
    assert [k for k, found in divisions.items() for before in found if any(scalar.match(i) for i in before)] == []
