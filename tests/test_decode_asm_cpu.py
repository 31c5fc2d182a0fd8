"""What the decode step's inline assembly owes, in the machine code of the built library: a load
into LDS goes where register M0 says, which the instruction before but one or earlier sets; between
the two there is no branch and no other use of M0. In every kernel of paged_attention.hip and
fp8_linear.hip."""

from __future__ import annotations

import subprocess

import pytest

from custom_cuda_kernals_amd import build
from tests.test_matrix_asm_cpu import OBJDUMP, _code_objects, _kernels

KERNELS = ("paged_attention", "block_product", "block_stream")


def places(lines) -> tuple[list, int]:
    """What is wrong, and how many loads were looked at."""
    found, seen = [], 0
    for kernel, code, labels in _kernels(lines):
        if not any(k in kernel for k in KERNELS):
            continue
        starts, place = set(labels.values()), None
        for i, ins in enumerate(code):
            if place is not None and (i in starts or ins.target):
                found.append((kernel, ins.line, "between a place and its load"))
            if "m0" in ins.operands:
                if ins.op != "s_mov_b32" or ins.operands[0] != "m0" or place is not None:
                    found.append((kernel, ins.line, "M0"))
                place = i
            elif ins.line.endswith(" lds") or ins.op.startswith("global_load_lds"):
                seen += 1
                if place is None or i - place < 2:
                    found.append((kernel, ins.line, "no place, or only just"))
                place = None
    return found, seen


NAME = "<_ZN3cck12_GLOBAL__N_115paged_attentionE>:"
LOAD = "global_load_lds_dwordx4 v[2:3], off nt"


@pytest.mark.parametrize("lines,wrong", [
    (["s_mov_b32 m0, s2", "s_nop 0", LOAD], 0),
    (["s_mov_b32 m0, s2", LOAD], 1),
    (["s_nop 0", LOAD], 1),
    (["s_mov_b32 m0, s2", "s_mov_b32 m0, s3", "s_nop 0", LOAD], 1),
    (["s_mov_b32 m0, s2", "s_branch L0", "<L0>:", LOAD], 2),
    (["s_mov_b32 m0, s2", "s_nop 0", LOAD, LOAD], 1),
])
def test_the_check_finds_what_is_wrong(lines, wrong):
    assert len(places([NAME, "s_nop 7", *lines])[0]) == wrong


def test_places_in_the_built_library(tmp_path):
    total = 0
    for i, code in enumerate(_code_objects(build.LIB.read_bytes())):
        if not any(k.encode() in code for k in KERNELS):
            continue
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        text = subprocess.run([OBJDUMP, "-d", "--symbolize-operands", "--no-show-raw-insn", str(path)], check=True,
                              capture_output=True, text=True).stdout
        found, seen = places(text.splitlines())
        assert not found, (len(found), found[:5])
        total += seen
    assert total > 500, total  # the kernels were there, and read as expected
