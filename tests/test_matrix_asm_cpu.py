"""The wait states that the matrix products' inline assembly owes, in the machine
code of the built library. The compiler keeps the distances of the instructions it
knows; those of csrc/tile_product.hpp written as text (matrix products into the
accumulation registers, loads into LDS whose place is in register M0) it does not
see, so a copy that it puts beside one goes unguarded. Checked here, on the
disassembly of what this tree's sources were built to:

* no vector instruction writes an operand of a matrix product into accumulation
  registers within two states before it, on any path;
* nothing but another product into the same registers touches a sum within 18
  states behind its product (more than any of its kind needs: eight passes, 11);

both in the kernels whose products are text (the others' distances the compiler
keeps), and in all:

* between `s_mov_b32 m0` and the load that reads it there is an instruction and no
  branch, and nothing else names M0.
"""

from __future__ import annotations

import re
import struct
import subprocess
from typing import NamedTuple

import pytest

from custom_cuda_kernals_amd import build

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"
BEFORE, BEHIND = 2, 18


def _code_objects(data: bytes):
    """gfx950 code objects of a library's offload bundles: the magic, a count, and of
    each entry its offset, size and the triple's length, then the triple."""
    for m in re.finditer(BUNDLE, data):
        at = m.start()
        (count,) = struct.unpack_from("<Q", data, at + len(BUNDLE))
        p = at + len(BUNDLE) + 8
        for _ in range(count if count <= 4 else 0):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            if b"gfx950" in data[p + 24:p + 24 + length]:
                yield data[at + offset:at + offset + size]
            p += 24 + length


def _registers(operand: str) -> set:
    m = re.match(r"^([va])\[(\d+):(\d+)\]$", operand)
    if m:
        return {(m[1], i) for i in range(int(m[2]), int(m[3]) + 1)}
    m = re.match(r"^([va])(\d+)$", operand)
    return {(m[1], int(m[2]))} if m else set()


def _products_as_text(kernel: str) -> bool:
    """Tiles of 8 x 8 fragments a wave, and MXFP4 tiles loaded straight into LDS (Product::kSumsApart); from the
    mangled template arguments <..., WP, WQ, FP, FQ, DIRECT, ...>."""
    m = re.search(r"(?:rows_product|grouped_weights).*Li\dELi\dELi(\d)ELi(\d)ELb(\d)E", kernel)
    return bool(m) and ((m[1], m[2]) == ("8", "8") or ("ElemFP4" in kernel and m[3] == "1"))


class Instruction(NamedTuple):
    op: str
    operands: list  # without their modifiers
    line: str

    @property
    def states(self) -> int:
        return 1 + int(self.operands[0]) if self.op == "s_nop" else 1

    @property
    def target(self) -> str | None:
        return self.operands[0] if re.match(r"s_c?branch", self.op) else None

    def stores(self) -> bool:
        return self.op.startswith(("ds_write", "global_store", "buffer_store", "flat_store", "scratch_store"))

    def reads(self) -> set:
        return set().union(*map(_registers, self.operands if self.stores() else self.operands[1:]))

    def writes(self) -> set:
        return set() if self.stores() or not self.operands else _registers(self.operands[0])


def _kernels(lines):
    """(name, instructions, index of each label) of a disassembly."""
    name, code, labels = "", [], {}
    for raw in lines:
        line = raw.split("//")[0].strip()
        label = re.match(r"^(?:[0-9a-f]+ )?<(.*)>:$", line)
        if label and re.match(r"^L\d+$", label[1]):
            labels[label[1]] = len(code)
        elif label:
            if code:
                yield name, code, labels
            name, code, labels = label[1], [], {}
        elif m := re.match(r"^([a-z]\w+)\s*(.*)$", line):
            code.append(Instruction(m[1], [o.split(" ")[0] for o in re.split(r",\s*", m[2])] if m[2] else [], line))
    if code:
        yield name, code, labels


def _behind(code, labels, i, states):
    """Instructions that can be issued behind code[i] with fewer than `states` states between."""
    todo, nearest = [(i + 1, 0)], {}
    while todo:
        j, passed = todo.pop()
        if j >= len(code) or passed >= min(states, nearest.get(j, states)):
            continue
        nearest[j] = passed
        if code[j].target:
            todo.append((labels[code[j].target], passed + 1))
        if code[j].op not in ("s_branch", "s_endpgm"):
            todo.append((j + 1, passed + code[j].states))
    return nearest


def check(lines) -> tuple[list, dict]:
    """What is too near, and how many of each kind were looked at."""
    found, seen = [], {"products": 0, "reads": 0, "places": 0}
    for kernel, code, labels in _kernels(lines):
        if _products_as_text(kernel):
            product = [ins.op.startswith("v_mfma") for ins in code]
            reads, writes = [ins.reads() for ins in code], [ins.writes() for ins in code]
            sums = set().union(*(w for w, p in zip(writes, product) if p))
            seen["reads"] += sum(bool(r & sums) for r, p in zip(reads, product) if not p)
            for i, ins in enumerate(code):
                if product[i]:
                    seen["products"] += 1
                    if any(kind != "a" for kind, _ in writes[i]):
                        found.append((kernel, ins.line, "not into accumulation registers"))
                    for j, passed in _behind(code, labels, i, BEHIND).items():
                        if not product[j] and (reads[j] | writes[j]) & writes[i]:
                            found.append((kernel, ins.line, code[j].line, passed))
                elif ins.op.startswith("v_") and writes[i]:
                    for j, passed in _behind(code, labels, i, BEFORE).items():
                        if product[j] and reads[j] & writes[i]:
                            found.append((kernel, ins.line, code[j].line, passed))
        starts, place = set(labels.values()), None
        for i, ins in enumerate(code):
            if place is not None and (i in starts or ins.target):
                found.append((kernel, ins.line, "between a place and its load"))
            if "m0" in ins.operands:
                seen["places"] += 1
                if ins.op != "s_mov_b32" or ins.operands[0] != "m0" or place is not None:
                    found.append((kernel, ins.line, "M0"))
                place = i
            elif ins.line.endswith(" lds"):
                if place is None or i - place < 2:
                    found.append((kernel, ins.line, "no place, or only just"))
                place = None
    return found, seen


KERNEL = "<_ZN3cck12rows_productINS_8ElemBF16ENS_9CodecBF16ELb1ELi2ELi2ELi8ELi8ELb1ELb0EEEvNS_8RowsArgsE>:"
PRODUCT = "v_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], a[0:3]"


@pytest.mark.parametrize("lines,wrong", [
    (["v_mov_b32_e32 v9, v1", PRODUCT], 1),
    (["v_mov_b32_e32 v9, v1", "s_nop 0", PRODUCT], 1),
    (["v_mov_b32_e32 v9, v1", "s_nop 1", PRODUCT], 0),
    (["v_accvgpr_write_b32 a2, v1", "s_nop 0", PRODUCT], 1),
    (["v_mov_b32_e32 v9, v1", "s_nop 1", "v_mov_b32_e32 v12, v1", PRODUCT], 0),
    (["v_mov_b32_e32 v9, v1", "s_branch L1", "<L0>:", "s_nop 7", "<L1>:", PRODUCT], 1),
    (["<L0>:", PRODUCT, "s_nop 7", "v_mov_b32_e32 v9, v1", "s_cbranch_scc0 L0"], 1),
    ([PRODUCT, "v_accvgpr_read_b32 v1, a3"], 1),
    ([PRODUCT, "s_nop 15", "s_nop 0", "v_accvgpr_read_b32 v1, a3"], 1),
    ([PRODUCT, "s_nop 15", "s_nop 1", "v_accvgpr_read_b32 v1, a3"], 0),
    ([PRODUCT, PRODUCT, "v_accvgpr_read_b32 v1, a4"], 0),
    ([PRODUCT, "ds_write_b128 v20, a[0:3]"], 1),
    (["<L0>:", "v_accvgpr_read_b32 v1, a3", "s_nop 15", "s_nop 15", PRODUCT, "s_cbranch_scc0 L0"], 1),
    ([PRODUCT, "s_cbranch_scc0 L9", "s_nop 15", "s_nop 15", "<L9>:", "v_accvgpr_read_b32 v1, a3"], 1),
    (["s_mov_b32 m0, s2", "buffer_load_dwordx4 v1, s[0:3], 0 offen lds"], 1),
    (["s_mov_b32 m0, s2", "s_nop 0", "buffer_load_dwordx4 v1, s[0:3], 0 offen nt lds"], 0),
    (["s_mov_b32 m0, s2", "s_mov_b32 m0, s3", "s_nop 0", "buffer_load_dword v1, s[0:3], 0 offen lds"], 1),
    (["s_nop 0", "buffer_load_dword v1, s[0:3], 0 offen lds"], 1),
    (["s_mov_b32 m0, s2", "<L3>:", "s_nop 0", "buffer_load_dword v1, s[0:3], 0 offen lds"], 1),
    (["s_mov_b32 m0, s2", "s_add_u32 s4, m0, s5", "s_nop 0", "buffer_load_dword v1, s[0:3], 0 offen lds"], 1)])
def test_the_check_finds_what_is_too_near(lines, wrong):
    assert len(check([KERNEL, "s_nop 7", *lines])[0]) == wrong


def test_distances_in_the_built_library(tmp_path):
    total = {"products": 0, "reads": 0, "places": 0}
    for i, code in enumerate(_code_objects(build.LIB.read_bytes())):
        if b"rows_product" not in code:
            continue
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        text = subprocess.run([OBJDUMP, "-d", "--symbolize-operands", "--no-show-raw-insn", str(path)], check=True,
                              capture_output=True, text=True).stdout
        found, seen = check(text.splitlines())
        assert not found, (len(found), found[:5])
        total = {k: total[k] + seen[k] for k in total}
    assert min(total.values()) > 500, total  # the kernels were there, and read as expected
