"""Wait states around conversions in inline assembly, in the assembly that the sources compile to.

The compiler counts wait states for instructions that it sees, not for those of an assembly statement (common.h's v_cvt_pk_bf16_f32).  A matrix instruction
may read what a vector instruction wrote two wait states later at the earliest; a conversion may read a matrix instruction's result once the instruction is
through (8 wait states for the 16 x 16 forms as the compiler itself leaves them, 20 for the longest 32 x 32 form; asked for here: 12 and 20).  Every path through a
kernel is followed from each such instruction; any other instruction is one wait state, s_nop n is n + 1."""
import os
import re
import subprocess

import pytest

from custom_d_fine_amd.csrc import build

SOURCES = ["attn.hip", "stem.hip", "stem3.hip", "conv3s.hip"]       # the ones whose conversions stand next to matrix instructions
NO_RESULT = ("global_store", "buffer_store", "flat_store", "ds_write", "s_", "v_cmp")


def _registers(operand):
    m = re.match(r"-?\|?([va])(?:\[(\d+):(\d+)\]|(\d+)\b)", operand.strip())
    if not m:
        return set()
    first, last = (m[2], m[3]) if m[2] else (m[4], m[4])
    return {(m[1], i) for i in range(int(first), int(last) + 1)}


class _Instruction:
    def __init__(self, text, in_asm):
        self.text, (self.op, *rest) = text, text.split(None, 1)
        operands = re.split(r",(?![^\[]*\])", rest[0]) if rest else []
        at = 0 if self.op.startswith(NO_RESULT) else 1
        self.result = set().union(*map(_registers, operands[:at]))
        self.reads = set().union(*map(_registers, operands[at:]))
        self.matrix = "v_mfma" in self.op
        self.conversion = in_asm and self.op.startswith("v_") and not self.matrix
        self.states = int(operands[0], 0) + 1 if self.op == "s_nop" else 1
        self.target = operands[0].strip() if self.op.startswith(("s_branch", "s_cbranch")) else None


def _instructions(body):
    """The instructions of one kernel; each knows the places that may follow it."""
    out, labels, in_asm = [], {}, False
    for line in body.split("\n"):
        if "#ASMSTART" in line or "#ASMEND" in line:
            in_asm = "#ASMSTART" in line
            continue
        line = re.split(r";|//", line)[0].strip()
        label = re.match(r"(\.LBB\w+):", line)
        if label:
            labels[label[1]] = len(out)
        elif line and not line.startswith("."):
            out.append(_Instruction(line, in_asm))
    for n, i in enumerate(out):
        i.next = [] if i.op in ("s_endpgm", "s_branch") else [n + 1]
        if i.target:
            i.next.append(labels[i.target])
        i.next = [x for x in i.next if x < len(out)]
    return out


def _reader_within(code, start, limit, reader):
    """An instruction that `reader` names, that reads what code[start] wrote fewer than `limit` wait states later, on some path; None if there is none."""
    best, todo = {}, [(n, 0, frozenset(code[start].result)) for n in code[start].next]
    while todo:
        n, states, live = todo.pop()
        i = code[n]
        if states >= limit or not live or best.get((n, live), limit) <= states:
            continue
        best[n, live] = states
        if reader(i) and i.reads & live:
            return i
        todo += [(x, states + i.states, live - i.result) for x in i.next]
    return None


def _too_early(assembly):
    found = []
    for m in re.finditer(r"^(_Z\w+):[^\n]*\n(.*?)^\.Lfunc_end", assembly, re.S | re.M):
        code = _instructions(m[2])
        for n, i in enumerate(code):
            late = None
            if i.conversion and i.result:
                late = _reader_within(code, n, 2, lambda x: x.matrix)
            elif i.matrix:
                late = _reader_within(code, n, 20 if "32x32" in i.op else 12, lambda x: x.conversion)
            if late:
                found.append(f"{m[1]}: {i.text} -> {late.text}")
    return found


def test_the_search_itself():
    wrap = lambda *lines: "_Zk:\n" + "\n".join(lines) + "\n.Lfunc_end0:\n"  # noqa: E731
    convert, product = [";;#ASMSTART", "v_cvt_pk_bf16_f32 v5, v1, v2", ";;#ASMEND"], "v_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], a[0:3]"
    assert _too_early(wrap(*convert, "s_nop 0", product)) and _too_early(wrap(*convert, product))
    assert not _too_early(wrap(*convert, "s_nop 1", product)) and not _too_early(wrap(*convert, "v_mov_b32 v5, 0", product))
    loop = [".LBB0_1:", product, "s_nop 1", *convert, "s_cbranch_vccnz .LBB0_1", "s_endpgm"]
    assert _too_early(wrap(*loop)) and not _too_early(wrap(*loop[:-2], "s_nop 0", *loop[-2:]))
    back = ["v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]", "s_nop 7", *convert]
    assert _too_early(wrap(*back)) and not _too_early(wrap(back[0], "s_nop 11", *back[1:]))


@pytest.mark.parametrize("source", SOURCES)
def test_conversions_and_matrix_instructions_keep_their_distance(tmp_path, source):
    out = str(tmp_path / "kernels.s")
    subprocess.run([build._hipcc(), *build.COMMON, *build.sources()[source], "-S", "--cuda-device-only", os.path.join(build.HERE, source), "-o", out],
                   check=True, stderr=subprocess.DEVNULL)
    with open(out) as f:
        assembly = f.read()
    assert "v_mfma" in assembly and "#ASMSTART" in assembly
    assert not _too_early(assembly)
