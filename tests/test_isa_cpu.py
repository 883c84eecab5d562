"""What the built kernels' own machine code must not contain.

An fp32 matrix instruction reads its C operand over all its passes.  Where C is its destination the hardware and hipcc see to that; where C
is another register range, hipcc has been seen to overwrite it in the very next instruction, without a wait (a C operand that the source
uses again later, in the query gradient of attention at 96 and 128 channels: v_mfma_f32_32x32x2_f32 v[82:97], v68, v178, v[182:197], then
v_mov_b64 v[194:195]; the gradient came out wrong).  For the bf16 form it puts waits in.  No kernel may hold the fp32 form of this."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from shineon_virtual_tryon_amd import _lib

OBJDUMP = shutil.which("llvm-objdump", path=os.pathsep.join(["/opt/rocm/llvm/bin", os.environ.get("PATH", "")]))
PASSES = {"4x4": 2, "16x16": 8, "32x32": 16}


def registers(operand):
    m = re.fullmatch(r"([av])(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    first, last = (m[2], m[2]) if m[2] else (m[3], m[4])
    return {m[1] + str(i) for i in range(int(first), int(last) + 1)}


def overwritten_operands(instructions):
    """(matrix instruction, what overwrites its C operand too early) in a straight run of instructions."""
    found = []
    for i, (op, args) in enumerate(instructions):
        m = re.match(r"v_mfma_f32_(4x4|16x16|32x32)x\d+(?:_\d+b)?_?f32$", op)
        if not m:
            continue
        c = registers(args[3])
        if c == registers(args[0]):
            continue
        slots = 0
        for op2, args2 in instructions[i + 1:i + 1 + PASSES[m[1]]]:
            if slots >= PASSES[m[1]]:
                break
            if op2.startswith(("v_", "ds_read", "global_load", "buffer_load", "scratch_load")) and args2 and registers(args2[0]) & c:
                found.append((f"{op} {', '.join(args)}", f"{op2} {', '.join(args2)} after {slots} slots"))
                break
            slots += int(args2[0], 0) + 1 if op2 == "s_nop" else 1
    return found


def code_objects(path):
    """The device ELF files inside a library's offload bundles."""
    data = open(path, "rb").read()
    for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", data):
        (n,), at = struct.unpack_from("<Q", data, m.end()), m.end() + 8
        for _ in range(n):
            offset, size, length = struct.unpack_from("<QQQ", data, at)
            name = data[at + 24:at + 24 + length].decode()
            at += 24 + length
            if name.startswith("hip") and size:
                yield data[m.start() + offset:m.start() + offset + size]


def parse(line):
    m = re.match(r"\s+([a-z]\w+)(?:\s+(.*?))?\s*(?://.*)?$", line)
    return (m[1], re.split(r",\s*|\s+(?=[a-z]+:|offen|lds)", m[2]) if m[2] else []) if m else None


def test_the_rule_finds_an_early_overwrite():
    run = [parse(x) for x in ("\tv_mfma_f32_32x32x2_f32 v[82:97], v68, v178, v[182:197] // 0001", "\ts_nop 3", "\tv_mov_b64_e32 v[194:195], v[148:149]")]
    assert overwritten_operands(run) == [("v_mfma_f32_32x32x2_f32 v[82:97], v68, v178, v[182:197]", "v_mov_b64_e32 v[194:195], v[148:149] after 4 slots")]
    assert not overwritten_operands([run[0], parse("\ts_nop 15"), run[2]])
    assert not overwritten_operands([parse("\tv_mfma_f32_32x32x2_f32 v[182:197], v68, v178, v[182:197]"), run[2]])


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
def test_no_kernel_overwrites_a_matrix_instructions_operand(tmp_path):
    objects, matrix, found = 0, 0, []
    for i, blob in enumerate(code_objects(_lib.LIB_PATH)):
        objects += 1
        if b"amdgcn" not in blob[:64] and not blob.startswith(b"\x7fELF"):
            continue
        (tmp_path / f"{i}.o").write_bytes(blob)
        out = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(tmp_path / f"{i}.o")], capture_output=True, text=True, check=True).stdout
        for kernel in re.split(r"^[0-9a-f]+ <", out, flags=re.M)[1:]:
            if "v_mfma" not in kernel:
                continue
            instructions = [p for p in map(parse, kernel.split("\n")[1:]) if p]
            matrix += sum(op.startswith("v_mfma") for op, _ in instructions)
            found += [(kernel[:kernel.index(">")], *f) for f in overwritten_operands(instructions)]
    assert objects >= 15 and matrix > 10000, (objects, matrix)
    assert not found, found[:5]
