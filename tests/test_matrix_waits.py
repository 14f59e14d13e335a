"""Waits between a matrix instruction and the first use of its result, in the built library.

The hardware does not hold back an instruction that reads the registers of a matrix instruction still under way: the
compiler counts the cycles between and fills them up.  Where the two stand on different sides of a branch it has been seen
to count along one of the paths only, so that a result was read before it was there.  This walks all paths of every
kernel.  No GPU is needed: the code is that of this project's own kernels, as the disassembler prints it.
"""

import os
import re
import shutil
import subprocess

import pytest

from accelerated_scan import _abi

# Cycles from the issue of the instruction to that of one that may read its result: eight and ten are what the compiler keeps
# on a straight path.
WAITS = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x4_f32": 10}
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
STORES = ("ds_write", "global_store", "buffer_store", "flat_store", "scratch_store", "ds_min", "ds_add", "global_atomic")
REGISTER = re.compile(r"(?<![a-z0-9_])([va])(?:\[(\d+):(\d+)\]|(\d+))(?![0-9])")


def registers(text):
    found = set()
    for kind, first, last, one in REGISTER.findall(text):
        found.update((kind, i) for i in range(int(first or one), int(last or one) + 1))
    return found


class Code:
    """The instructions of a kernel: operation, registers written and read, places where it goes on."""

    def __init__(self, lines):
        self.ops, self.text = [], []
        at, jumps = {}, []
        for line in lines:
            body, _, note = line.partition("//")
            body = body.strip()
            if not body:
                continue
            at[int(note.split(":")[0], 16)] = len(self.ops)
            op, _, rest = body.partition(" ")
            operands = rest.split(",")
            # a bracketed pair like v[0:3] holds no comma, so the first operand is whole
            writes = set() if op.startswith(STORES) else registers(operands[0])
            reads = registers(rest if op.startswith(STORES) else ",".join(operands[1:]))
            sources = registers(",".join(operands[1:3])) if op.startswith("v_mfma") else reads
            jump = None
            if op.startswith(("s_cbranch", "s_branch")):
                address, offset = int(note.split(":")[0], 16), int(rest.strip())
                jump = address + 4 + 4 * (offset - 65536 if offset >= 32768 else offset)
            wait = int(rest, 0) + 1 if op == "s_nop" else 1
            self.ops.append((op, writes, sources, wait))
            self.text.append(body)
            jumps.append(jump)
        self.next = []
        for i, (op, jump) in enumerate(zip((o[0] for o in self.ops), jumps)):
            follow = [] if op in ("s_endpgm", "s_branch") or i + 1 == len(self.ops) else [i + 1]
            self.next.append(follow + ([at[jump]] if jump is not None else []))

    def early_uses(self):
        """(instruction, user, cycles) for every use of a result that can come too early."""
        most = max(WAITS.values())
        for i, (op, writes, _, _) in enumerate(self.ops):
            if not op.startswith("v_mfma"):
                continue
            need, seen = WAITS[op], {}
            todo = [(n, 0, frozenset(writes)) for n in self.next[i]]
            while todo:
                j, passed, live = todo.pop()
                if passed >= min(need, most) or not live or seen.get((j, live), need) <= passed:
                    continue
                seen[j, live] = passed
                _, written, read, wait = self.ops[j]
                if live & read:
                    yield self.text[i], self.text[j], passed
                live -= written | read
                todo += [(n, passed + wait, live) for n in self.next[j]]


def kernels(text):
    name, lines = None, []
    for line in text.splitlines():
        head = re.match(r"^[0-9a-f]+ <(\S+)>:", line)
        if head:
            if name:
                yield name, lines
            name, lines = head[1], []
        elif name and "//" in line:
            lines.append(line)
    if name:
        yield name, lines


def test_the_walk_finds_an_early_use_behind_a_branch():
    listing = """
        v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], 0  // 000000000100: 00
        s_cbranch_vccnz 3  // 000000000108: 00
        v_add_f32_e32 v20, v21, v22  // 00000000010C: 00
        s_nop 7  // 000000000110: 00
        v_add_f32_e32 v20, v21, v22  // 000000000114: 00
        v_mul_f32_e32 v12, v8, v1  // 000000000118: 00
        s_endpgm  // 00000000011C: 00"""
    (found,) = Code(listing.strip().splitlines()).early_uses()
    assert found[1].startswith("v_mul") and found[2] == 1
    assert not list(Code(listing.replace("s_cbranch_vccnz 3", "s_nop 6").strip().splitlines()).early_uses())


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_results_of_matrix_instructions_are_waited_for(tmp_path):
    library = shutil.copy(_abi.load()._name, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", library], cwd=tmp_path, check=True, capture_output=True)
    checked, early = 0, []
    for part in sorted(p for p in os.listdir(tmp_path) if "gfx950" in p):
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", part], cwd=tmp_path, check=True, capture_output=True,
                                 text=True).stdout
        if "v_mfma" not in listing:
            continue
        for name, lines in kernels(listing):
            if any("v_mfma" in line for line in lines):
                checked += 1
                early += [(name, *use) for use in Code(lines).early_uses()]
    assert checked >= 3 * 2 * 7  # three types, two key sizes, seven kernels with matrix instructions
    assert not early, early[:5]
