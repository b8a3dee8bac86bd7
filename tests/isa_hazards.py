"""Wait states between the instructions of the kernels built here.

gfx950 does not interlock some pairs of dependent instructions: a fixed number of
others (or s_nop) has to stand between them.  The compiler counts those for the
instructions that it selects, but it looks neither into inline assembly nor, for
most of the pairs, at its registers.  This reads the assembly of the library's own objects
and looks for such a pair that is too close, over every path that leads to it.

The pairs are those of AMD's CDNA3 ISA document, "manually inserted wait states", as far as the
kernels' inline assembly can make them (of the MFMA results one more, as the compiler keeps on gfx950):

  VALU writes an SGPR          -> VMEM reads it                        5
  VALU writes an SGPR          -> v_readlane / v_writelane selects by it  4
  SALU writes M0               -> VMEM -> LDS copy                     1
  VALU writes a VGPR           -> MFMA reads it                        2
  VALU writes a VGPR           -> v_permlane swap, DPP read it         2
  VALU writes a VGPR           -> v_readlane / v_readfirstlane read it 1
  MFMA (8 passes) writes       -> VALU, VMEM, LDS read or overwrite it 12
"""
from __future__ import annotations

import re
import subprocess
from pathlib import Path

from rdnattention import _build

LLVM = Path("/opt/rocm/llvm/bin")


def disassemble(obj: Path, tmp: Path) -> str:
    """Assembly of the gfx950 code in a built object ("" where it has none)."""
    fat, code = tmp / (obj.name + ".fat"), tmp / (obj.name + ".co")

    def run(*cmd):
        return subprocess.run([str(c) for c in cmd], capture_output=True, text=True, check=True).stdout

    run(LLVM / "llvm-objcopy", f"--dump-section=.hip_fatbin={fat}", obj, "/dev/null")
    run(LLVM / "clang-offload-bundler", "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
        f"--input={fat}", f"--output={code}")
    return run(LLVM / "llvm-objdump", "-d", "--no-show-raw-insn", code)


_REG = re.compile(r"\b(vcc|exec|m0)(?:_lo|_hi)?\b|\b([vsa])\[(\d+):(\d+)\]|\b([vsa])(\d+)\b")


def _regs(operand: str):
    out = set()
    for m in _REG.finditer(operand):
        if m.group(1):
            out.add(m.group(1))
        elif m.group(2):
            out.update(f"{m.group(2)}{i}" for i in range(int(m.group(3)), int(m.group(4)) + 1))
        else:
            out.add(m.group(5) + m.group(6))
    return out


class Instr:
    __slots__ = ("op", "text", "at", "defs", "uses", "target", "states", "valu", "vmem", "lds_copy", "mfma", "ds")

    def __init__(self, text, at, target):
        self.text, self.at, self.target = text, at, target
        self.op, _, rest = text.partition(" ")
        ops = [o.strip() for o in rest.split(",")] if rest.strip() else []
        op = self.op
        self.mfma = op.startswith(("v_mfma", "v_smfma"))
        self.valu = op.startswith("v_") and not self.mfma
        self.vmem = op.startswith(("buffer_", "global_", "flat_", "scratch_"))
        self.ds = op.startswith("ds_")
        self.lds_copy = "_lds_" in op and self.vmem or self.vmem and re.search(r"\blds\b", rest) is not None
        self.states = int(ops[0], 0) + 1 if op == "s_nop" else 1
        n = 1  # operands that are written
        if op.startswith(("v_mad_u64_u32", "v_mad_i64_i32", "v_div_scale", "v_add_co", "v_sub_co", "v_addc_co", "v_subb_co",
                          "v_subrev_co", "v_subbrev_co", "v_permlane32_swap", "v_permlane16_swap", "v_swap")):
            n = 2
        elif op.startswith("s_") and (op.startswith(("s_cmp", "s_bitcmp", "s_cbranch", "s_branch", "s_waitcnt", "s_nop",
                                                     "s_barrier", "s_setprio", "s_endpgm", "s_store", "s_sleep"))):
            n = 0
        elif self.vmem and (self.lds_copy or "_store" in op):
            n = 0
        elif self.ds and op.startswith("ds_write"):
            n = 0
        self.defs = set().union(*map(_regs, ops[:n])) if n else set()
        self.uses = set().union(*map(_regs, ops[n:])) if ops[n:] else set()
        if n == 2 and "swap" in op or op.startswith(("v_writelane", "v_dot2c", "v_fmac", "v_pk_fmac")):
            self.uses |= set().union(*map(_regs, ops[:n]))
        if op.endswith("_e32") and op.startswith(("v_cndmask", "v_addc", "v_subb")):
            self.uses.add("vcc")


def kernels(asm: str):
    """{function: [Instr]} of llvm-objdump's output."""
    out, cur = {}, None
    for line in asm.splitlines():
        head = re.match(r"[0-9a-f]+ <(\S+)>:$", line)
        if head:
            cur = out.setdefault(head.group(1), [])
            base = int(line.split()[0], 16)
            continue
        m = re.match(r"\s+(\S.*?)\s*//\s*([0-9A-F]+):?(.*)$", line)
        if cur is None or not m:
            continue
        target = None
        t = re.search(r"<\S+?(?:\+0x([0-9a-f]+))?>\s*$", m.group(3))
        if t:
            target = base + int(t.group(1) or "0", 16)
        cur.append(Instr(m.group(1), int(m.group(2), 16), target))
    return out


def _sgprs(regs):
    return {r for r in regs if r[0] == "s" or r == "vcc"}


def _vgprs(regs):
    return {r for r in regs if r[0] in "va" and r != "vcc"}


def rules(i: Instr):
    """(states, registers, kind of writer) that instruction i needs."""
    if i.vmem:
        yield 5, _sgprs(i.uses), "valu"
        if i.lds_copy:
            yield 1, {"m0"}, "salu"
    if i.op.startswith(("v_readlane", "v_writelane")):
        yield 4, _sgprs(_regs(i.text.split(",")[2])), "valu"
    if i.mfma or "swap" in i.op or "row_" in i.text or "quad_perm" in i.text:
        yield 2, _vgprs(i.uses), "valu"
    if i.op.startswith(("v_readlane", "v_readfirstlane")):
        yield 1, _vgprs(i.uses), "valu"
    if i.valu or i.vmem or i.ds:
        yield 12, _vgprs(i.uses | i.defs), "mfma"


def too_close(code):
    """[(writer, reader, states between, states needed)] of one function."""
    index = {i.at: n for n, i in enumerate(code)}
    preds = [[] for _ in code]
    for n, i in enumerate(code):
        if i.target in index:
            preds[index[i.target]].append(n)
        if n + 1 < len(code) and i.op not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            preds[n + 1].append(n)

    def wrote(i, kind):
        return i.valu if kind == "valu" else i.mfma if kind == "mfma" else i.op.startswith("s_")

    found = []
    for n, i in enumerate(code):
        for need, regs, kind in rules(i):
            if not regs:
                continue
            todo, seen = [(p, 0, frozenset(regs)) for p in preds[n]], {}
            while todo:
                at, states, want = todo.pop()
                if states >= need or seen.get((at, want), need) <= states:
                    continue
                seen[at, want] = states
                w = code[at]
                hit = w.defs & want
                if hit and wrote(w, kind):
                    found.append((w, i, states, need))
                want = want - hit  # written again since: an earlier write does not count
                if want:
                    todo += [(p, states + w.states, want) for p in preds[at]]
    return found


def report(code):
    """A line for each pair in {function: [Instr]} that is too close."""
    return [f"{name}: {w.text}  -> {i.text}: {have} wait states, {need} needed"
            for name, instrs in code.items() for w, i, have, need in too_close(instrs)]
