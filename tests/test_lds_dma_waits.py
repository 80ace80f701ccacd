"""The wait states in front of every LDS DMA of the built gfx950 code.

The hardware does not hold an LDS DMA (global_load_lds_*) back for a register written right before
it: a scalar write of M0 needs one wait state before it, a vector instruction's write of a
scalar register that it reads five.  The compiler inserts them for its own instructions and not for
inline asm, which is how the kernels issue their DMA, so they are counted here in the code itself,
along every path.
"""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from jjjetson_ops_amd import build

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
LINE = re.compile(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):")
REG = re.compile(r"\bs(\d+)\b|\bs\[(\d+):(\d+)\]|\b(vcc|m0|exec)\b")
AFTER_M0, AFTER_VALU = 1, 5
TWO_DESTINATIONS = ("v_add_co", "v_addc_co", "v_sub_co", "v_subb_co", "v_subrev_co", "v_subbrev_co", "v_div_scale",
                    "v_mad_u64", "v_mad_i64")


def _registers(operand):
    out = set()
    for one, first, last, name in REG.findall(operand):
        if name:
            out.add(name)
        else:
            out.update(range(int(one or first), int(one or last) + 1))
    return out


def _functions(text):
    """[(name, [(mnemonic, operands, address)])] of a disassembly."""
    out = []
    for line in text.splitlines():
        if line.endswith(">:"):
            out.append((line.split("<", 1)[1][:-2], []))
        elif out:
            m = LINE.match(line)
            if m:
                out[-1][1].append((m[1], m[2], int(m[3], 16)))
    return out


def _successors(code, i, at):
    op, args, address = code[i]
    to = []
    if op == "s_branch" or op.startswith("s_cbranch"):
        offset = int(args.split()[0])
        to.append(at.get(address + 4 + 4 * (offset - 65536 if offset >= 32768 else offset)))
    if op not in ("s_branch", "s_endpgm", "s_setpc_b64") and i + 1 < len(code):
        to.append(i + 1)
    return [j for j in to if j is not None]


def _too_early(code):
    """(address of the write, address of the DMA) of every pair without its wait states."""
    at = {c[2]: i for i, c in enumerate(code)}
    faults = set()
    for i, (op, args, address) in enumerate(code):
        operands = args.split(",")
        if op.startswith("s_"):
            if operands[0].strip() != "m0" or op.startswith(("s_cmp", "s_bitcmp")):
                continue
            written, need = {"m0"}, AFTER_M0
        elif op.startswith("v_"):
            written = _registers(operands[0])
            if op.startswith(TWO_DESTINATIONS):
                written |= _registers(operands[1])
            need = AFTER_VALU
            if not written:
                continue
        else:
            continue
        todo, seen = [(j, 0) for j in _successors(code, i, at)], set()
        while todo:
            j, waited = todo.pop()
            if waited >= need or (j, waited) in seen:
                continue
            seen.add((j, waited))
            nop, nargs, naddress = code[j]
            if "_lds_" in nop and nop.startswith(("global_load", "buffer_load", "scratch_load")):
                if written & (_registers(nargs) | {"m0"}):
                    faults.add((address, naddress))
            states = int(nargs.split()[0]) + 1 if nop == "s_nop" else 1
            todo += [(k, waited + states) for k in _successors(code, j, at)]
    return sorted(faults)


def _code(text):
    return [(m[1], m[2], int(m[3], 16)) for m in map(LINE.match, text.strip("\n").splitlines())]


def test_the_count():
    """The count itself, on lines written for it."""
    def faults(*lines):
        return _too_early(_code("\n".join(f"  {line}  // {4 * i:08X}: 0" for i, line in enumerate(lines))))

    dma = "global_load_lds_dwordx4 v1, s[8:9]"
    assert faults("s_mov_b32 m0, s4", dma) == [(0, 4)]
    assert faults("s_add_i32 m0, s4, 16", "s_nop 0", dma) == []
    assert faults("s_mov_b32 m0, s4", "v_mov_b32_e32 v1, v2", dma) == []
    assert faults("v_readfirstlane_b32 s9, v1", "s_nop 3", dma) == [(0, 8)]
    assert faults("v_readfirstlane_b32 s9, v1", "s_nop 4", dma) == []
    assert faults("v_readfirstlane_b32 s10, v1", dma) == []
    assert faults("v_add_co_u32_e64 v1, s[8:9], v2, v3", dma) == [(0, 4)]
    assert faults("s_mov_b32 m0, s4", "s_branch 0", dma) == []
    assert faults("v_readlane_b32 s8, v1, 3", "s_cbranch_scc1 2", "s_nop 7", "s_nop 7", dma) == [(0, 16)]


def test_every_dma_has_its_wait_states(tmp_path):
    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    shutil.copy(build.LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    kernels, faults = 0, []
    for obj in sorted(tmp_path.glob("lib.so.*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", obj], check=True, capture_output=True, text=True).stdout
        for name, code in _functions(text):
            if any("_lds_dword" in c[0] for c in code):
                kernels += 1
                faults += [(name, hex(a), hex(b)) for a, b in _too_early(code)]
    assert kernels > 40
    assert not faults, (len(faults), faults[:4])
