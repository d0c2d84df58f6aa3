"""The built library's gfx950 code: the wait states that no hardware check supplies.

A memory instruction that reads a scalar register needs 5 wait states after a vector
instruction that wrote it (gfx9).  The compiler keeps them between its own instructions;
a memory instruction in an asm string has to bring them along, whatever comes before."""

import os
import re
import shutil
import subprocess

import pytest

from torch_spyre_amd import build as B

NEEDED = 5
OBJDUMP = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(shutil.which(B.HIPCC) or B.HIPCC))), "llvm", "bin",
                       "llvm-objdump")
_LINE = re.compile(r"^\s+([a-z]\w+)\s*(.*?)\s*// ([0-9A-F]{12,16}): [0-9A-F ]+(?:<(.+)\+0x([0-9a-f]+)>|<(.+)>)?\s*$")
_SYMBOL = re.compile(r"^([0-9a-f]{16}) <(.+)>:$")
_SGPR = re.compile(r"(?<![a-z0-9_])(?:s(\d+)|s\[(\d+):(\d+)\]|(vcc))(?![a-z0-9_])")


def sgprs(operand):
    """The scalar registers that an operand names (vcc: 106, 107)."""
    out = set()
    for one, lo, hi, vcc in _SGPR.findall(operand):
        out |= {106, 107} if vcc else {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return out


def parse(text):
    """[(address, op, operands, address of a branch's target)] in order."""
    code, symbols = [], {}
    for line in text.splitlines():
        s = _SYMBOL.match(line)
        if s:
            symbols[s[2]] = int(s[1], 16)
            continue
        m = _LINE.match(line)
        if m:
            code.append((int(m[3], 16), m[1], m[2].split(", ") if m[2] else [], (m[4] or m[6], int(m[5] or "0", 16)) if m[4] or m[6] else None))
    return [(at, op, ops, symbols[to[0]] + to[1] if to and op.startswith(("s_branch", "s_cbranch")) else None)
            for at, op, ops, to in code]


def written_by_valu(op, ops):
    if op.startswith(("v_readlane", "v_readfirstlane", "v_cmp_")):
        return sgprs(ops[0])
    if "_co_" in op or op.startswith("v_div_scale"):
        return sgprs(ops[1])
    return set()


def reads_as_memory(op, ops):
    if not op.startswith(("buffer_", "global_", "flat_", "scratch_")):
        return set()
    return sgprs(", ".join(ops))


def hazards(code):
    """(address of the vector instruction, of the memory instruction, wait states between them)."""
    index = {at: i for i, (at, *_) in enumerate(code)}
    found = []
    for i, (at, op, ops, _) in enumerate(code):
        regs = written_by_valu(op, ops) if op.startswith("v_") else set()
        if not regs:
            continue
        paths = [(i + 1, 0, frozenset(regs))]
        while paths:
            j, states, live = paths.pop()
            while j < len(code) and states < NEEDED and live:
                at2, op2, ops2, target = code[j]
                if live & reads_as_memory(op2, ops2):
                    found.append((at, at2, states))
                    break
                if op2.startswith("s_endpgm"):
                    break
                if op2.startswith("s_") and ops2 and not op2.startswith(("s_cmp", "s_bitcmp")):
                    live = live - sgprs(ops2[0])  # a scalar write: no such wait behind it
                states += int(ops2[0], 0) + 1 if op2 == "s_nop" else 1
                if target is not None:
                    paths.append((index[target], states, live))
                    if op2 == "s_branch":
                        break
                j += 1
    return found


def test_the_search_sees_what_it_looks_for():
    def code(*lines):
        return parse("0000000000001000 <k>:\n" + "\n".join(f"\t{x} // {0x1000 + 4 * i:012X}: 00000000{to}" for i, (x, to) in enumerate(lines)))

    lane, load = ("v_readlane_b32 s3, v220, 57", ""), ("buffer_load_dwordx4 v2, s[72:75], s3 offen lds", "")
    m0, nop = ("s_mov_b32 m0, s0", ""), lambda n: (f"s_nop {n}", "")
    assert [h[2] for h in hazards(code(lane, m0, nop(0), load))] == [2]
    assert [h[2] for h in hazards(code(lane, m0, nop(2), load))] == [4]
    assert not hazards(code(lane, m0, nop(3), load))
    assert not hazards(code(lane, ("s_mov_b32 s3, s7", ""), load))
    assert hazards(code(("v_readfirstlane_b32 s74, v1", ""), load)) and not hazards(code(("v_readfirstlane_b32 s76, v1", ""), load))
    assert hazards(code(load, m0, lane, ("s_cbranch_scc0 65530", " <k>")))  # round a loop
    assert not hazards(code(("v_add_f32_e32 v3, s3, v4", ""), load))
    assert hazards(code(("v_cmp_eq_u32_e64 s[2:3], v1, v2", ""), load))


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump beside the compiler")
def test_memory_instructions_wait_for_their_scalars(tmp_path):
    lib = shutil.copy(B.OUT, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, capture_output=True)
    objects = sorted(f for f in os.listdir(tmp_path) if f.endswith(B.ARCH))
    assert objects, "the library holds device code"
    bad, loads = [], 0
    for f in objects:
        text = subprocess.run([OBJDUMP, "-d", str(tmp_path / f)], check=True, capture_output=True,
                              text=True).stdout
        code = parse(text)
        loads += sum(op.startswith("buffer_load") and ops[-1].endswith("lds") for _, op, ops, _ in code)
        bad += [(f, hex(a), hex(b), n) for a, b, n in hazards(code)]
    assert loads, "loads into LDS are found"
    assert not bad, f"{len(bad)} memory instructions read a scalar too early: {bad[:8]}"
