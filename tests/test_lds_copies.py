"""The built library's copies from global memory into LDS keep gfx950's wait states: the
compiler inserts none around and inside inline assembly, where most of them are issued.

One wait state between a write of m0 (the LDS address) and the copy that reads it; five between
a vector instruction's write of a scalar register and a copy that takes its address from it.
Every instruction is one, ``s_nop N`` is N + 1.
"""
import os
import re
import shutil
import subprocess

import pytest

from smat_attention_amd import _build

OBJDUMP = next((p for p in ("/opt/rocm/llvm/bin/llvm-objdump", shutil.which("llvm-objdump") or "")
                if p and os.path.exists(p)), None)


def _scalars(operand):
    """Scalar registers of an operand: s7, s[4:5]."""
    m = re.fullmatch(r"s(\d+)", operand)
    if m:
        return {int(m.group(1))}
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    return set(range(int(m.group(1)), int(m.group(2)) + 1)) if m else set()


def faults(lines):
    """(function, line) of each copy that comes too early, and the number of copies."""
    found, copies, name, at, m0, vector = [], 0, "", 0, -100, {}
    for line in lines:
        if line.endswith(">:"):
            name, at, m0, vector = line, 0, -100, {}
            continue
        word, _, rest = line.strip().partition(" ")
        rest = rest.split("//")[0]
        ops = [o for o in re.split(r"[,\s]+", rest.strip()) if o]
        if word == "s_nop":
            at += int(ops[0], 0) + 1
            continue
        if word.startswith(("global_load_lds", "buffer_load")) and (
                "_lds_" in word or "lds" in ops):
            copies += 1
            read = set().union(*(_scalars(o) for o in ops)) if ops else set()
            if at - m0 < 2 or any(at - vector.get(s, -100) < 6 for s in read):
                found.append((name, line.strip()))
        elif ops and ops[0] == "m0":
            m0 = at
        elif word.startswith("v_") and ops:
            for o in ops[:2]:                      # (a carry or a condition is the second one)
                for s in _scalars(o):
                    if o == ops[0] or re.match(r"v_(add|sub|subrev|addc|subb|div|mad)_", word):
                        vector[s] = at
        elif word.startswith("s_") and ops:        # a scalar write behind it takes its place
            for s in _scalars(ops[0]):
                vector.pop(s, None)
        at += 1
    return found, copies


def test_the_rule_sees_what_it_should():
    early = ["0 <k>:", "  s_mov_b32 m0, s4", "  global_load_lds_dwordx4 v[2:3], off"]
    assert faults(early) == ([("0 <k>:", "global_load_lds_dwordx4 v[2:3], off")], 1)
    assert faults(early[:2] + ["  s_nop 0"] + early[2:]) == ([], 1)
    base = ["0 <k>:", "  v_readlane_b32 s8, v255, 3", "  s_mov_b32 s4, m0", "  s_mov_b32 m0, s5",
            "  s_nop 1", "  global_load_lds_dwordx4 v2, s[8:9]"]
    assert len(faults(base)[0]) == 1
    assert faults(base[:4] + ["  s_nop 2"] + base[5:]) == ([], 1)
    assert faults(base[:2] + ["  s_mov_b64 s[8:9], s[2:3]"] + base[2:]) == ([], 1)


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
def test_lds_copies_keep_their_wait_states(tmp_path):
    lib = shutil.copy(_build.LIB, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True, cwd=tmp_path)
    found, copies = [], 0
    for f in sorted(os.listdir(tmp_path)):
        if "gfx950" not in f:
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", os.path.join(tmp_path, f)],
                              check=True, capture_output=True, text=True).stdout
        bad, n = faults(text.splitlines())
        found, copies = found + bad, copies + n
    assert copies > 1000
    assert not found, f"{len(found)} of {copies} copies come too early, the first {found[0]}"
