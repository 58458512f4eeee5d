"""CPU: the built kernels' code keeps the wait states that the hardware does not keep by itself around loads to LDS. The
compiler keeps them between its own instructions, but puts nothing inside an inline assembly statement, where the direct loads
stand, and does not look at what such a statement reads:

  a scalar write of M0, then a load to LDS (M0 is where it goes): one instruction in between;
  a vector write of a scalar register, then a memory instruction that reads it: five.
"""

import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "flower_amd", "libflower_amd.so")
OBJDUMP = next((p for p in ("/opt/rocm/llvm/bin/llvm-objdump", "/opt/rocm/lib/llvm/bin/llvm-objdump") if os.path.exists(p)), None)


def sgprs(operand):
    out = {"vcc"} if "vcc" in operand else set()
    for one, lo, hi in re.findall(r"\bs(?:(\d+)\b|\[(\d+):(\d+)\])", operand):
        out |= {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return out


def faults(lines):
    """(kernel, instruction, what) for each place in the disassembly that lacks its wait states, read from top to bottom."""
    kernel, m0, written, found, loads = None, 0, {}, [], 0
    for line in lines:
        head = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if head:
            kernel, m0, written = head.group(1), 0, {}
            continue
        text = line.split("//")[0].strip()
        if not text:
            continue
        op, _, rest = text.partition(" ")
        if op.startswith(("global_", "buffer_")):
            if "_lds_" in op or text.endswith(" lds"):
                loads += 1
                if m0 > 0:
                    found.append((kernel, text, "M0 just written"))
            late = [r for r in sgprs(rest) if written.get(r, 0) > 0]
            if late:
                found.append((kernel, text, f"{late} written by the vector unit"))
        states = int(rest, 0) + 1 if op == "s_nop" else 1
        m0, written = max(0, m0 - states), {r: n - states for r, n in written.items() if n > states}
        to = re.sub(r"\[.*?\]", lambda m: m.group().replace(",", ";"), rest).split(",")[0].strip()
        if op.startswith("s_") and to == "m0":
            m0 = 1
        if op.startswith(("v_cmp_", "v_readlane", "v_readfirstlane")):
            written.update({r: 5 for r in sgprs(to)})
    return found, loads


def test_the_rule_finds_what_it_is_for():
    bad = """0000 <k>:
        s_mov_b32 m0, s2 // 00
        global_load_lds_dwordx4 v2, s[4:5]
        v_readlane_b32 s7, v1, 3
        s_nop 3
        buffer_load_dwordx4 v1, s[4:7], 0 offen"""
    good = bad.replace("m0, s2 // 00", "m0, s2\ns_nop 0").replace("s_nop 3", "s_nop 4")
    assert len(faults(bad.splitlines())[0]) == 2 and faults(good.splitlines()) == ([], 1)


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump of ROCm")
def test_direct_loads_to_lds_keep_their_wait_states(tmp_path):
    from flower_amd import _lib
    _lib.load()
    data = open(LIB, "rb").read()
    at = [m.start() for m in re.finditer(b"\x7fELF", data)][1:] + [len(data)]          # the device code objects within
    assert len(at) > 1
    loads = 0
    for n, (begin, end) in enumerate(zip(at, at[1:])):
        path = tmp_path / f"{n}.elf"
        path.write_bytes(data[begin:end])
        text = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", "--no-show-raw-insn", str(path)], capture_output=True, text=True, check=True)
        found, some = faults(text.stdout.splitlines())
        loads += some
        assert not found, (len(found), found[:4])
    assert loads > 1000                          # the GEMMs', the bf16 attention backward's and the paged attention's
