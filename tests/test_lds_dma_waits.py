"""Loads into LDS written in asm blocks keep the wait states that gfx950 wants and that
the compiler puts before its own: one between a scalar write of m0 and the load, five
between a vector instruction's write of a scalar register (a reloaded spill among
them) and a load that reads it.  Read from the assembly that the package's own flags make of the
sources; runs on the CPU, skipped where hipcc is absent."""
import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "mtlqwen_amd", "csrc")


def _scalars(text):
    """The scalar registers that operands name."""
    out = set()
    for a, b, one in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", text):
        out.update([int(one)] if one else range(int(a), int(b) + 1))
    return out


def _shortfalls(lines):
    """(loads into LDS in asm blocks, [(kernel, line, what)] of those with too few wait states before them)."""
    kernel, block, seen, before, bad = "", False, 0, [], []
    for number, line in enumerate(lines, 1):
        name = re.match(r"(_Z\w+):", line)
        if name:
            kernel, before = name.group(1), []
        if "ASMSTART" in line or "ASMEND" in line:
            block = "ASMSTART" in line
            continue
        text = line.split(";")[0].strip()
        if not text or text.startswith(".") or text.endswith(":"):
            continue
        op, operands = re.split(r"\s+", text, maxsplit=1) if re.search(r"\s", text) else (text, "")
        if block and "load_lds" in op:
            seen += 1
            reads, states = _scalars(operands), 0
            for wait, vector, m0 in reversed(before):
                if m0 and states < 1:
                    bad.append((kernel, number, "m0"))
                if vector & reads and states < 5:
                    bad.append((kernel, number, "scalar operand"))
                states += wait
        vector = set()
        if op.startswith("v_"):
            places = operands.split(",")
            vector = _scalars(places[0]) if re.match(r"s[\[\d]", places[0].strip()) else set()
            if "_co_" in op and len(places) > 1:
                vector |= _scalars(places[1])
        wait = int(operands, 0) + 1 if op == "s_nop" else 1
        before = (before + [(wait, vector, op.startswith("s_") and operands.startswith("m0"))])[-6:]
    return seen, bad


def test_shortfalls_are_found():
    asm = ["_Zk:", "v_readlane_b32 s4, v1, 0", ";;#ASMSTART", "s_mov_b32 m0, s2", "%s", "global_load_lds_dwordx4 v0, s[4:5] offset:0", ";;#ASMEND"]
    for nop, want in (("", ["m0", "scalar operand"]), ("s_nop 0", ["scalar operand"]), ("s_nop 2", ["scalar operand"]), ("s_nop 3", [])):
        assert _shortfalls([x % nop if x == "%s" else x for x in asm]) == (1, [("_Zk", 6, w) for w in want])
    assert _shortfalls([x.replace("s4", "s6").replace("%s", "s_nop 0") for x in asm]) == (1, [])


def test_lds_loads_wait(tmp_path):
    sys.path.insert(0, os.path.join(ROOT, "mtlqwen_amd"))
    import build  # the package's own build recipe (flags)
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    sources = [s for s in build.SOURCES if s.endswith(".hip") and "lds_dma" in open(os.path.join(CSRC, s)).read()]
    assert len(sources) >= 4

    def assembly(source):
        out = str(tmp_path / (source + ".s"))
        run = subprocess.run([hipcc, *build.HIPCC_FLAGS, "-w", "--offload-device-only", "-S", os.path.join(CSRC, source), "-o", out], capture_output=True,
                             text=True)
        assert run.returncode == 0, run.stderr[-2000:]
        return out

    with ThreadPoolExecutor(max_workers=len(sources)) as pool:
        for source, path in zip(sources, pool.map(assembly, sources)):
            with open(path) as lines:
                seen, bad = _shortfalls(lines)
            assert seen > 100 and not bad, f"{source}: {len(bad)} of {seen}, {bad[:3]}"
