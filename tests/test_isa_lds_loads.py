"""Loads that write LDS without passing through registers (global_load_lds),
checked on the code the compiler emits (CPU only: hipcc cross-compiles gfx950).

Such a load is counted by vmcnt. A wavefront that passes a barrier before its own
have arrived lets the others read what is not there yet, and a workgroup barrier
does not wait for them by itself: on every path from such a load to a barrier the
wavefront has to wait for vmcnt(0).
"""

import os
import re
import shutil
import subprocess

import pytest

from sparda import build as B
from test_isa_dpp import kernels


def unwaited(asm_lines):
    """Barriers that some path reaches with loads to LDS still in flight: [(load, barrier index)]."""
    ins, labels = [], {}
    for l in asm_lines:
        s = l.split(";")[0].strip()
        if not s or (s.startswith(".") and not s.endswith(":")):
            continue
        if s.endswith(":"):
            labels[s[:-1]] = len(ins)
        ins.append(s)
    nexts = []
    for i, s in enumerate(ins):
        op = s.split()[0]
        n = [labels[s.split()[1]]] if op.startswith(("s_branch", "s_cbranch")) else []
        if i + 1 < len(ins) and op not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            n.append(i + 1)
        nexts.append(n)
    bad = []
    for i, s in enumerate(ins):
        if "load_lds" not in s.split()[0]:
            continue
        seen, todo = set(), list(nexts[i])
        while todo:
            j = todo.pop()
            if j in seen:
                continue
            seen.add(j)
            if ins[j].startswith("s_waitcnt") and re.search(r"vmcnt\(0\)", ins[j]):
                continue
            if ins[j].startswith("s_barrier"):
                bad.append((s, j))
                continue
            todo += nexts[j]
    return bad


def test_checker_flags_a_planted_path():
    load, wait, bar = "global_load_lds_dwordx4 v[0:1], off", "s_waitcnt vmcnt(0)", "s_barrier"
    assert unwaited([load, wait, bar, "s_endpgm"]) == []
    assert len(unwaited([load, bar, "s_endpgm"])) == 1
    assert len(unwaited([load, "s_waitcnt vmcnt(1)", bar, "s_endpgm"])) == 1
    assert len(unwaited([load, "s_cbranch_scc1 .L1", wait, ".L1:", bar, "s_endpgm"])) == 1     # the wait on one path
    assert unwaited([load, "s_cbranch_scc1 .L1", bar.replace("barrier", "nop 0"), ".L1:", wait, bar, "s_endpgm"]) == []
    assert len(unwaited([".L0:", bar, load, "s_cbranch_scc1 .L0", "s_endpgm"])) == 1           # round the loop
    assert unwaited([load, "s_waitcnt vmcnt(0) lgkmcnt(0)", bar, "s_endpgm"]) == []


SOURCES = [os.path.basename(s) for s in B.sources() if "load_lds" in open(s).read()]


@pytest.mark.skipif(shutil.which(B.HIPCC) is None and not os.path.exists(B.HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("src", SOURCES)
def test_loads_to_lds_have_arrived_before_a_barrier(src):
    r = subprocess.run([B.HIPCC, *B.FLAGS, "--cuda-device-only", "-S", os.path.join(B.CSRC, src), "-o", "-"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    n, problems = 0, []
    for name, lines in kernels(r.stdout).items():
        n += sum("load_lds" in l for l in lines)
        problems += [f"{name[:70]}: {load} -> barrier {at}" for load, at in unwaited(lines)]
    assert n > 0, "no loads to LDS found; the check would be vacuous"
    assert not problems, "\n".join(problems[:20])
