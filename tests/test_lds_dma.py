"""Wait states of the loads into LDS, in the device code that is built.

A load into LDS takes its LDS address from M0 and, as a buffer load, its descriptor from scalar registers.
gfx9's instruction set asks for one wait state between a scalar write of M0 and the load, and for five between a
vector instruction's write of a scalar register and a vector-memory instruction that reads it; hardware does
not wait by itself, and the compiler does not look into the helpers' inline assembly.  Compiled on the CPU only.
"""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from tinyvllm_amd import build

HERE = Path(__file__).resolve().parent


def registers(token):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", token)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.fullmatch(r"s(\d+)", token)
    return {int(m[1])} if m else set()


def wait_states(line):
    return int(line.split()[1], 0) + 1 if line.startswith("s_nop") else 1


def short_waits(lines):
    """(loads into LDS, [(wait states, the write, the load)] of those that come too early).  Straight-line code."""
    loads, early = 0, []
    for i, line in enumerate(lines):
        op = line.split()[0]
        if not (op.startswith("buffer_load") and line.endswith(" lds") or op.startswith("global_load_lds")):
            continue
        loads += 1
        reads = set().union(*(registers(t) for t in re.split(r"[,\s]+", line)[1:]))
        waited, m0 = 0, True
        for before in reversed(lines[:i]):
            target = re.split(r"[,\s]+", before)[1] if " " in before else ""
            if m0 and target == "m0":
                m0 = False
                if waited < 1:
                    early.append((waited, before, line))
            if before.startswith("v_") and registers(target) & reads and waited < 5:
                early.append((waited, before, line))
            waited += wait_states(before)
            if waited >= 5:
                break
    return loads, early


def test_the_rule_itself():
    head = ["v_readfirstlane_b32 s7, v1", "s_mov_b32 m0, s2"]
    load = "buffer_load_dwordx4 v1, s[4:7], 0 offen nt lds"
    assert [w for w, *_ in short_waits([*head, load])[1]] == [0, 1]
    assert [w for w, *_ in short_waits([*head, "s_nop 0", load])[1]] == [2]
    assert short_waits([*head, "s_nop 3", load]) == (1, [])
    assert short_waits(["s_mov_b32 m0, s2", "global_load_lds_dwordx4 v[0:1], off"])[1][0][0] == 0
    assert short_waits(["s_mov_b32 m0, s2", "s_nop 0", "global_load_lds_dwordx4 v[0:1], off"]) == (1, [])


def test_loads_into_lds_wait_for_m0_and_their_descriptor(tmp_path):
    if not Path(build.HIPCC).exists() and not shutil.which(build.HIPCC):
        pytest.skip("hipcc not available")
    out = tmp_path / "lds_dma.s"
    res = subprocess.run([build.HIPCC, *build.CFLAGS, "-S", "--cuda-device-only", str(HERE / "lds_dma_check.hip"), "-o",
                          str(out)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
    lines = [t for t in (x.split(";")[0].strip() for x in out.read_text().splitlines()) if t and t[0] not in "._#"]
    loads, early = short_waits(lines)
    assert loads == 3
    assert not early, early
