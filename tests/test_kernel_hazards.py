"""Loads to LDS written in inline assembly keep the distances that the compiler
does not keep for them (CPU: the built library's kernels are listed, not run).

On CDNA a vector memory instruction may read a scalar register no sooner than
five wait states after a vector instruction wrote it, and a load to LDS may
follow a write of m0 after one. An instruction is one wait state, s_nop n is
n + 1.
"""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

WRITES = re.compile(r"v_(?:readfirstlane_b32|readlane_b32|cmp\w*)\s+s(?:(\d+)|\[(\d+):(\d+)\])")
LOAD = re.compile(r"global_load_lds_dword\w*\s+v(?:\d+|\[\d+:\d+\]),\s*(?:s\[(\d+):(\d+)\]|off)")


def close(instructions, i):
    """Instructions before number i with the wait states between, of up to five states."""
    states = 0
    for j in range(i - 1, -1, -1):
        if states >= 5 or instructions[j].startswith(("s_branch", "s_setpc", "s_endpgm")):
            return
        yield instructions[j], states
        nop = re.match(r"s_nop\s+(\d+)", instructions[j])
        states += int(nop[1]) + 1 if nop else 1


def faults(instructions):
    loads, bad = 0, []
    for i, text in enumerate(instructions):
        load = LOAD.match(text)
        if not load:
            continue
        loads += 1
        base = range(int(load[1]), int(load[2]) + 1) if load[1] else range(0)
        for before, states in close(instructions, i):
            wrote = WRITES.match(before)
            if wrote:
                first, last = (int(wrote[1]),) * 2 if wrote[1] else (int(wrote[2]), int(wrote[3]))
                if any(first <= s <= last for s in base):
                    bad.append((before, states, text))
            if states < 1 and re.match(r"s_\w+\s+m0,", before):
                bad.append((before, states, text))
    return loads, bad


def test_the_rule_finds_what_is_too_close():
    near = ["v_readfirstlane_b32 s67, v1", "v_readfirstlane_b32 s45, v2", "s_mov_b32 m0, s45", "s_nop 0",
            "global_load_lds_dwordx4 v188, s[66:67]"]
    assert faults(near) == (1, [(near[0], 3, near[4])])
    assert faults(near[:3] + ["s_nop 2"] + near[4:]) == (1, [])
    assert faults(near[:3] + near[4:])[1][0][0] == near[2]
    assert faults(["v_cmp_eq_u32_e64 s[66:67], 0, v1", "s_nop 3", near[4]])[1]
    assert faults(near[:3] + ["s_nop 0", "global_load_lds_dwordx4 v[2:3], off"]) == (1, [])


def test_loads_to_lds_keep_their_distances(tmp_path):
    from jasper_amd import build_lib
    objdump = build_lib.ROCM / "llvm" / "bin" / "llvm-objdump"
    if not objdump.exists():
        pytest.skip("no llvm-objdump")
    if not build_lib.LIB.exists():
        build_lib.build(verbose=False)
    shutil.copy(build_lib.LIB, tmp_path / "lib.so")
    subprocess.run([objdump, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    loads = 0
    for part in sorted(Path(tmp_path).glob("lib.so.*amdgcn*")):
        if b"shared_kernel" not in part.read_bytes():
            continue
        listing = subprocess.run([objdump, "-d", "--no-show-raw-insn", str(part)], check=True, capture_output=True, text=True)
        text = [line.split("//")[0].strip() for line in listing.stdout.splitlines() if line.startswith("\t")]
        n, bad = faults(text)
        loads += n
        assert not bad, bad[:5]
    assert loads > 0
