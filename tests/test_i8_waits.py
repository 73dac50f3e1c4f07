"""The waits of the tiled product of 8-bit integers, read from its machine code (CPU-only).

k_i8_tiles loads its tiles straight into LDS and, at the workgroup barrier in the middle of each step of K, waits only
until what the next step reads has landed: the number of younger loads that may still be under way is written in the
source and holds as long as the loop issues the loads it is meant to between one barrier and the next, and no other
access to vector memory.  Per wave that is, with px loads of x (two steps) and pw of weights (one step): pw between an
even step's barrier and the odd one's, px + pw from there to the next even one's; under way may be 2 pw at the odd one's
and 2 pw + px at the even one's.  Before each barrier every read of LDS has returned."""
import os
import re
import shutil
import subprocess

import pytest

from mojollama_amd import kernels
from test_gemm16_waits import OBJDUMP, code_objects

# (MF, NF, WM, WN, KG) of the tiles: 32 MF WM tokens x 32 NF WN rows, KG groups of waves
TILES = [(4, 4, 2, 2, 1), (2, 4, 2, 2, 1), (2, 2, 2, 2, 1), (1, 2, 2, 2, 1), (1, 1, 1, 4, 1), (1, 2, 2, 2, 2), (1, 1, 1, 4, 2)]


@pytest.fixture(scope="module")
def bodies(tmp_path_factory):
    if not (shutil.which("llvm-objdump") or os.path.exists(OBJDUMP)):
        pytest.skip("no llvm-objdump")
    if not os.path.exists(kernels.LIB_PATH):
        kernels.build()
    obj = [c for c in code_objects(kernels.LIB_PATH) if b"k_i8_tilesI" in c]
    assert len(obj) == 1
    f = tmp_path_factory.mktemp("co") / "i8_gemm.co"
    f.write_bytes(obj[0])
    text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(f)], capture_output=True, text=True, check=True).stdout
    return {tuple(map(int, re.findall(r"Li(\d+)E", name)[:5])): body.splitlines()
            for name, body in re.findall(r"^[0-9a-f]+ <(_Z\S*10k_i8_tilesI\S*?)>:\n(.*?)(?=^\S|\Z)", text, re.M | re.S)}


def events(lines):
    """(what, argument, address): 'D' a load into LDS, 'V' another access to vector memory, 'W' a wait (vmcnt or None,
    lgkmcnt or None), 'R' an access to LDS, 'M' a matrix instruction, 'B' a barrier, 'J' a jump back."""
    out, base = [], None
    for line in lines:
        m = re.match(r"\s+(\S+)(.*?)//\s*([0-9A-F]+)", line)
        if not m:
            continue
        op, arg, at = m.group(1), m.group(2), int(m.group(3), 16)
        base = at if base is None else base
        if "lds" in arg.split() or "load_lds" in op:
            out.append(("D", None, at - base))
        elif re.match(r"(buffer|global|flat|scratch)_(load|store|atomic)", op):
            out.append(("V", None, at - base))
        elif op.startswith("ds_"):
            out.append(("R", None, at - base))
        elif op.startswith("v_mfma"):
            out.append(("M", None, at - base))
        elif op == "s_waitcnt":
            n = {k: int(v) for k, v in re.findall(r"(vmcnt|lgkmcnt)\((\d+)\)", arg)}
            out.append(("W", (n.get("vmcnt"), n.get("lgkmcnt")), at - base))
        elif op == "s_barrier":
            out.append(("B", None, at - base))
        elif op.startswith(("s_branch", "s_cbranch")):
            t = re.search(r"\+0x([0-9a-f]+)>", line)
            out.append(("J", int(t.group(1), 16) if t else 0, at - base))
    return out


@pytest.mark.parametrize("tile", TILES)
def test_loop(bodies, tile):
    MF, NF, WM, WN, _ = tile
    px, pw = 32 * MF * WM // 8 // (WM * WN), 32 * NF * WN // 16 // (WM * WN)
    ev = events(bodies[tile])
    # the loop of K: the jump back over the most matrix instructions
    jumps = [(sum(1 for e in ev if e[0] == "M" and to <= e[2] <= at), to, at) for what, to, at in ev if what == "J" and to < at]
    n, to, at = max(jumps)
    body = [e for e in ev if to <= e[2] <= at]
    assert n == 4 * 2 * MF * NF and not [e for e in body if e[0] == "V"]
    cut = [i for i, e in enumerate(body) if e[0] == "B"]
    assert len(cut) == 4
    waits, loads = [], []
    for k, i in enumerate(cut):
        # the wait right before the barrier, with no access between
        j = i - 1
        while body[j][0] not in "WDRM":
            j -= 1
        assert body[j][0] == "W" and body[j][1][1] == 0, body[j]
        waits.append(body[j][1][0])
        behind = body[cut[k - 1] + 1:i] if k else body[cut[-1] + 1:] + body[:i]
        loads.append(sum(e[0] == "D" for e in behind))
        # no wait of the loop stops for younger loads than its barrier's
        assert all(e[1][0] is None or e[1][0] >= 2 * pw for e in behind if e[0] == "W")
    assert waits == [2 * pw + px, 2 * pw] * 2 and loads == [px + pw, pw] * 2
