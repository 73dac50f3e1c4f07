"""The waits of the product of few 8-bit integer rows (k_i8_stream), read from its machine code (CPU-only).

A wave loads the x of its blocks straight into LDS, blocks in turn, and no barrier stands between a load and the read of
it: before a block's reads the source waits until no more loads are outstanding than a block has (4 TF of x, 4 of weights)
where a later block is under way, and for all of them where none is.  That holds as long as each block issues just that
many loads, with nothing else between.  So this follows every path of the built kernels up to the workgroup's barrier: no
read of a block's x may come with one of its loads outstanding, and no load may go to LDS that is still being read."""
import os
import re
import shutil
import subprocess

import pytest

from mojollama_amd import kernels
from test_gemm16_waits import OBJDUMP, code_objects


@pytest.fixture(scope="module")
def bodies(tmp_path_factory):
    if not (shutil.which("llvm-objdump") or os.path.exists(OBJDUMP)):
        pytest.skip("no llvm-objdump")
    if not os.path.exists(kernels.LIB_PATH):
        kernels.build()
    obj = [c for c in code_objects(kernels.LIB_PATH) if b"k_i8_streamI" in c]
    assert len(obj) == 1
    f = tmp_path_factory.mktemp("co") / "i8_gemm.co"
    f.write_bytes(obj[0])
    text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(f)], capture_output=True, text=True, check=True).stdout
    out = {}
    for part in re.split(r"^[0-9a-f]+ <", text, flags=re.M):
        name = part.split(">:", 1)[0]
        if "k_i8_streamI" in name:
            out[tuple(map(int, re.findall(r"Li(\d+)E", name)))] = part.splitlines()
    return out


def events(lines):
    """[(what, argument)], {address: index}: 'D' a load into LDS, 'V' another access to vector memory, 'W' a wait (vmcnt or
    None, lgkmcnt or None), 'R' an access to LDS, 'B' a barrier, 'J' / 'C' a branch always / at times, 'E' the end."""
    ev, at, base = [], {}, None
    for line in lines:
        m = re.match(r"\s+(\S+)(.*?)//\s*([0-9A-F]+)", line)
        if not m:
            continue
        op, arg, adr = m.group(1), m.group(2), int(m.group(3), 16)
        base = adr if base is None else base
        at[adr - base] = len(ev)
        if "lds" in arg.split() or "load_lds" in op:
            ev.append(("D", None))
        elif re.match(r"(buffer|global|flat|scratch)_(load|store|atomic)", op):
            ev.append(("V", None))
        elif op.startswith("ds_"):
            ev.append(("R", None))
        elif op == "s_waitcnt":
            n = {k: int(v) for k, v in re.findall(r"(vmcnt|lgkmcnt)\((\d+)\)", arg)}
            ev.append(("W", (n.get("vmcnt"), n.get("lgkmcnt"))))
        elif op in ("s_barrier", "s_endpgm"):
            ev.append(("B" if op == "s_barrier" else "E", None))
        elif op == "s_branch" or op.startswith("s_cbranch"):
            t = re.search(r"\+0x([0-9a-f]+)>", line)
            ev.append(("J" if op == "s_branch" else "C", int(t.group(1), 16) if t else 0))
    return ev, at


def follow(ev, at, TF, weakest):
    """What is wrong on some path.  A state: the place; the outstanding loads, each by its block (0: the oldest that is not
    read yet); blocks issued and not read; loads of the youngest so far; reads of the oldest so far; whether reads may be
    outstanding; the source's waits since the last read.  The source takes one of its two waits before a block, for all
    loads if and only if no later block was loaded, and comes to
    every block that was loaded and no other: other paths are none."""
    x, loads = 4 * TF, 4 * TF + 4
    bad, seen, blocks = set(), set(), 0
    todo = [(0, (), 0, loads, 0, False, 0)]
    while todo:
        st = todo.pop()
        while st not in seen:
            seen.add(st)
            i, q, live, got, reads, r, waits = st
            what, arg = ev[i]
            i += 1
            if what in "DV":
                if got == loads:
                    if what == "V":
                        bad.add("an access between the blocks")
                    live, got = live + 1, 0
                if (what == "D") != (got < x):
                    bad.add("a block of other loads")
                if what == "D" and r:
                    bad.add("a load over what is read")
                q, got = q + (live - 1,), got + 1
            elif what == "R":
                if not reads and waits != 1:
                    break
                if got != loads or not live or 0 in q:
                    bad.add("a read ahead of its load")
                r, reads = True, reads + 1
                if reads == x:
                    q, live, reads, waits, blocks = tuple(b - 1 for b in q), live - 1, 0, 0, blocks + 1
            elif what == "W":
                vm, lgkm = arg
                if lgkm == 0 and not reads and (vm == 0 or vm == weakest):
                    if not live or (vm == 0) == (live > 1):
                        break
                    waits += 1
                if vm is not None:
                    q = q[max(0, len(q) - vm):]
                r = r and lgkm != 0
            elif what in "BE":
                if not live and q:
                    bad.add("a load behind the barrier")
                break
            elif what == "J":
                i = at[arg]
            else:
                todo.append((at[arg], q, live, got, reads, r, waits))
            st = (i, q, live, got, reads, r, waits)
    return bad, blocks


@pytest.mark.parametrize("TF", [1, 2])
def test_every_block_waits_for_its_loads(bodies, TF):
    assert set(bodies) == {(1, 8), (2, 8)}
    bad, blocks = follow(*events(bodies[TF, 8]), TF, 4 * TF + 4)
    assert blocks >= 4 and not bad, bad


@pytest.mark.parametrize("more", [1, 8])
def test_a_wait_too_weak_is_found(bodies, more):
    """The same code with one or eight more loads let through; the compiler's own waits, for weights, left out."""
    ev, at = events(bodies[2, 8])
    weak = [(w, a) if w != "W" or a[0] in (None, 0) and a[1] == 0 else (w, (12 + more if a == (12, 0) else None, a[1])) for w, a in ev]
    assert "a read ahead of its load" in follow(weak, at, 2, 12 + more)[0]
