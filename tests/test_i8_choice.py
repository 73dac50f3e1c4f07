"""The choice among the kernels of mllm_i8_gemm (CPU-only): the sizes of the GPU tests reach every kernel and every tile, with
K whole and split, so that a change of the choice cannot leave one untested.  The choice is sizes and constants alone: its
lines of i8_gemm.hip are compiled for the host here."""
import ctypes
import os
import subprocess

import pytest

import test_gpu_i8_gemm as G
from mojollama_amd import kernels

HEAD = r"""
#include <algorithm>
#include <cmath>
typedef void *hipStream_t;
struct gemm_args;
template <int MF, int NF, int WM, int WN> struct tile_of { static constexpr int TT = 32 * MF * WM, TR = 32 * NF * WN; };
template <int, int, int, int, int, int> void go_tiles(const gemm_args &, int, hipStream_t) {}
"""
TAIL = r"""
extern "C" int choice(int T, int R, int cols, int *kind)
{
    const plan p = plan_of(T, R, (cols + 511) / 512 * 8, cols);
    kind[0] = p.kind ? p.kind->TT : 0, kind[1] = p.kind ? p.kind->TR : 0, kind[2] = p.kind ? p.kind->groups : 0;
    kind[3] = p.kind ? p.splits : p.few;
    return p.kind ? 1 : 0;
}
extern "C" int tiles(int i, int *kind)
{
    if (i >= (int)(sizeof kinds / sizeof *kinds)) return 0;
    kind[0] = kinds[i].TT, kind[1] = kinds[i].TR, kind[2] = kinds[i].groups;
    return 1;
}
"""


@pytest.fixture(scope="module")
def choice(tmp_path_factory):
    src = open(os.path.join(os.path.dirname(kernels.LIB_PATH), "csrc", "i8_gemm.hip")).read()
    part = src[src.index("struct tile_kind {"):src.index("// Bytes of the sums of any plan")]
    a = part.index("template <int MF, int NF, int WM, int WN, int KG, int OCC> void go_tiles")
    b = part.index("template <int MF, int NF, int WM, int WN, int KG, int OCC> constexpr tile_kind kind_of")
    d = tmp_path_factory.mktemp("choice")
    (d / "choice.cpp").write_text(HEAD + part[:a] + part[b:] + TAIL)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-o", str(d / "choice.so"), str(d / "choice.cpp")], check=True)
    return ctypes.CDLL(str(d / "choice.so"))


def cases():
    """(T, rows, columns) of the GPU tests that compare every result."""
    out = [(T, R, C) for T in G.TOKENS for R, C in ((200, 320), (1000, 2048), (33, 4100))]
    for test in (G.test_ragged_tiles, G.test_large, G.test_outputs):
        out += [s for m in test.pytestmark if m.name == "parametrize" and m.args[0] == "T,R,C" for s in m.args[1]]
    args = {m.args[0]: m.args[1] for m in G.test_shapes.pytestmark if m.name == "parametrize"}
    out += [(T, R, C) for T in args["T"] for R, C in args["R,C"]]
    return out


def test_every_kernel_is_reached(choice):
    kind, reached = (ctypes.c_int * 4)(), {}
    for T, R, C in cases():
        if choice.choice(T, R, C, kind):
            reached.setdefault((kind[0], kind[1], kind[2], kind[3] > 1), []).append((T, R, C))
        else:
            reached.setdefault(("few", kind[3]), []).append((T, R, C))
    tiles = []
    while choice.tiles(len(tiles), kind):
        tiles.append(tuple(kind[:3]))
    assert len(tiles) == 7 and len(cases()) > 300
    want = {t + (split,) for t in tiles for split in (False, True)} | {("few", n) for n in (1, 2, 3)}
    assert not want - set(reached), sorted(map(str, want - set(reached)))
    # with ragged ends in each direction
    for t in tiles:
        for split in (False, True):
            assert any(T % t[0] and R % t[1] for T, R, C in reached[t + (split,)]), (t, split)
