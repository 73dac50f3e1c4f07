"""The ramp of MLLM_ROPE_YARN pair by pair (host code; no GPU)."""
import ctypes
import math
import os

import pytest

from mojollama_amd import kernels as K


@pytest.fixture(scope="module")
def so():
    if not os.path.exists(K.LIB_PATH):
        K.build()
    return K.load_kernels()


@pytest.mark.parametrize("r,base", [(64, 150000.0), (128, 500000.0), (96, 10000.0), (20, 10000.0), (2, 10000.0)])
@pytest.mark.parametrize("factor,ctx,fast,slow", [(32.0, 4096.0, 0.0, 0.0), (4.0, 64.0, 32.0, 1.0), (8.0, 32768.0, 20.0, 2.5),
                                                  (1.0, 4096.0, 0.0, 0.0), (0.5, 300.0, 8.0, 7.9)])
def test_every_pair(so, r, base, factor, ctx, fast, slow):
    """From the whole pair below that of beta_fast turns to the one above that of beta_slow, linear in the pair."""
    f, m = (ctypes.c_double * (r // 2))(), ctypes.c_float()
    assert so.mllm_rotary_freqs(K.ROPE_YARN, r, base, factor, ctx, fast, slow, f, ctypes.byref(m)) == 0
    first, last = (r * math.log(ctx / (2 * math.pi * b)) / (2 * math.log(base)) for b in (fast or 32.0, slow or 1.0))
    first, last = max(math.floor(first), 0), min(math.ceil(last), r - 1)
    between = 0
    for j in range(r // 2):
        w = base ** (-2 * j / r)
        s = min(max((j - first) / (last - first if last > first else 0.001), 0.0), 1.0)
        between += 0 < s < 1
        assert math.isclose(f[j], w / factor * s + w * (1 - s), rel_tol=1e-12), j
    assert between > 0 or r <= 20 or last - first < 2
    assert math.isclose(m.value, 0.1 * math.log(factor) + 1 if factor > 1 else 1.0, rel_tol=1e-6)
