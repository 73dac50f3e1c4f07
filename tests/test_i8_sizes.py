"""Sizes that the C entries' 32-bit integers do not hold, refused by the calls on tensors (host code; no GPU: the tensors
have no memory)."""
import os
from types import SimpleNamespace

import pytest
import torch

from mojollama_amd import kernels as K


@pytest.fixture(scope="module")
def dev():
    if not os.path.exists(K.LIB_PATH):
        K.build()
    d = K.DeviceOps()
    d._cur_raw = d._cur = lambda: 0
    return d


def rows(T, n, dtype=torch.float32):
    return torch.empty((T, n), dtype=dtype, device="meta")


@pytest.mark.parametrize("T,n", [((1 << 30) + 1, 1), ((1 << 31) - 1, 1), ((1 << 32) + 3, 1), (1, (1 << 30) + 1), (3, (1 << 32) + 5), (1 << 33, 64)])
def test_rows(dev, T, n):
    """(1 << 32) + 3 rows are 3 in 32 bits: three rows would be formed and the rest left as they were."""
    x, q, s = rows(T, n), rows(T, n, torch.int8), torch.empty(T, device="meta")
    w = SimpleNamespace(n_rows=64, n_cols=n, _device=0)
    for call in (lambda: K.I8Weights(dev, x), lambda: dev.i8_quantize(x), lambda: dev.i8_dequant(q, s),
                 lambda: dev.i8_rms_norm(x, s, 1e-6), lambda: dev.i8_silu_mul(x, x), lambda: dev.i8_gemm(w, q, s)):
        with pytest.raises(ValueError, match=r"2\^30"):
            call()


@pytest.mark.parametrize("T", [-1, -1 << 32, (1 << 30) + 1, (1 << 32) + 1, 1 << 40])
def test_workspace(dev, T):
    with pytest.raises(ValueError):
        dev.i8_gemm_workspace(SimpleNamespace(n_rows=64, n_cols=64), T)


def test_largest(dev):
    assert tuple(dev._sizes(rows(1 << 30, 1), "x")) == (1 << 30, 1) and tuple(dev._sizes(rows(1, 1 << 30), "x")) == (1, 1 << 30)
