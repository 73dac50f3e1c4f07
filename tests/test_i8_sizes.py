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


def test_workspaces_lie_densely(dev):
    """A workspace's address and bytes go to the entries: what is not dense would be written beyond itself.  (The
    entries stand in for themselves here: nothing is launched.)"""
    class Entries:
        def __getattr__(self, name):
            return lambda *a: 0

    class Here(torch.Tensor):
        """On GPU 0, as far as the checks ask."""
        get_device = lambda self: 0  # noqa: E731

    ops = K.DeviceOps(Entries())
    ops._cur_raw = ops._cur = lambda: 0
    ops._stream_of = ops._raw_stream = lambda cur: None
    t = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype).as_subclass(Here)  # noqa: E731
    dense = t(64, 16, dtype=torch.uint8)
    apart = [dense[:, :8], dense[::2], torch.zeros(1, dtype=torch.uint8).as_subclass(Here).expand(1 << 40)]
    w = SimpleNamespace(n_rows=8, n_cols=16, _device=0, _packed=0, _scale=0)
    kv = SimpleNamespace(_device=0, head_dim=16)
    m = SimpleNamespace(_device=0)
    ints = t(3, dtype=torch.int32)
    calls = [lambda ws: ops.i8_gemm(w, t(2, 16, dtype=torch.int8), t(2), out=t(2, 8), ws=ws),
             lambda ws: ops._attn(kv, t(2, 32), 2, 2, 2, 16, 0, None, t(2, 32), None, ws, 0),
             lambda ws: ops._pages_args(m, 3, ints[:1], ws, 0)]
    for call in calls:
        call(dense)
        for ws in apart:
            with pytest.raises(ValueError, match="workspace"):
                call(ws)


def test_streams_without_the_raw_call(monkeypatch):
    """A torch whose runtime does not hand out raw streams: the current stream's handle, from every call."""
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=1000 + device))
    ops = K.DeviceOps(SimpleNamespace())
    assert ops._stream_of(3) == 1003 and ops._raw_stream(2) == 1002
