"""What the calls of layers in 8-bit integers refuse, before any launch, and their sizes (host code; no GPU)."""
import pytest

from mojollama_amd import kernels as K

P = 4096   # an address that is checked and never read
BIG = 1 << 40


@pytest.fixture(scope="module")
def so():
    import os
    if not os.path.exists(K.LIB_PATH):
        K.build()
    return K.load_kernels()


def quantize(so, **c):
    a = dict(type=K.T_BF16, x=P, x_ld=100, T=3, n=100, q=P, q_ld=112, scale=P) | c
    return so.mllm_i8_quantize(*a.values(), None)


def dequant(so, **c):
    a = dict(q=P, q_ld=112, scale=P, T=3, n=100, type=K.T_BF16, x=P, x_ld=100) | c
    return so.mllm_i8_dequant(*a.values(), None)


def norm(so, **c):
    a = dict(type=K.T_BF16, x=P, x_ld=100, res_type=K.T_F32, res=2 * P, res_ld=100, res_out=3 * P, res_out_ld=100,
             w_type=K.T_F32, w=P, eps=1e-6, T=3, n=100, q=P, q_ld=112, scale=P) | c
    return so.mllm_i8_rms_norm(*a.values(), None)


def silu(so, **c):
    a = dict(type=K.T_BF16, x=P, x_ld=200, up=P + 200, up_ld=200, T=3, n=100, q=P, q_ld=112, scale=P) | c
    return so.mllm_i8_silu_mul(*a.values(), None)


def gemm(so, **c):
    a = dict(packed=P, ws=P, x=P, x_ld=112, xs=P, T=3, rows=40, cols=100, bias=None, type=K.T_BF16, out=P, out_ld=40, work=P,
             n=BIG) | c
    return so.mllm_i8_gemm(*a.values(), None)


def pack(so, **c):
    a = dict(type=K.T_F32, w=P, w_ld=100, rows=40, cols=100, packed=P, scale=P) | c
    return so.mllm_i8_pack(*a.values(), None)


ROWS = [dict(T=(1 << 30) + 1), dict(type=K.T_E4M3), dict(type=K.T_I8), dict(type=-1), dict(T=-1), dict(n=0), dict(n=-5), dict(x_ld=99), dict(q_ld=99),
        dict(x=None), dict(q=None), dict(scale=None), dict(n=(1 << 30) + 1, x_ld=BIG, q_ld=BIG)]


@pytest.mark.parametrize("c", ROWS)
def test_rows(so, c):
    for call in (quantize, dequant, norm, silu):
        assert call(so, **(c | ({"up_ld": BIG} if call is silu and "x_ld" in c and c["x_ld"] == BIG else {}))) == -1
        assert so.mllm_last_error().startswith(b"mllm_i8_")


@pytest.mark.parametrize("c", [dict(w=None), dict(w_type=K.T_E4M3), dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")),
                               dict(res_type=K.T_E4M3), dict(res_ld=99), dict(res_out_ld=99), dict(res_out=None),
                               dict(res_out=2 * P, res_out_ld=104), dict(res_out=P), dict(res_out=P, res_type=K.T_BF16, res_out_ld=104)])
def test_norm(so, c):
    assert norm(so, **c) == -1 and so.mllm_last_error().startswith(b"mllm_i8_rms_norm")


@pytest.mark.parametrize("c", [dict(up=None), dict(up_ld=99)])
def test_silu(so, c):
    assert silu(so, **c) == -1 and so.mllm_last_error().startswith(b"mllm_i8_silu_mul")


@pytest.mark.parametrize("c", [dict(T=-1), dict(T=(1 << 30) + 1), dict(rows=0), dict(rows=-3), dict(cols=0), dict(cols=131072, x_ld=131072),
                               dict(type=K.T_I8), dict(type=K.T_E4M3), dict(x_ld=96), dict(x_ld=100), dict(x_ld=104), dict(out_ld=39),
                               dict(x=P + 1), dict(x=P + 8), dict(packed=P + 4), dict(work=P + 8), dict(packed=None), dict(ws=None),
                               dict(x=None), dict(xs=None), dict(out=None)])
def test_gemm(so, c):
    assert gemm(so, **c) == -1 and so.mllm_last_error().startswith(b"mllm_i8_gemm")


@pytest.mark.parametrize("c", [dict(type=K.T_E4M3), dict(w=None), dict(w_ld=99), dict(rows=0), dict(cols=0),
                               dict(cols=131072, w_ld=131072), dict(packed=None), dict(packed=P + 8), dict(scale=None)])
def test_pack(so, c):
    assert pack(so, **c) == -1 and so.mllm_last_error().startswith(b"mllm_i8_pack")


def test_nothing(so):
    """No rows: nothing is launched, addresses are not asked for."""
    none = dict(T=0, x=None, q=None, scale=None)
    assert quantize(so, **none) == 0 and dequant(so, **none) == 0
    assert norm(so, **none, w=None, res=None) == 0 and silu(so, **none, up=None) == 0
    assert gemm(so, T=0, packed=None, ws=None, x=None, xs=None, out=None, work=None, n=0) == 0


def test_sizes(so):
    assert so.mllm_i8_packed_size(1, 1) == 32 * 512
    assert so.mllm_i8_packed_size(33, 513) == 64 * 1024
    assert so.mllm_i8_packed_size(40, 131071) == 64 * 131072
    for rows, cols in ((0, 5), (5, 0), (-1, 5), (5, 131072)):
        assert so.mllm_i8_packed_size(rows, cols) == -1 and so.mllm_i8_gemm_workspace_size(3, rows, cols) == -1
    assert so.mllm_i8_gemm_workspace_size(-1, 5, 5) == -1


@pytest.mark.parametrize("rows,cols", [(16, 33), (256, 16384), (2883, 2881), (32000, 2048), (8192, 8192), (100000, 64), (64, 131071)])
def test_workspace_never_decreases(so, rows, cols):
    """A workspace for T tokens serves every smaller T."""
    f = lambda T: so.mllm_i8_gemm_workspace_size(T, rows, cols)  # noqa: E731
    Ts = list(range(0, 1200)) + [1 << i for i in range(11, 20)] + [(1 << i) + 1 for i in range(11, 20)]
    sizes = [f(T) for T in sorted(Ts)]
    assert sizes == sorted(sizes) and sizes[0] >= 0


@pytest.mark.parametrize("rows,cols", [(16, 33), (256, 16384), (2883, 2881), (64, 131071)])
def test_workspace_too_small(so, rows, cols):
    for T in (1, 5, 17, 64, 200, 1000):
        n = so.mllm_i8_gemm_workspace_size(T, rows, cols)
        if n > 0:
            c = dict(T=T, rows=rows, cols=cols, x_ld=(cols + 15) // 16 * 16, out_ld=rows)
            assert gemm(so, **c, n=n - 1) == -1 and gemm(so, **c, work=None) == -1
