"""A layer in 8-bit integers step by step: every product and every scale of the pass that test_gpu_i8_layer runs, and the
workspace that a product asks for."""
import pytest
import torch

from mojollama_amd import kernels as K
from test_gpu_i8_layer import EPS, FF, Layer, batch, half_codes, product
from test_gpu_i8_rows import U, far

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return K.DeviceOps()


def near_product(out, ref, top):
    """Half a step of the output's type (below its normal numbers theirs), and the roundings of fp32 before."""
    eps = torch.finfo(out.dtype)
    tol = eps.eps / 2 * 1.01 * ref.abs().clamp_min(eps.tiny) + 4 * U * 1.01 * (ref.abs() + top)
    return ((out.cpu().double() - ref).abs() <= tol).all()


def near_scale(scale, want, roundings):
    return ((scale.cpu().double() - want).abs() <= U * roundings * 1.01 * want).all()


@pytest.mark.parametrize("lens,new", [([1, 1, 1], [1, 1, 1]), ([70, 33, 128], [70, 33, 128]), ([50, 20, 90], [1, 2, 40])])
def test_every_product_and_scale(dev, lens, new):
    L = Layer(dev, 1, 256, 3)
    h, y, args = batch(lens, new, 2)
    out, st = L.run(h, y, *args)
    att, qa, sa = st["attention"]
    q2, s2, o, h2 = st["norm2"]
    gu, qs, ss = st["silu"]
    for (q, s, got), w, bias in (((qa, sa, o), "o", None), ((q2, s2, gu), "gu", None), (st["qkv"], "qkv", L.bias),
                                 (st["down"], "down", None)):
        ref = product(q, s, L.w[w], bias)
        # a sum of the bias and a product of the other sign may be small beside either: its roundings are of theirs
        top = 0.0 if bias is None else ref.abs() + 2 * bias.cpu().double().abs()
        assert near_product(got, ref, top), w
    q1, s1, h1 = st["norm"]
    for q, s, x, w in ((q1, s1, h1, L.n1), (q2, s2, h2, L.n2)):
        v = x.cpu().double()
        z = v * w.cpu().double()
        assert half_codes(z, q)
        # as for the rows of a norm anywhere: w h; the sum under the root; the mean, the sum with eps, root, reciprocal, two products
        assert near_scale(s, z.abs().amax(1) / torch.sqrt((v * v).mean(1) + EPS) / 127, 1 + far(v.shape[1]) / 2 + 1 + 1 + 2 + 2)
    a = att.cpu().double()
    assert half_codes(a, qa) and near_scale(sa, a.abs().amax(1) / 127, 1)
    g = gu.cpu().double()
    z = torch.nn.functional.silu(g[:, :FF]) * g[:, FF:]
    assert half_codes(z, qs) and near_scale(ss, z.abs().amax(1) / 127, 5 + 1)


@pytest.mark.parametrize("T", [64, 300, 700])
def test_workspace_that_is_too_small(dev, T):
    """300 x 4096 has a workspace at these sizes, and a call with less is refused before anything is written."""
    R, C = 300, 4096
    need = dev.so.mllm_i8_gemm_workspace_size(T, R, C)
    assert need > 0
    W = dev.i8_weights(torch.ones((R, C), dtype=torch.int8, device="cuda"), torch.ones(R, device="cuda"))
    q, s = torch.ones((T, C), dtype=torch.int8, device="cuda"), torch.ones(T, device="cuda")
    out = torch.full((T, R), 7.0, device="cuda")
    ws = dev.i8_gemm_workspace(W, T)
    assert ws.nbytes >= need
    with pytest.raises(RuntimeError, match="too small"):
        dev.i8_gemm(W, q, s, out=out, ws=ws[:need - 16])
    assert (out == 7.0).all()
    dev.i8_gemm(W, q, s, out=out, ws=ws)
    assert (out == float(C)).all()
