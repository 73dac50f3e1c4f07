"""The ends of fp32 in the rows of layers in 8-bit integers (mllm_i8_rms_norm), against the formulas in 64 bits."""
import pytest
import torch

from mojollama_amd import kernels as K
from test_gpu_i8_rows import U, check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return K.DeviceOps()


@pytest.mark.parametrize("n", [1, 3, 2048, 40000])
@pytest.mark.parametrize("size", [1e-44, 1e-40, 2.0 ** -127, 1e-38, 1e37, 8e37])
@pytest.mark.parametrize("where", ["none", "apart", "res"])
def test_norm_scale_at_both_ends(dev, n, size, where):
    """eps 0 and w 1: the row's factor lies beyond fp32's normal numbers, the scale does not.  The largest |y| has no
    rounding of its own; the scale is its product with the factor, rounded once."""
    g = torch.Generator().manual_seed(n)
    x, res = (torch.randn((3, n), generator=g).clamp(-4, 4) * s for s in (size, 0.0 if n == 1 else size * 0.01))
    x[x == 0] = size
    h = x if where == "none" else x + res
    rc = None if where == "none" else res.cuda()
    out = None if where != "apart" else torch.empty_like(rc)
    q, scale = dev.i8_rms_norm(x.cuda(), torch.ones(n, device="cuda"), 0.0, res=rc, res_out=out)
    v = h.double()
    top, _, _ = check("quantize", v, q, scale)
    want = top / torch.sqrt((v * v).mean(1)) / 127
    assert ((scale.cpu().double() - want).abs() <= U * 1.01 * want).all()
    if where == "apart":
        assert torch.equal(out.cpu(), h)
