"""The ends of fp32 in the rows of layers in 8-bit integers (mllm_i8_rms_norm, _silu_mul), against the formulas in 64
bits."""
import math

import pytest
import torch

from mojollama_amd import kernels as K
from test_gpu_i8_rows import TYPES, U, check, far, scales

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


# h and w of which w h leaves fp32 on either side, wholly or for the smaller elements, though y does not
PRODUCTS = [(3e30, 1e9, 1e-6), (1e38, 50.0, 0.0), (1e-30, 1e-12, 0.0), (1e-38, 1e-3, 0.0), (1e-20, 1e-30, 1e-45), (1.0, 1e-40, 1e-6),
            (1e-35, 1e-2, 0.0), (2e37, 4e36, 0.0), (1e-40, 1e36, 0.0), (1e-3, 1e-37, 1e-6)]


@pytest.mark.parametrize("n", [1, 7, 700, 4096, 5000, 40000])
@pytest.mark.parametrize("h,w,eps", PRODUCTS)
@pytest.mark.parametrize("where", ["none", "apart", "res", "x"])
def test_norm_products_beyond_fp32(dev, n, h, w, eps, where):
    """Beside rows that do not come near the ends: those have the bits that they have alone."""
    eps = torch.tensor(eps).double().item()          # the entry takes eps in fp32: 1e-45 is 2^-149 = 1.4e-45 there
    g = torch.Generator().manual_seed(n)
    x = torch.randn((6, n), generator=g).clamp(-3, 3)
    x[:, 0] = 2.0
    x[::2] *= h
    wt = (1.0 + 0.2 * torch.rand(n, generator=g)) * w
    r = None if where == "none" else (0.1 * x).cuda()
    xc = x.cuda()
    v = x if r is None else x + r.cpu()
    out = {"none": None, "apart": torch.empty_like(xc), "res": r, "x": xc}[where]
    q, scale = dev.i8_rms_norm(xc, wt.cuda(), eps, res=r, res_out=out)
    if out is not None:
        assert torch.equal(out.cpu(), v)
    v = v.double()
    y = v * wt.double()
    assert (v.abs().amax(1) / torch.sqrt((v * v).mean(1) + eps) * 1.2 * w < 3e38).all()
    top, _, _ = check("norm", y, q, scale, names=(n, h, w))
    scales(scale, top / torch.sqrt((v * v).mean(1) + eps) / 127, 1 + far(n) / 2 + 1 + 1 + 2 + 2, names=(n, h, w))
    a, s = dev.i8_rms_norm(v[1::2].float().cuda(), wt.cuda(), eps)
    assert torch.equal(a, q[1::2]) and torch.equal(s, scale[1::2])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n", [5, 2048, 9001])
def test_norm_products_of_16_bits(dev, kind, n):
    g = torch.Generator().manual_seed(n)
    x = (torch.randn((3, n), generator=g).clamp(-3, 3) * 1e4).to(TYPES[kind])
    x[1] = (torch.randn(n, generator=g) * 6e-8).to(TYPES[kind])
    x[1, 0] = 1e-6
    for w, eps in ((1e36, torch.tensor(1e-5).double().item()), (1e-34, 0.0)):
        wt = torch.full((n,), w)
        q, scale = dev.i8_rms_norm(x.cuda(), wt.cuda(), eps)
        v = x.double()
        y = v * wt.double()
        top, _, _ = check("norm", y, q, scale)
        scales(scale, top / torch.sqrt((v * v).mean(1) + eps) / 127, 1 + far(n) / 2 + 1 + 1 + 2 + 2)


@pytest.mark.parametrize("n", [1024, 40000])
def test_norm_values_beyond_fp32(dev, n):
    """y itself beyond fp32 is an infinity; infinities, NaNs and zeros where products leave fp32."""
    x = torch.zeros((8, n))
    x[0, 5] = 1.0                  # y = sqrt(n) w: beyond fp32
    x[1] = 1.0                     # y = w: inside
    x[2], x[2, n - 1] = 1e30, math.inf
    x[3], x[3, 0] = 1e30, math.nan
    x[4] = 1e-44
    x[6] = -1e-30
    x[7, n // 2] = -3e38
    w = torch.full((n,), 3e38)
    q, scale = dev.i8_rms_norm(x.cuda(), w.cuda(), 0.0)
    q, scale = q.cpu(), scale.cpu()
    for i in (0, 2, 3, 7):
        assert scale[i].isnan() and not q[i].any(), i
    assert scale[5] == 0 and not q[5].any()
    for i, code in ((1, 127), (4, 127), (6, -127)):
        assert (q[i] == code).all() and abs(scale[i].item() / (w[0].double().item() / 127) - 1) <= 4 * U, i
    q, scale = dev.i8_rms_norm(x.cuda(), torch.zeros(n, device="cuda"), 0.0)
    finite = torch.tensor([0, 1, 4, 5, 6, 7], device="cuda")
    assert not q.any() and not scale[finite].any() and scale[2:4].isnan().all()


@pytest.mark.parametrize("n", [1, 9, 700, 40000])
@pytest.mark.parametrize("least,most,up", [(-80.0, -69.5, 1.0), (-103.0, -88.0, 1e30), (-120.0, -104.0, 1e38), (-150.0, -60.0, 1e35)])
def test_silu_of_far_gates(dev, n, least, most, up):
    """Gates whose silu is below fp32's normal numbers, or below all of them, and an up that takes the product back into
    range.  Roundings of y there: e^(g / 2), within one step, twice (four halves), and three products."""
    g = torch.Generator().manual_seed(n)
    gate = least + (most - least) * torch.rand((4, n), generator=g)
    gate[:, 0] = most
    u = (0.5 + torch.rand((4, n), generator=g)) * up
    u[:, 0] = 1.5 * up
    q, scale = dev.i8_silu_mul(gate.cuda(), u.cuda())
    a = gate.double()
    e = torch.exp(a)
    y = a * e / (1 + e) * u.double()
    top = y.abs().amax(1)
    assert (top > 2.0 ** -100).all()
    off = (q.cpu().double() - 127 * y / top[:, None]).abs().max().item()
    assert off <= 0.5 + 127 * U * (2 * 7 + 3) * 1.01, off
    assert ((scale.cpu().double() - top / 127).abs() <= U * (7 + 1) * 1.01 * top / 127).all()
