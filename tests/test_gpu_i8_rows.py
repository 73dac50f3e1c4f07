"""Rows into 8-bit integers with a scale (mllm_i8_quantize, _rms_norm, _silu_mul) and back (mllm_i8_dequant), against
the formulas in 64 bits.

A code may differ from the 64-bit quotient y / (max|y| / 127) by the half step of its rounding and by what fp32 does
to the quotient before: 2^-24 of 127 for each rounding of y, of the largest (which the reciprocal takes over), of the
reciprocal, of 127 times it and of the product with y."""
import math

import pytest
import torch

from mojollama_amd import kernels as K

pytestmark = pytest.mark.gpu
U = 2.0 ** -24                       # half a step of fp32, relative
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# roundings of y: none; w h; e^-g (within one step: two halves), 1 + e, the quotient, the product
ROUNDINGS = {"quantize": 0, "norm": 1, "silu": 5}


@pytest.fixture(scope="module")
def dev():
    return K.DeviceOps()


def rand(g, T, n, kind, lead=0, tail=0):
    """[T, n] inside a wider buffer."""
    x = torch.randn((T, lead + n + tail), generator=g) * torch.exp(torch.randn((T, 1), generator=g))
    return x.to(TYPES[kind]).cuda()[:, lead:lead + n]


def room(T, n, ld, dtype, fill):
    buf = torch.full((T, ld), fill, dtype=dtype, device="cuda")
    return buf, buf[:, :n]


def stepwise(x):
    """The formula in fp32, operation by operation, on the CPU: the same bits."""
    x = x.cpu().float()
    top = x.abs().amax(1, keepdim=True)
    inv = torch.where(top > 0, torch.ones_like(top) / top * 127.0, 0.0)
    return torch.round(x * inv).to(torch.int8), (top / torch.full_like(top, 127.0))[:, 0]


def far(n):
    """Roundings in a sum of n squares: a lane's own chain (at least 64 lanes a row), six exchanges, 16 waves."""
    return 8 * math.ceil(n / 512) + 6 + 16 + 1


def check(kind, y, q, scale, extra=0.0, names=""):
    """y: the values in 64 bits; extra: roundings in a factor that the scale alone has."""
    y, q, scale = y.cpu(), q.cpu().double(), scale.cpu().double()
    top = y.abs().amax(1)
    live = top > 0
    k = ROUNDINGS[kind]
    assert torch.equal(q[~live], torch.zeros_like(q[~live])) and not scale[~live].any(), names
    if not live.any():
        return
    ratio = y[live] / (top[live, None] / 127)
    off = (q[live] - ratio).abs().max().item()
    assert off <= 0.5 + 127 * U * (2 * k + 3) * 1.01, (names, off)
    assert q.abs().max() <= 127
    return top, live, k


def scales(scale, want, roundings, names=""):
    scale, want = scale.cpu().double(), want.cpu()
    err = ((scale - want).abs() - 2.0 ** -149) / want.abs().clamp_min(1e-300)
    assert err.max().item() <= U * roundings * 1.01, (names, err.max().item() / U)


SIZES = [(1, 1), (1, 7), (3, 8), (1, 64), (5, 100), (2, 511), (3, 512), (9, 513), (1, 2048), (7, 2049), (1, 2880), (4, 4095),
         (2, 4097), (3, 8191), (2, 8200), (1, 16385), (2, 32768), (1, 32777), (2, 70001), (130, 33), (1021, 257), (1025, 1000), (256, 4097), (256, 9001),
         (257, 12300), (260, 16383), (256, 20000)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,n", SIZES)
def test_quantize(dev, T, n, kind):
    g = torch.Generator().manual_seed(T * 100003 + n)
    for lead, tail, pad in ((0, 0, 0), (3, 2, 5), (0, 1, 16)):
        x = rand(g, T, n, kind, lead, tail)
        buf, q = room(T, n, n + pad, torch.int8, 77)
        scale = torch.full((T,), -1.0, device="cuda")
        dev.i8_quantize(x, q=q, scale=scale)
        assert (buf[:, n:] == 77).all()
        y = x.cpu().double()
        check("quantize", y, q, scale, names=(T, n, kind, lead))
        scales(scale, y.abs().amax(1) / 127, 1)
        assert torch.equal(q.cpu(), stepwise(x)[0]) and torch.equal(scale.cpu(), stepwise(x)[1])
        for out in TYPES.values():
            obuf, o = room(T, n, n + pad, out, 5.0)
            dev.i8_dequant(q, scale, out=o)
            assert (obuf[:, n:] == 5.0).all()
            assert torch.equal(o, (q.float() * scale[:, None]).to(out))


@pytest.mark.parametrize("x,r,w", [("f32", None, "f32"), ("bf16", None, "bf16"), ("f16", None, "f32"), ("f32", "f32", "f32"),
                                   ("bf16", "bf16", "bf16"), ("f16", "f16", "f16"), ("bf16", "f32", "f32"),
                                   ("f16", "f32", "bf16"), ("f32", "bf16", "f16")])
@pytest.mark.parametrize("T,n", SIZES)
def test_norm(dev, T, n, x, r, w):
    g = torch.Generator().manual_seed(T * 100003 + n + 1)
    eps = 1e-5
    for lead, pad, where in ((0, 0, "apart"), (1, 3, "res"), (0, 0, "x")):
        if r is None and where != "apart" or where == "x" and x != r:
            continue
        xs = rand(g, T, n, x, lead, 1)
        wt = (1 + 0.3 * torch.randn(n, generator=g)).to(TYPES[w]).cuda()
        res = out = None
        h = xs
        if r is not None:
            res = rand(g, T, n, r, 0, lead)
            h = (xs.float() + res.float()).to(TYPES[r])
            obuf, out = room(T, n, n + pad, TYPES[r], 3.0)
            if where != "apart":
                obuf, out = None, res if where == "res" else xs
        buf, q = room(T, n, n + pad, torch.int8, 77)
        q, scale = dev.i8_rms_norm(xs, wt, eps, res=res, res_out=out, q=q)
        assert (buf[:, n:] == 77).all()
        if r is not None:
            assert torch.equal(out, h)
            if obuf is not None:
                assert (obuf[:, n:] == 3.0).all()
        v = h.cpu().double()
        y = v * wt.cpu().double()
        top, live, _ = check("norm", y, q, scale, names=(T, n, x, r, w))
        f = 1 / torch.sqrt((v * v).mean(1) + eps)
        # w h; the sum under the root; the mean, the sum with eps, root, reciprocal and two products
        scales(scale, top * f / 127, 1 + far(n) / 2 + 1 + 1 + 2 + 2, names=(T, n, x, r, w))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,n", SIZES)
def test_silu(dev, T, n, kind):
    g = torch.Generator().manual_seed(T * 100003 + n + 2)
    for halves in (True, False):
        if halves:
            both = rand(g, T, 2 * n, kind)
            gate, up = both[:, :n], both[:, n:]
        else:
            gate, up = rand(g, T, n, kind, 1, 0), rand(g, T, n, kind, 0, 2)
        buf, q = room(T, n, n + 3, torch.int8, 77)
        q, scale = dev.i8_silu_mul(gate, up, q=q)
        assert (buf[:, n:] == 77).all()
        a = gate.cpu().double()
        y = a / (1 + torch.exp(-a)) * up.cpu().double()
        top, live, k = check("silu", y, q, scale, names=(T, n, kind))
        scales(scale, top / 127, k + 1)


def test_silu_ends(dev):
    """Gates far out: silu(g) is g or (almost) 0, and stays a number."""
    gate = torch.tensor([[-3e38, -200.0, -100.0, -88.0, -20.0, -1e-30, 0.0, 1e-30, 20.0, 100.0, 60000.0]]).cuda()
    up = torch.ones_like(gate)
    q, scale = dev.i8_silu_mul(gate, up)
    y = torch.nn.functional.silu(gate.cpu().double())
    check("silu", y, q, scale)
    small = gate[:, :4].contiguous()
    q, scale = dev.i8_silu_mul(small, up[:, :4].contiguous())
    # the largest is silu(-88) = -88 e^-88, a normal fp32 number; the others are zeros beside it or below fp32
    assert q.cpu().tolist()[0][3] == -127 and scale.isfinite().all()


@pytest.mark.parametrize("n", [1, 9, 600, 5000, 40000])
def test_rows_that_stand_out(dev, n):
    """Zeros; an infinity; a NaN; the smallest and largest numbers; among ordinary rows."""
    g = torch.Generator().manual_seed(n)
    x = torch.randn((9, n), generator=g)
    x[1] = 0
    x[2, n // 2] = math.inf
    x[3, n - 1] = math.nan
    x[4, 0] = -math.inf
    x[5] *= 1e-41                 # below fp32's normal numbers
    x[6] *= 1e37 if n > 1 else 3e38 / x[6].abs()
    x[7] = -0.0
    x[8] = 1e-45
    xc, w = x.cuda(), torch.ones(n, device="cuda")
    bad = torch.tensor([i in (2, 3, 4) for i in range(9)])
    for name in ("quantize", "norm", "silu"):
        if name == "quantize":
            q, scale = dev.i8_quantize(xc)
        elif name == "norm":
            q, scale = dev.i8_rms_norm(xc, w, 1e-6)
        else:
            q, scale = dev.i8_silu_mul(torch.full_like(xc, 40.0), xc / 40)
        q, scale = q.cpu(), scale.cpu()
        assert scale[bad].isnan().all() and not q[bad].any(), name
        assert scale[~bad].isfinite().all(), name
        for i in (1, 7):
            assert scale[i] == 0 and not q[i].any(), name
        if name != "silu":
            ok = [0, 5, 6]
            ratio = x[ok].double() / x[ok].double().abs().amax(1, keepdim=True) * 127
            assert (q[ok].double() - ratio).abs().max() <= 0.5 + 127 * U * 5 * 1.01, name
            assert (q[8] == 127).all(), name
        out = dev.i8_dequant(q.cuda(), scale.cuda(), out_dtype=torch.float32).cpu()
        assert out[bad].isnan().all() and out[~bad].isfinite().all(), name


@pytest.mark.parametrize("n", [5, 2048, 33333])
@pytest.mark.parametrize("size", [1e25, 1e-25])
@pytest.mark.parametrize("where", ["none", "apart", "res"])
def test_norm_beyond_squares(dev, n, size, where):
    """Rows whose squares leave fp32 on either side, with eps 0: the factor is formed in 64 bits."""
    g = torch.Generator().manual_seed(n)
    x, res = torch.randn((3, n), generator=g) * size, torch.randn((3, n), generator=g) * size
    w = 1 + 0.3 * torch.randn(n, generator=g)
    h = x if where == "none" else x + res
    xc, rc = x.cuda(), None if where == "none" else res.cuda()
    out = None if where != "apart" else torch.empty_like(rc)
    q, scale = dev.i8_rms_norm(xc, w.cuda(), 0.0, res=rc, res_out=out)
    v = h.double()
    y = v * w.double()
    top, _, _ = check("norm", y, q, scale)
    scales(scale, top / torch.sqrt((v * v).mean(1)) / 127, 1 + 1 + 2 + 1)


def test_zero_rows_and_eps(dev):
    x, w = torch.zeros((2, 100), device="cuda"), torch.ones(100, device="cuda")
    for eps in (0.0, 1e-6):
        q, scale = dev.i8_rms_norm(x, w, eps)
        assert not q.any() and not scale.any()
    for call in (lambda: dev.i8_quantize(x[:0]), lambda: dev.i8_rms_norm(x[:0], w, 1e-6), lambda: dev.i8_silu_mul(x[:0], x[:0])):
        q, scale = call()
        assert q.shape == (0, 100) and scale.shape == (0,)


def test_many_short_rows(dev):
    x = torch.randn((70000, 24), generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    q, scale = dev.i8_quantize(x)
    assert torch.equal(q.cpu(), stepwise(x)[0]) and torch.equal(scale.cpu(), stepwise(x)[1])
    assert torch.equal(dev.i8_dequant(q, scale), (q.float() * scale[:, None]).bfloat16())


def test_many_elements(dev):
    """More than 2^31 elements: the last rows lie behind 32-bit offsets."""
    T, n = 65600, 32776
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty((T, n), dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, 32767, 65520, 65535, 65536, T - 1], device="cuda")
    rows = torch.randn((len(at), n), device="cuda", generator=g).bfloat16()
    x[at] = rows
    w = torch.ones(n, device="cuda")
    for call, alone in ((lambda: dev.i8_quantize(x), lambda: dev.i8_quantize(rows)),
                        (lambda: dev.i8_rms_norm(x, w, 1e-6), lambda: dev.i8_rms_norm(rows, w, 1e-6)),
                        (lambda: dev.i8_silu_mul(x, x), lambda: dev.i8_silu_mul(rows, rows))):
        (q, s), (q1, s1) = call(), alone()
        assert torch.equal(q[at], q1) and torch.equal(s[at], s1)
    assert torch.equal(dev.i8_dequant(q, s)[at], dev.i8_dequant(q1, s1))


@pytest.mark.parametrize("T,n", [((1 << 26) + 70, 8), ((1 << 24) + 5, 1032)])
def test_very_many_rows(dev, T, n):
    """More rows than one dimension of a launch has workgroups for."""
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.empty((T, n), dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, (1 << 21) - 1, 1 << 21, 1 << 23, T - 2, T - 1], device="cuda")
    rows = torch.randn((len(at), n), device="cuda", generator=g).bfloat16()
    x[at] = rows
    (q, s), (q1, s1) = dev.i8_quantize(x), dev.i8_quantize(rows)
    assert torch.equal(q[at], q1) and torch.equal(s[at], s1)
    del x
    assert torch.equal(dev.i8_dequant(q, s)[at], dev.i8_dequant(q1, s1))


def test_refused_tensors(dev):
    x, w = torch.zeros((3, 64), device="cuda"), torch.ones(64, device="cuda")
    cpu = torch.zeros((3, 64))
    q, scale = dev.i8_quantize(x)
    for bad, error in ((cpu, ValueError), (x.double(), TypeError), (x.to(torch.float8_e4m3fn), TypeError), (x.T, ValueError),
                       (x[0], ValueError), (x.to(torch.int8), TypeError)):
        for call in (lambda: dev.i8_quantize(bad), lambda: dev.i8_rms_norm(bad, w, 1e-6), lambda: dev.i8_silu_mul(bad, x),
                     lambda: dev.i8_silu_mul(x, bad), lambda: dev.i8_rms_norm(x, w, 1e-6, res=bad),
                     lambda: dev.i8_dequant(q, scale, out=bad)):
            with pytest.raises(error):
                call()
    for call in (lambda: dev.i8_quantize(x, q=x), lambda: dev.i8_quantize(x, q=q[:2]), lambda: dev.i8_quantize(x, scale=w),
                 lambda: dev.i8_rms_norm(x, w[:9], 1e-6), lambda: dev.i8_rms_norm(x, w.cpu(), 1e-6),
                 lambda: dev.i8_rms_norm(x, w, 1e-6, res_out=x), lambda: dev.i8_rms_norm(x, w, 1e-6, res=x, res_out=x.half()),
                 lambda: dev.i8_silu_mul(x, x.half()), lambda: dev.i8_dequant(q, scale[:2]), lambda: dev.i8_dequant(x, scale)):
        with pytest.raises((TypeError, ValueError)):
            call()
    with pytest.raises(RuntimeError, match="eps"):
        dev.i8_rms_norm(x, w, -1.0)
