"""The product of 8-bit integer rows with 8-bit integer weights (mllm_i8_gemm), against the sums in whole numbers.

acc is exact, (float)acc, its product with x_scale and that with w_scale round once each, the sum with the bias once
more, and the result to its type: |error| <= 2^-24 (3 |p| + |y|) + half a step of the type at y."""
import pytest
import torch

from mojollama_amd import kernels as K

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def dev():
    return K.DeviceOps()


def codes(g, T, n, lo=-128):
    return torch.randint(lo, 128, (T, n), dtype=torch.int8, generator=g)


def padded(q, fill=93, extra=0):
    """The rows at multiples of 16 bytes on the GPU, what lies behind them filled with other codes."""
    T, n = q.shape
    buf = torch.full((T, (n + 15) // 16 * 16 + 16 * extra), fill, dtype=torch.int8, device="cuda")
    buf[:, :n] = q.cuda()
    return buf[:, :n]


def want(w, ws, q, xs, bias):
    p = (q.cuda().double() @ w.cuda().double().T.contiguous()).cpu() * xs.double()[:, None] * ws.double()
    return p, p if bias is None else p + bias.double()


def near(out, p, y):
    out = out.cpu()
    eps = torch.finfo(out.dtype)
    # near zero the step is that of the type's smallest normal number
    tol = U * (3 * p.abs() + y.abs()) * 1.01 + (0 if out.dtype == torch.float32 else
                                               eps.eps / 2 * 1.01 * y.abs().clamp_min(eps.tiny))
    bad = (out.double() - y).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


def case(dev, T, R, C, out="bf16", bias=False, ld=0, extra=0, ws=None, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * T + 1009 * R + 104729 * C)
    w, q = codes(g, R, C), codes(g, T, C)
    wsc, xs = torch.rand(R, generator=g) * 0.01 + 1e-4, torch.rand(T, generator=g) + 0.01
    b = torch.randn(R, generator=g) if bias else None
    W = dev.i8_weights(w.cuda(), wsc.cuda())
    buf = torch.full((T, R + ld), 7.0, dtype=TYPES[out], device="cuda")
    o = buf[:, :R]
    dev.i8_gemm(W, padded(q, extra=extra), xs.cuda(), bias=None if b is None else b.cuda(), out=o, ws=ws)
    assert (buf[:, R:] == 7.0).all()
    near(o, *want(w, wsc, q, xs, b))


TOKENS = [1, 2, 3, 5, 8, 9, 15, 16, 17, 24, 31, 32, 33, 47, 48, 49, 63, 64, 65, 96, 100, 127, 128, 129, 160, 191, 192, 193, 255, 256,
          257, 300, 383, 385, 511, 512, 513, 700, 1021]


@pytest.mark.parametrize("T", TOKENS)
def test_tokens(dev, T):
    """Every number of tokens on both sides of the tiles, against a few shapes."""
    case(dev, T, 200, 320, "bf16", bias=True)
    case(dev, T, 1000, 2048, "f32")
    case(dev, T, 33, 4100, "f16", bias=True, ld=3)


@pytest.mark.parametrize("R,C", [(1, 1), (1, 16), (2, 15), (15, 17), (16, 33), (17, 64), (31, 127), (32, 128), (33, 129), (63, 255),
                                 (64, 256), (65, 257), (127, 383), (129, 1), (255, 640), (257, 1000), (300, 2881), (2883, 65),
                                 (4097, 130), (513, 16384), (7, 60000)])
@pytest.mark.parametrize("T", [1, 4, 16, 30, 70, 130, 270, 600])
def test_shapes(dev, T, R, C):
    case(dev, T, R, C, "f32", bias=True, ld=1)


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("ld", [0, 1, 2, 8])
@pytest.mark.parametrize("T,R,C", [(1, 257, 500), (12, 260, 512), (40, 264, 512), (100, 300, 2000), (300, 555, 700), (520, 1040, 256)])
def test_outputs(dev, T, R, C, out, bias, ld):
    """Types, bias and strides of out; x inside wider rows."""
    case(dev, T, R, C, out, bias, ld, extra=ld)


@pytest.mark.parametrize("T", [1, 20, 60, 150, 600])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_out_inside_a_wider_tensor(dev, T, out):
    """out begins at an odd element of its rows."""
    g = torch.Generator().manual_seed(T)
    w, q = codes(g, 333, 500), codes(g, T, 500)
    buf = torch.full((T, 341), 9.0, dtype=TYPES[out], device="cuda")
    dev.i8_gemm(dev.i8_weights(w.cuda(), torch.full((333,), 2.0 ** -8, device="cuda")), padded(q), torch.ones(T, device="cuda"),
                out=buf[:, 3:336])
    assert (buf[:, :3] == 9).all() and (buf[:, 336:] == 9).all()
    assert torch.equal(buf[:, 3:336].cpu(), (q.double() @ w.double().T / 256).to(TYPES[out]))


@pytest.mark.parametrize("T,R,C", [(1, 32000, 2048), (16, 4096, 4096), (96, 11264, 2048), (1021, 2883, 2881), (2048, 4096, 4096),
                                   (700, 8200, 1024), (5000, 256, 8192), (4099, 2048, 640), (3, 201088, 2880)])
def test_large(dev, T, R, C):
    case(dev, T, R, C, "bf16", bias=True)


@pytest.mark.parametrize("T,R,C", [(4395, 2808, 588), (803, 16265, 542), (2722, 900, 13500), (2538, 1589, 1056), (213, 5577, 11771),
                                   (3235, 962, 69), (598, 5345, 67), (3216, 41, 8198), (4278, 138, 74), (105, 8620, 65),
                                   (1203, 41, 3636), (556, 1800, 5351), (4341, 129, 1744), (1502, 45, 10297), (393, 473, 19424)])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_ragged_tiles(dev, T, R, C, out):
    """Tiles of every size with ragged ends in each direction, K whole and split."""
    case(dev, T, R, C, out, bias=True, ld=5, extra=1)


@pytest.mark.parametrize("T", [1, 20, 150, 400])
@pytest.mark.parametrize("x,w", [(-128, -128), (127, -128), (127, 127)])
def test_largest_sums(dev, T, x, w):
    """131071 products of the largest codes stay inside 32 bits."""
    R, C = 40, 131071
    W = dev.i8_weights(torch.full((R, C), w, dtype=torch.int8, device="cuda"), torch.ones(R, device="cuda"))
    q = padded(torch.full((T, C), x, dtype=torch.int8), fill=w)
    out = dev.i8_gemm(W, q, torch.ones(T, device="cuda"), out_dtype=torch.float32)
    assert (out == float(x * w * C)).all()


@pytest.mark.parametrize("T", [1, 17, 80, 300])
def test_scales_that_stand_out(dev, T):
    """A NaN or zero in a scale has its row or column alone, large and small scales do not leave fp32 in between."""
    g = torch.Generator().manual_seed(T)
    R, C = 130, 200
    w, q = codes(g, R, C, -127), codes(g, T, C, -127)
    w[3], q[T - 1, :] = 1, 1                       # a sum that is not zero at the corner
    wsc, xs = torch.ones(R), torch.ones(T)
    wsc[0], wsc[1], wsc[3], wsc[129] = float("nan"), 0.0, 1e-30, float("nan")
    xs[T - 1] = 1e30
    out = dev.i8_gemm(dev.i8_weights(w.cuda(), wsc.cuda()), padded(q), xs.cuda(), out_dtype=torch.float32)
    assert out[:, [0, 129]].isnan().all() and (out[:, 1] == 0).all() and not out[:, 2:129].isnan().any()
    assert abs(out[T - 1, 3].item() - 200.0) <= 200 * 4 * U
    if T > 1:
        xs[0] = float("nan")
        out = dev.i8_gemm(dev.i8_weights(w.cuda(), torch.ones(R).cuda()), padded(q), xs.cuda())
        assert out[0].isnan().all() and not out[1:].isnan().any()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,C,lead", [(1, 1, 0), (33, 100, 0), (40, 2881, 3), (70, 513, 1), (5, 40000, 0), (64, 2048, 0), (300, 9001, 2), (1100, 700, 0)])
def test_weights(dev, kind, R, C, lead):
    """Weights quantised here are those of i8_quantize: the product is the same, bit by bit."""
    g = torch.Generator().manual_seed(R + C)
    w = (0.02 * torch.randn((R, C + lead), generator=g)).to(TYPES[kind]).cuda()[:, lead:]
    if R > 2:
        w[1] = 0
    W = dev.i8_weights(w)
    q, s = dev.i8_quantize(w)
    assert torch.equal(W.scale, s)
    V = dev.i8_weights(q, s)
    assert torch.equal(W.packed, V.packed)
    x, xs = dev.i8_quantize(torch.randn((7, C), generator=g).cuda())
    assert torch.equal(dev.i8_gemm(W, x, xs), dev.i8_gemm(V, x, xs))


def test_weights_from_gguf(dev):
    """A Q4_K matrix of the framework, through dequant."""
    import numpy as np
    from mojollama_amd import workloads as WL
    rng = np.random.default_rng(3)
    raw = torch.from_numpy(WL.gen_weights(rng, WL.QT_Q4_K, 96, 512)).cuda()
    sem = dev.so.mllm_sem_for(K.ENT_BMM, WL.QT_Q4_K)
    dense = dev.dequant(sem, dev.pack(sem, raw, 96, 512), 96, 512)
    W = dev.i8_weights(dense)
    x = torch.randn((5, 512), generator=torch.Generator().manual_seed(0)).cuda()
    q, s = dev.i8_quantize(x)
    y = dev.i8_gemm(W, q, s, out_dtype=torch.float32).cpu().double()
    ref = x.cpu().double() @ dense.cpu().double().T
    # half a step of 1 / 127 of the largest on either side of each product
    xa, wa = x.cpu().double().abs(), dense.cpu().double().abs()
    dx, dw = xa.amax(1) / 254, wa.amax(1) / 254
    tol = dx[:, None] * wa.sum(1) + xa.sum(1)[:, None] * dw + 512 * dx[:, None] * dw
    assert ((y - ref).abs() <= tol * 1.001).all()


def test_workspace_of_more_tokens(dev):
    """A workspace for many tokens, filled with anything, serves fewer."""
    g = torch.Generator().manual_seed(0)
    w = codes(g, 300, 4096).cuda()
    W = dev.i8_weights(w, torch.ones(300, device="cuda"))
    ws = dev.i8_gemm_workspace(W, 700)
    for T in (700, 300, 257, 129, 128, 65, 64, 33, 17, 16, 3, 1):
        ws.fill_(255)
        q, s = padded(codes(g, T, 4096)), torch.ones(T, device="cuda")
        out = dev.i8_gemm(W, q, s, out_dtype=torch.float32, ws=ws)
        assert torch.equal(out.double(), q.double() @ w.double().T.contiguous())
    with pytest.raises(RuntimeError):
        need = dev.so.mllm_i8_gemm_workspace_size(300, 300, 4096)
        if need == 0:
            raise RuntimeError("no workspace is needed")
        dev.i8_gemm(W, padded(codes(g, 300, 4096)), torch.ones(300, device="cuda"), ws=ws[:need - 16])


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,C", [(200, 320), (1000, 2881), (70, 20000)])
def test_a_token_alone_or_among_others(dev, R, C, out):
    """A token's results are the same bits whatever the number of tokens, and whichever kernel that takes."""
    g = torch.Generator().manual_seed(R)
    W = dev.i8_weights(codes(g, R, C).cuda(), (torch.rand(R, generator=g) * 0.01).cuda())
    bias = torch.randn(R, generator=g).cuda()
    q, s = padded(codes(g, 1100, C)), torch.rand(1100, generator=g).cuda()
    for b in (None, bias):
        want = dev.i8_gemm(W, q, s, bias=b, out_dtype=TYPES[out])
        for T in (1, 5, 16, 17, 32, 40, 64, 70, 128, 200, 300, 600):
            at = slice(1100 - T, 1100)
            assert torch.equal(dev.i8_gemm(W, q[at], s[at], bias=b, out_dtype=TYPES[out]), want[at]), T


@pytest.mark.parametrize("T", [1, 30, 64, 200, 300])
def test_wide_strides(dev, T):
    """Rows of x just below 4 MB apart (32-bit offsets inside a tile) and at 4 MB (addresses of 64 bits)."""
    R, C = 150, 1000
    g = torch.Generator().manual_seed(T)
    w = codes(g, R, C).cuda()
    W, s = dev.i8_weights(w, torch.ones(R, device="cuda")), torch.ones(T, device="cuda")
    for ld in ((1 << 22) - 16, 1 << 22):
        q = torch.empty(T * ld, dtype=torch.int8, device="cuda").view(T, ld)[:, :C]
        q.copy_(codes(g, T, C))
        out = dev.i8_gemm(W, q, s, out_dtype=torch.float32)
        assert torch.equal(out.double(), q.double() @ w.double().T.contiguous())


def test_many_results(dev):
    """More than 2^31 results."""
    T, R, C = 70001, 32768, 48
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randint(-128, 128, (R, C), dtype=torch.int8, device="cuda", generator=g)
    q = torch.randint(-128, 128, (T, C), dtype=torch.int8, device="cuda", generator=g)
    out = dev.i8_gemm(dev.i8_weights(w, torch.ones(R, device="cuda")), q, torch.ones(T, device="cuda"))
    at = torch.tensor([0, 1, 255, 256, 30000, 65535, 65536, 69999, 70000], device="cuda")
    assert torch.equal(out[at], (q[at].double() @ w.double().T.contiguous()).float().bfloat16())


@pytest.mark.parametrize("R", [(1 << 26) - 16, (1 << 26) + 1])
def test_very_many_weight_rows(dev, R):
    """Rows on both sides of where the kernels of few tokens end."""
    C = 16
    g = torch.Generator(device="cuda").manual_seed(4)
    w = torch.randint(-128, 128, (R, C), dtype=torch.int8, device="cuda", generator=g)
    q = torch.randint(-128, 128, (2, C), dtype=torch.int8, device="cuda", generator=g)
    W = dev.i8_weights(w, torch.ones(R, device="cuda"))
    out = dev.i8_gemm(W, q, torch.ones(2, device="cuda"), out_dtype=torch.float32)
    at = torch.tensor([0, 1, 1 << 20, (1 << 25) + 7, R - 17, R - 1], device="cuda")
    assert torch.equal(out[:, at].double(), q.double() @ w[at].double().T.contiguous())


def test_far_rows(dev):
    """Rows of x and out beyond 2^31 bytes from the first."""
    T, C, R = 40, 100, 70
    g = torch.Generator().manual_seed(1)
    ld = (1 << 31) // 32 + 16
    big = torch.zeros(T * ld, dtype=torch.int8, device="cuda")
    q = big.view(T, ld)[:, :C]
    q.copy_(codes(g, T, C))
    far = torch.empty(T * (ld // 2 + 8), dtype=torch.bfloat16, device="cuda").view(T, -1)[:, :R]
    w = codes(g, R, C).cuda()
    dev.i8_gemm(dev.i8_weights(w, torch.ones(R, device="cuda")), q, torch.ones(T, device="cuda"), out=far)
    assert torch.equal(far, (q.double() @ w.double().T.contiguous()).float().bfloat16())


def test_refused_tensors(dev):
    W = dev.i8_weights(torch.zeros((40, 100), dtype=torch.int8, device="cuda"), torch.ones(40, device="cuda"))
    x = torch.zeros((3, 112), dtype=torch.int8, device="cuda")
    q, s = x[:, :100], torch.ones(3, device="cuda")
    dev.i8_gemm(W, q, s)
    for call in (lambda: dev.i8_gemm(W, x, s), lambda: dev.i8_gemm(W, q.cpu(), s), lambda: dev.i8_gemm(W, q.float(), s),
                 lambda: dev.i8_gemm(W, q, s[:2]), lambda: dev.i8_gemm(W, q, s, bias=s), lambda: dev.i8_gemm(W, q, s.double()),
                 lambda: dev.i8_gemm(W, q, s, out=torch.empty((3, 39), device="cuda")),
                 lambda: dev.i8_gemm(W, q, s, out_dtype=torch.int8), lambda: dev.i8_weights(x),
                 lambda: dev.i8_weights(x.float(), s), lambda: dev.i8_weights(x.float().T),
                 lambda: dev.i8_weights(torch.zeros((2, 131072), device="cuda")), lambda: dev.i8_weights(x.double()),
                 lambda: dev.i8_gemm(W, q, s, ws=torch.empty(256, dtype=torch.uint8))):
        with pytest.raises((TypeError, ValueError)):
            call()
    with pytest.raises(RuntimeError, match="16 bytes"):
        dev.i8_gemm(W, torch.zeros((3, 100), dtype=torch.int8, device="cuda"), s)
    with pytest.raises(RuntimeError, match="16 bytes"):
        dev.i8_gemm(W, x[:, 1:101], s)
    # one row needs no stride
    dev.i8_gemm(W, torch.zeros((1, 100), dtype=torch.int8, device="cuda"), s[:1])
    assert dev.i8_gemm(W, q[:0], s[:0]).shape == (0, 40)
