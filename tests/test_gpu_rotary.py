"""mllm_rotary_append against the rotation in 64 bits: layouts, widths, scalings,
far positions, types, strides, in place, and what is stored into paged caches
of each type -- an 8-bit cache code by code."""
import math

import pytest
import torch

from mojollama_amd import kernels as K
from paged_ref import BF16, E4M3, F16, F32, Cache, quantise_e4m3

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return K.DeviceOps(K.load_kernels())


def turn(x, pos, rot, layout):
    """x [T][heads][HD] in 64 bits."""
    r = rot.rope_dim
    f = rot._tensors[0].cpu()[:r // 2]
    a = pos.double()[:, None] * f
    c, s = (y[:, None] * rot.mscale for y in (torch.cos(a), torch.sin(a)))
    y = x.clone()
    if layout == K.ROPE_HALF:
        p, q = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = p * c - q * s, q * c + p * s
    else:
        p, q = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = p * c - q * s, q * c + p * s
    return y


def near(got, want, x, dtype, mscale):
    """fp32 cosine and sine of an angle reduced in 64 bits are off by at most 2^-22 (the reduced angle's rounding,
    pi 2^-25 .. pi 2^-24, and the function's), the products and their sum by 2^-23 of a pair's size, at most sqrt(2) of
    its larger element; then one rounding to the type."""
    big = x.abs().amax(-1, keepdim=True)
    tol = 4 * mscale * big * 2.0 ** -22 + want.abs() * torch.finfo(dtype).eps / 2 + (2.0 ** -24 if dtype == F16 else 1e-30)
    assert ((got.double().cpu().view(want.shape) - want).abs() <= tol).all()


@pytest.mark.parametrize("layout", [K.ROPE_HALF, K.ROPE_PAIRS])
@pytest.mark.parametrize("HD,r", [(64, 64), (128, 128), (96, 48), (80, 20), (256, 256), (16, 2), (64, 0), (80, 76)])
@pytest.mark.parametrize("inp,out,cache", [(F32, BF16, BF16), (BF16, BF16, BF16), (F16, F16, F16), (F32, F32, E4M3),
                                           (BF16, F32, E4M3)])
def test_rotary_append(dev, layout, HD, r, inp, out, cache):
    NH, NKH, page = 6, 3, 16
    c = Cache(HD + r, [70, 40, 5], NKH, HD, page, cache)
    kv = c.view(dev)
    seqs, pos = [0] * 20 + [2] + [1] * 12, list(range(40, 60)) + [4] + list(range(3, 15))
    T = len(pos)
    x = torch.randn(T, NH + 2 * NKH, HD, generator=torch.Generator().manual_seed(r)).to(inp)
    rot = dev.rotary(r, layout=layout, base=10000.0)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    qkv = x.view(T, -1).cuda()
    a, b = NH * HD, NKH * HD
    q_out = torch.zeros(T, a, dtype=out, device="cuda")
    k_out = torch.zeros(T, b, dtype=out, device="cuda")
    dev.rotary_append(rot, qkv[:, :a], qkv[:, a:a + b], qkv[:, a + b:], i32(pos), NH=NH, kv=kv, seqs=i32(seqs), q_out=q_out,
                      k_out=k_out)
    w = x.double()
    near(q_out, turn(w[:, :NH], torch.tensor(pos), rot, layout), w[:, :NH], out, rot.mscale)
    want_k = turn(w[:, NH:NH + NKH], torch.tensor(pos), rot, layout)
    near(k_out, want_k, w[:, NH:NH + NKH], out, rot.mscale)
    stored(kv, c, seqs, pos, want_k, w[:, NH + NKH:], w[:, NH:NH + NKH], rot.mscale)


def stored(kv, c, seqs, rows, want_k, want_v, x, mscale):
    """The rows hold the tokens' k and v, every other byte of the pools what it held."""
    at = c.tables[torch.tensor(seqs).long(), torch.tensor(rows) // c.page].long()
    row = torch.tensor(rows) % c.page
    for i, (pool, exp, want) in enumerate(zip(kv._tensors[:2], kv._tensors[3:], (want_k, want_v))):
        bits = lambda t: t.contiguous().view(torch.uint8 if c.dtype == E4M3 else torch.int16)  # noqa: E731
        was, now = bits(c.pools[i]).clone(), bits(pool.cpu())
        if c.dtype == E4M3:
            y, e = quantise_e4m3(want)
            was[at, row] = y.float().to(E4M3).view(torch.uint8)
            assert torch.equal(now, was)
            wexp = c.exps[i].clone()
            wexp.transpose(1, 2)[at, row] = (e + 127).to(torch.uint8)
            assert torch.equal(exp.cpu(), wexp)
        else:
            got = pool.cpu()[at, row]
            if i == 0:
                near(got, want, x, c.dtype, mscale)
            else:
                assert torch.equal(got, want.to(c.dtype))
            now[at, row] = was[at, row]
            assert torch.equal(now, was)


@pytest.mark.parametrize("scaling", [K.ROPE_NONE, K.ROPE_LINEAR, K.ROPE_NTK, K.ROPE_YARN, K.ROPE_BANDS])
def test_far_positions(dev, scaling):
    """Positions up to 2^31 - 1 keep their angle."""
    rot = dev.rotary(64, base=150000.0, scaling=scaling, factor=32.0, ctx=4096.0)
    pos = torch.tensor([0, 1, 4095, 131071, 1 << 24, (1 << 31) - 1], dtype=torch.int32)
    x = torch.randn(len(pos), 4, 64, generator=torch.Generator().manual_seed(1))
    out = torch.empty(len(pos), 256, device="cuda")
    dev.rotary_append(rot, x.view(len(pos), -1).cuda(), None, None, pos.cuda(), NH=4, HD=64, q_out=out)
    near(out, turn(x.double(), pos, rot, K.ROPE_HALF), x.double(), F32, rot.mscale)


def test_in_place_strides_and_left_out_tokens(dev):
    """q and k in place inside a fused buffer whose rows are not multiples of 16 bytes; tokens at negative positions
    keep their values, tokens of sequences or rows outside the tables are turned and not stored."""
    NH, NKH, HD, T = 3, 2, 64, 9
    c = Cache(3, [40, 20], NKH, HD, 16, BF16)
    kv = c.view(dev)
    ld = (NH + 2 * NKH) * HD + 3
    buf = torch.randn(T, ld, generator=torch.Generator().manual_seed(2))
    pos = torch.tensor([3, -1, 5, 17, 39, 2, 1000, -7, 8], dtype=torch.int32)
    seqs = torch.tensor([0, 0, 1, -1, 0, 2, 0, 1, 1], dtype=torch.int32)
    rot = dev.rotary(64, layout=K.ROPE_HALF)
    g = buf.cuda()
    a, b = NH * HD, NKH * HD
    q, k, v = g[:, 1:1 + a], g[:, 1 + a:1 + a + b], g[:, 1 + a + b:1 + a + 2 * b]
    dev.rotary_append(rot, q, k, v, pos.cuda(), NH=NH, kv=kv, seqs=seqs.cuda(), q_out=q, k_out=k)
    x = buf[:, 1:1 + a + b].double().view(T, NH + NKH, HD)
    want = turn(x, pos.clamp(min=0), rot, K.ROPE_HALF)
    keep = pos < 0
    want[keep] = x[keep]
    got = g.cpu()
    near(got[:, 1:1 + a + b], want, x, F32, 1.0)
    assert torch.equal(got[keep], buf[keep])
    assert torch.equal(got[:, 1 + a + b:], buf[:, 1 + a + b:]) and torch.equal(got[:, 0], buf[:, 0])
    on = [0, 2, 4, 8]
    stored(kv, c, seqs[on].tolist(), pos[on].tolist(), want[on][:, NH:], buf[on][:, 1 + a + b:1 + a + 2 * b].double().view(
        len(on), NKH, HD), x[on][:, NH:], 1.0)


def test_rows_apart_from_positions(dev):
    """Cache rows given beside the rotary positions, without rotation of the stored tokens' order."""
    NKH, HD = 2, 32
    c = Cache(3, [64], NKH, HD, 16, F16)
    kv = c.view(dev)
    pos, rows = [100, 7, 0], [0, 63, 30]
    x = torch.randn(3, 2 * NKH, HD, generator=torch.Generator().manual_seed(2)).to(F16)
    rot = dev.rotary(16, layout=K.ROPE_PAIRS)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    g = x.view(3, -1).cuda()
    dev.rotary_append(rot, None, g[:, :NKH * HD], g[:, NKH * HD:], i32(pos), kv=kv, seqs=i32([0, 0, 0]), rows=i32(rows))
    w = x.double()
    stored(kv, c, [0, 0, 0], rows, turn(w[:, :NKH], torch.tensor(pos), rot, K.ROPE_PAIRS), w[:, NKH:], w[:, :NKH], 1.0)


def test_e4m3_edges(dev):
    """Rows of zeros, of one element, at 448 2^k and just above, tiny and huge rows, ties between codes, infinities
    and NaN."""
    NKH, HD = 1, 16
    rows = torch.zeros(10, HD, dtype=torch.float64)
    rows[1, 3] = -5.0
    rows[2] = torch.arange(HD) * 2.0 ** 20
    rows[2, 15] = 448.0 * 2.0 ** 17
    rows[3, 0], rows[3, 1] = 449.0, 1.0
    rows[4] = torch.linspace(1, 2, HD, dtype=torch.float64) * 1e-37
    rows[5] = torch.linspace(-1, 1, HD, dtype=torch.float64) * 3e38
    rows[6, 0], rows[6, 1:] = 448.0, torch.arange(1, HD) * 2.0 ** -10          # halves of the least step
    rows[7, 0], rows[7, 1:] = 256.0, 17.0 + torch.arange(HD - 1)               # ties between codes
    rows[8, 0], rows[8, 1], rows[8, 2], rows[8, 3] = math.inf, -math.inf, math.nan, 1000.0
    rows[9] = torch.randn(HD, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    c = Cache(3, [10], NKH, HD, 16, E4M3)
    kv = c.view(dev)
    x = rows.float().cuda()
    pos = torch.arange(10, dtype=torch.int32).cuda()
    dev.rotary_append(dev.rotary(0), None, x, x, pos, kv=kv, seqs=torch.zeros_like(pos))
    y, e = quantise_e4m3(rows.float().double())
    e[8] = 0
    y[8] = torch.where(torch.isfinite(rows[8]), rows[8].clamp(-448, 448), math.nan)
    p = int(c.tables[0, 0])
    for pool, exp in zip(kv._tensors[:2], kv._tensors[3:]):
        got = pool[p, :10, 0].cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(y))
        assert torch.equal(got.nan_to_num(), y.nan_to_num())
        assert torch.equal(exp[p, 0, :10].cpu().int(), (e + 127).int())


def test_wrapper_refusals(dev):
    rot = dev.rotary(64)
    q = torch.zeros(2, 128, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (dict(q=q[:, :64]), dict(q_out=q[:1]), dict(pos=pos.long()), dict(HD=32), dict(q_out=None), dict(q=q.double())):
        a = dict(q=q, k=None, v=None, pos=pos, NH=2, HD=64, q_out=q) | bad
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            dev.rotary_append(rot, **a)
    with pytest.raises(RuntimeError):
        dev.rotary(63)
