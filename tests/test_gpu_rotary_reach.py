"""mllm_rotary_append where its stores go past the caches (more than 32 MB of
output), rows for an 8-bit cache whose rotation leaves fp32's range, and
frequencies of the caller's own."""
import math

import pytest
import torch

from mojollama_amd import kernels as K
from paged_ref import BF16, E4M3, F16, F32, Cache
from test_gpu_rotary import near, stored, turn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return K.DeviceOps(K.load_kernels())


def i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


@pytest.mark.parametrize("layout,r", [(K.ROPE_HALF, 128), (K.ROPE_PAIRS, 64), (K.ROPE_HALF, 40)])
@pytest.mark.parametrize("act,cache", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F32, E4M3)])
@pytest.mark.parametrize("odd", [0, 3])
def test_stores_past_the_caches(dev, layout, r, act, cache, odd):
    """q and k in place in a fused buffer, its rows multiples of 16 bytes or not; two sequences whose tokens alternate,
    every 97th token left out, some rows outside the tables."""
    NH, NKH, HD, T = 32, 8, 128, 2800
    assert T * (NH * HD * 2 + 2 * NKH * HD * 2) > 32 << 20
    c = Cache(r + odd, [1390, 1400], NKH, HD, 16, cache, wide=0)
    kv = c.view(dev)
    seqs = torch.arange(T) % 2
    pos = torch.arange(T) // 2
    pos[::97] = -1
    a, b = NH * HD, NKH * HD
    g = torch.Generator().manual_seed(r)
    buf = torch.randn(T, a + 2 * b + odd, generator=g).to(act)
    d = buf.cuda()
    q, k, v = d[:, odd:odd + a], d[:, odd + a:odd + a + b], d[:, odd + a + b:]
    rot = dev.rotary(r, layout=layout, base=10000.0)
    dev.rotary_append(rot, q, k, v, pos.int().cuda(), NH=NH, kv=kv, seqs=seqs.int().cuda(), q_out=q, k_out=k)
    x = buf[:, odd:].double().view(T, NH + 2 * NKH, HD)
    got, keep = d.cpu(), pos < 0
    assert torch.equal(got[keep], buf[keep]) and torch.equal(got[:, odd + a + b:], buf[:, odd + a + b:])
    assert torch.equal(got[:, :odd], buf[:, :odd])
    want = turn(x[:, :NH + NKH], pos.clamp(min=0), rot, layout)
    near(got[~keep][:, odd:odd + a + b], want[~keep], x[~keep][:, :NH + NKH], act, 1.0)
    on = ~keep & (pos < torch.where(seqs == 0, 87 * 16, 88 * 16))        # 87 and 88 pages are mapped
    assert int((~on & ~keep).sum()) > 0
    stored(kv, c, seqs[on].tolist(), pos[on].tolist(), want[on][:, NH:], x[on][:, NH + NKH:], x[on][:, NH:NH + NKH], 1.0)


def test_e4m3_beyond_fp32(dev):
    """Elements that the rotation takes past fp32's largest number saturate, at the largest scale in a row of finite
    ones, at 448 in a row that holds an infinity."""
    NKH, HD, big = 1, 16, 3e38
    c = Cache(3, [2], NKH, HD, 16, E4M3)
    kv = c.view(dev)
    x = torch.zeros(2, HD)
    x[:, 0] = x[:, 8] = big                      # 3e38 (cos 1 - sin 1), 3e38 (cos 1 + sin 1)
    x[1, 3] = math.inf                           # and of its pair's other element, 0, infinity times sin
    dev.rotary_append(dev.rotary(16), None, x.cuda(), x.cuda(), i32([1, 1]), kv=kv, seqs=i32([0, 0]), rows=i32([0, 1]))
    p = int(c.tables[0, 0])
    code = kv._tensors[0][p, :2, 0].cpu().double()
    assert kv._tensors[3][p, 0, :2].tolist() == [227, 127]                # 2^100, the largest scale, and 2^0
    assert code[0, [0, 8]].tolist() == [-448.0, 448.0]
    assert code[1, [0, 8]].tolist() == [-448.0, 448.0]
    assert torch.isnan(code[1, [3, 11]]).all() and not torch.isnan(code[1, [1, 2, 4, 9, 15]]).any()


@pytest.mark.parametrize("layout", [K.ROPE_HALF, K.ROPE_PAIRS])
def test_own_frequencies(dev, layout):
    """Frequencies and a factor of the caller's own: here a ramp whose ends are not rounded to whole pairs."""
    r, base, f, ctx, pos = 64, 150000.0, 32.0, 4096.0, torch.tensor([0, 1, 77, 4095, 131071], dtype=torch.int32)
    j = torch.arange(r // 2, dtype=torch.float64)
    w = base ** (-2 * j / r)
    lo, hi = (r * math.log(ctx / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (32.0, 1.0))
    ramp = ((j - lo) / (hi - lo)).clamp(0, 1)
    own = w / f * ramp + w * (1 - ramp)
    x = torch.randn(len(pos), 2, r, generator=torch.Generator().manual_seed(1))
    for freqs in (own, own.cuda(), own.tolist()):
        rot = dev.rotary(r, layout=layout, freqs=freqs, mscale=1.25)
        assert torch.equal(rot._tensors[0].cpu(), own) and rot.mscale == 1.25
        out = torch.empty(len(pos), 2 * r, device="cuda")
        dev.rotary_append(rot, x.view(len(pos), -1).cuda(), None, None, pos.cuda(), NH=2, HD=r, q_out=out)
        near(out, turn(x.double(), pos, rot, layout), x.double(), F32, 1.25)
    assert dev.rotary(r, freqs=own).mscale == 1.0
    assert dev.rotary(r, scaling=K.ROPE_YARN, factor=f, ctx=ctx, mscale=2.0).mscale == 2.0
    for bad in (own[:-1], own[None], [0.0] * 33, torch.full_like(own, math.nan)):
        with pytest.raises(ValueError):
            dev.rotary(r, freqs=bad)
    with pytest.raises(ValueError):
        dev.rotary(r, freqs=own, scaling=K.ROPE_YARN, factor=f, ctx=ctx)
    with pytest.raises(ValueError):
        dev.rotary(r, mscale=math.nan)
    with pytest.raises(ValueError):
        dev.rotary(63, freqs=[1.0] * 31)
