"""mllm_rotary_append where its stores go past the caches (more than 32 MB of
output)."""
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
