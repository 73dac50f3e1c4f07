"""How finely attention over a paged cache keeps the weights of its softmax with
16-bit queries and outputs: inputs whose scores and sums are exact in fp32, so
that nothing but the weights' precision and the output's one rounding is left."""
import math

import pytest
import torch

from mojollama_amd import kernels as K
from paged_ref import BF16, E4M3, F16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return K.DeviceOps(K.load_kernels())


def i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def setup(dev, cache, S, NKH, HD, page):
    """One sequence of S rows; elements of K and V are multiples of 1/8 up to 1, which every type holds."""
    g = torch.Generator().manual_seed(S + HD)
    n = -(-S // page)
    k, v = (torch.randint(-8, 9, (n, page, NKH, HD), generator=g) / 8 for _ in range(2))
    raw = [x.to(cache).cuda() for x in (k, v)]
    exps = [torch.full((n, NKH, page), 127, dtype=torch.uint8, device="cuda")] * 2 if cache == E4M3 else []
    view = dev.paged_kv(*raw, torch.arange(n, dtype=torch.int32)[None].cuda(), *exps)
    return view, *(x.double().reshape(-1, NKH, HD)[:S] for x in (k, v))


def check(got, q, pos, k, v, window, cache, scale):
    """Scores are exact (multiples of 1/8, at most HD of them at most 1); times scale * log2(e), itself rounded three
    times, they are off by 4 |z| 2^-24, the subtraction of the maximum by as much again and the exponential by 2^-23:
    with |z| < 12 a weight by d < 2^-17, a normalised one by 2 d.  The two sums over n rows are fp32, n 2^-24 each.  Two
    planes keep a weight to 2^-15 (bf16: truncated to 8 + 8 bits) or 2^-22 (fp16: 11 + 11, one bit for the order of
    the roundings).  Then the output's rounding, half a step."""
    rep = q.shape[1] // k.shape[1]
    s = torch.arange(len(k))
    see = s[None] <= pos[:, None]
    if window:
        see &= s[None] > pos[:, None] - window
    k, v = (x.repeat_interleave(rep, 1).transpose(0, 1).contiguous() for x in (k, v))       # [NH][S][HD]
    z = torch.matmul(q.transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) * scale
    z = z.masked_fill(~see[None], -math.inf)
    assert z[z > -math.inf].abs().max() / math.log(2) < 12
    w = torch.softmax(z, -1)
    o, mag = torch.matmul(w, v).transpose(0, 1), torch.matmul(w, v.abs()).transpose(0, 1)
    n = int(see.sum(1).max())
    rel = 2 * 2.0 ** -17 + 2 * (n + 32) * 2.0 ** -24 + (2.0 ** -22 if cache == F16 else 2.0 ** -15)
    half = torch.finfo(F16 if cache == F16 else BF16).eps / 2
    bound = mag * rel * (1 + half) + o.abs() * half + (2.0 ** -25 if cache == F16 else 0.0)
    off = (got.double().cpu().view(o.shape) - o).abs()
    assert (off <= bound).all(), (float((off / bound).max()), int((off > bound).sum()), off.numel())


def queries(seed, n, NH, HD):
    """-1, 0 and 1: exact products, scores of a few units."""
    return torch.randint(-1, 2, (n, NH * HD), generator=torch.Generator().manual_seed(seed)).float()


# rows of the cache: few enough that the sums' own bound stays below a weight rounded to one plane
SIZES = [(BF16, 30), (BF16, 400), (E4M3, 30), (E4M3, 400), (F16, 30)]


@pytest.mark.parametrize("cache,S", SIZES)
@pytest.mark.parametrize("HD", [64, 128, 256])
def test_decode_keeps_two_planes(dev, cache, S, HD):
    NH, NKH, scale = 8, 2, HD ** -0.5
    kv, k, v = setup(dev, cache, S, NKH, HD, 16)
    act = F16 if cache == F16 else BF16
    q = queries(HD, 1, NH, HD)
    got = dev.paged_attn_decode(kv, q.to(act).cuda(), i32([S]), S, NH, scale=scale)
    check(got, q.double().view(1, NH, HD), torch.tensor([S - 1]), k, v, 0, cache, scale)


@pytest.mark.parametrize("cache,S", SIZES)
@pytest.mark.parametrize("HD,page", [(64, 16), (128, 64), (80, 25), (256, 64)])
def test_prompt_keeps_two_planes(dev, cache, S, HD, page):
    NH, NKH, scale = 8, 2, HD ** -0.5
    kv, k, v = setup(dev, cache, S, NKH, HD, page)
    act = F16 if cache == F16 else BF16
    q = queries(HD, S, NH, HD)
    got = dev.paged_attn_prompt(kv, q.to(act).cuda(), i32([0, S]), i32([S]), S, NH, scale=scale)
    check(got, q.double().view(S, NH, HD), torch.arange(S), k, v, 0, cache, scale)


@pytest.mark.parametrize("cache,HD", [(BF16, 64), (BF16, 128), (F16, 64), (F16, 128), (E4M3, 128)])
def test_long_prompt_keeps_two_planes(dev, cache, HD):
    """From 65536 rows of queries on, on pages of multiples of 64 rows, in tiles of 256; a window keeps the sums short."""
    NH, NKH, S, window, scale = 32, 8, 2100, 30, HD ** -0.5
    kv, k, v = setup(dev, cache, S, NKH, HD, 64)
    act = F16 if cache == F16 else BF16
    q = queries(HD, S, NH, HD)
    got = dev.paged_attn_prompt(kv, q.to(act).cuda(), i32([0, S]), i32([S]), S, NH, scale=scale, window=window)
    at = torch.tensor([0, 1, 29, 30, 31, 63, 64, 65, 127, 128, 1000, 1023, 1024, 2047, 2048, 2098, 2099])
    check(got[at.cuda()], q.double().view(S, NH, HD)[at], at, k, v, window, cache, scale)
