"""Attention over a paged 16- or 8-bit cache (mllm_paged_attn_decode, _prompt)
against the definition in 64 bits: cache types, fp32 and 16-bit queries, head
layouts and sizes, pages that end inside a tile, lengths from none to some
thousands, windows, sinks, unmapped pages, NaN in every row that no query sees."""
import pytest
import torch

from mojollama_amd import kernels as K
from paged_ref import BF16, E4M3, F16, F32, Cache, attend, attend_bound

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return K.DeviceOps(K.load_kernels())


def queries(seed, n, NH, HD, dtype):
    return (1.5 * torch.randn(n, NH * HD, generator=torch.Generator().manual_seed(seed))).to(dtype)


def check(got, cache, b, q, pos, scale, window, sinks, q_dtype, out_dtype, NH):
    o, mag, za, zq = attend(cache, b, q.double().view(len(q), NH, cache.HD), pos, scale, window, sinks)
    got = got.double().cpu().view(o.shape)
    assert torch.isfinite(got).all()
    bound = attend_bound(o, mag, za, zq, cache.rows[b], cache.HD, cache.dtype, q_dtype, out_dtype)
    worst = ((got - o).abs() / bound).max() if o.numel() else 0
    assert worst <= 1, (b, float(worst), float((got - o).abs().max()))


def decode(dev, cache, lens, NH, q_dtype, out_dtype, window=0, sinks=None, seqs=None, max_len=None, scale=None, seed=0):
    B, HD = len(lens), cache.HD
    q = queries(seed, B, NH, HD, q_dtype)
    if sinks is not None:
        sinks = torch.randn(NH, generator=torch.Generator().manual_seed(seed + 1)) * 3
    s = None if seqs is None else torch.tensor(seqs, dtype=torch.int32).cuda()
    got = dev.paged_attn_decode(cache.view(dev), q.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                max(lens) if max_len is None else max_len, NH, scale=scale, window=window,
                                sinks=None if sinks is None else sinks.cuda(), seqs=s, out_dtype=out_dtype)
    scale = HD ** -0.5 if scale is None else scale
    for i, n in enumerate(lens):
        b = i if seqs is None else seqs[i]
        if max_len is not None:
            n = min(n, max_len)
        if not 0 <= b < len(cache.rows):
            assert not got[i].any()
            continue
        check(got[i:i + 1], cache, b, q[i:i + 1], torch.tensor([n - 1]), scale, window, sinks, q_dtype, out_dtype, NH)
    return got


TYPES = [(BF16, BF16, BF16), (F16, F16, F16), (E4M3, BF16, BF16), (BF16, F32, F32), (F16, F32, F32), (E4M3, F32, F32),
         (BF16, BF16, F32), (F16, F32, F16)]


@pytest.mark.parametrize("cache,q,out", TYPES)
@pytest.mark.parametrize("NH,NKH,HD", [(8, 1, 64), (12, 3, 80), (32, 8, 128), (7, 7, 16), (20, 1, 96), (6, 2, 256)])
def test_decode_types_and_heads(dev, cache, q, out, NH, NKH, HD):
    lens = [1, 40, 257, 16, 31, 700]
    decode(dev, Cache(HD + NH, lens, NKH, HD, 32, cache), lens, NH, q, out, seed=HD)


@pytest.mark.parametrize("page", [1, 16, 48, 64, 100, 1000])
@pytest.mark.parametrize("cache,q", [(BF16, BF16), (E4M3, BF16), (F16, F32)])
@pytest.mark.parametrize("lens", [[1], [0], [15, 17, 64, 65, 0, 1, 129], [2500, 3], [333] * 9])
def test_decode_pages_and_lengths(dev, page, cache, q, lens):
    decode(dev, Cache(page + len(lens), lens, 2, 64, page, cache), lens, 8, q, q, seed=page)


@pytest.mark.parametrize("cache,q", [(BF16, BF16), (E4M3, F32)])
@pytest.mark.parametrize("window", [1, 31, 64, 200, 100000])
@pytest.mark.parametrize("sinks", [None, True])
def test_decode_windows_and_sinks(dev, cache, q, window, sinks):
    lens = [1, 64, 65, 1500, 0, 333]
    decode(dev, Cache(window, lens, 2, 128, 16, cache), lens, 14, q, q, window=window, sinks=sinks, seed=window)


@pytest.mark.parametrize("cache,q", [(BF16, BF16), (E4M3, BF16), (F16, F32)])
@pytest.mark.parametrize("head_major", [False, True])
def test_decode_unmapped_pages_and_slots(dev, cache, q, head_major):
    """Unmapped pages take no part (a sequence of nothing else gives zeros); sequences by slot, one twice, two
    outside the tables; lengths above max_len are cut."""
    rows = [200, 33, 64, 500]
    c = Cache(5, rows, 3, 64, 16, cache, head_major=head_major,
              unmapped=[(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (3, 31)])
    decode(dev, c, rows, 6, q, q, seed=3)
    slots = [3, 1, 3, -1, 2, 7]
    decode(dev, c, [500, 33, 100, 40, 64, 5], 6, q, q, seqs=slots, max_len=450, seed=4)


def test_decode_long_pool_past_32_bits(dev):
    """Rows more than 2^32 bytes, and 2^31 elements, into the pools."""
    NKH, HD, page = 8, 128, 64
    n_pages = 2 ** 31 // (page * NKH * HD) + 40
    k = torch.zeros(n_pages, page, NKH, HD, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    c = Cache(9, [300, 77], NKH, HD, page, BF16)
    at = torch.arange(c.n_pages, device="cuda") + n_pages - c.n_pages
    k[at], v[at] = c.pools[0].cuda(), c.pools[1].cuda()
    t = c.tables.clone()
    t[t >= 0] += n_pages - c.n_pages
    q = queries(1, 2, 16, HD, BF16)
    got = dev.paged_attn_decode(dev.paged_kv(k, v, t.cuda()), q.cuda(), torch.tensor(c.rows, dtype=torch.int32).cuda(), 300, 16)
    for b, n in enumerate(c.rows):
        check(got[b:b + 1], c, b, q[b:b + 1], torch.tensor([n - 1]), HD ** -0.5, 0, None, BF16, BF16, 16)


def test_decode_strided_rows_and_outputs(dev):
    """q and out as slices of wider rows; what lies beside out keeps its contents."""
    lens, NH, HD = [90, 7], 4, 64
    c = Cache(2, lens, 2, HD, 32, F16)
    q = queries(5, 2, NH + 3, HD, F32)
    out = torch.full((2, (NH + 1) * HD), 7.0, dtype=F16, device="cuda")
    dev.paged_attn_decode(c.view(dev), q.cuda()[:, HD:(NH + 1) * HD], torch.tensor(lens, dtype=torch.int32).cuda(), 90, NH,
                          out=out[:, :NH * HD])
    assert (out[:, NH * HD:] == 7).all()
    for b, n in enumerate(lens):
        check(out[b:b + 1, :NH * HD], c, b, q[b:b + 1, HD:(NH + 1) * HD], torch.tensor([n - 1]), HD ** -0.5, 0, None, F32,
              F16, NH)


def test_decode_extreme_scores(dev):
    """Scores of hundreds: the maximum carries the softmax, and equal maxima share it."""
    lens = [600]
    for cache, q in ((BF16, BF16), (F16, F32), (E4M3, F32)):
        decode(dev, Cache(8, lens, 1, 64, 64, cache), lens, 4, q, q, scale=20.0 if q == F32 else 3.0, seed=8)


# ------------------------------------------------------------------ prompt
def prompt(dev, cache, new, NH, q_dtype, out_dtype, window=0, sinks=None, seqs=None, behind=0, lens=None, scale=None,
           shrink=1.0, seed=0):
    """Sequence i's last new[i] rows are its new tokens; `behind` rows of q and out behind the last sequence."""
    HD, B = cache.HD, len(new)
    slots = list(range(B)) if seqs is None else seqs
    lens = [cache.rows[b] for b in slots] if lens is None else lens
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    T = starts[-1] + behind
    q = (queries(seed, T, NH, HD, F32) * shrink).to(q_dtype)
    scale = HD ** -0.5 if scale is None else scale
    if sinks is not None:
        sinks = torch.randn(NH, generator=torch.Generator().manual_seed(seed + 1)) * 3
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    out = torch.full((T, NH * HD), 7.0, dtype=out_dtype, device="cuda")
    dev.paged_attn_prompt(cache.view(dev), q.cuda(), i32(starts), i32(lens), max(lens + [0]), NH, scale=scale, window=window,
                          sinks=None if sinks is None else sinks.cuda(), seqs=None if seqs is None else i32(seqs), out=out)
    assert (out[starts[-1]:] == 7).all()
    for i, n in enumerate(new):
        if n:
            pos = torch.arange(n) + lens[i] - n
            check(out[starts[i]:starts[i] + n], cache, slots[i], q[starts[i]:starts[i] + n], pos, scale, window,
                  sinks, q_dtype, out_dtype, NH)


@pytest.mark.parametrize("cache,q,out", TYPES)
@pytest.mark.parametrize("NH,NKH,HD", [(8, 1, 64), (12, 3, 80), (16, 4, 128), (7, 7, 16), (20, 1, 96), (6, 2, 256)])
def test_prompt_types_and_heads(dev, cache, q, out, NH, NKH, HD):
    new, past = [1, 40, 131, 16], [0, 3, 70, 200]
    prompt(dev, Cache(HD + NH, [a + b for a, b in zip(new, past)], NKH, HD, 32, cache), new, NH, q, out, seed=HD)


@pytest.mark.parametrize("page", [1, 16, 48, 64, 100])
@pytest.mark.parametrize("cache,q", [(BF16, BF16), (E4M3, BF16), (F16, F32)])
@pytest.mark.parametrize("new,past", [([1], [0]), ([5, 5, 3], [900, 1300, 0]), ([0, 300, 0, 64, 65], [10, 0, 0, 64, 63]),
                                      ([515], [0]), ([1] * 20, list(range(20)))])
def test_prompt_pages_and_lengths(dev, page, cache, q, new, past):
    prompt(dev, Cache(page + len(new), [a + b for a, b in zip(new, past)], 2, 64, page, cache), new, 8, q, q, behind=3,
           seed=page)


@pytest.mark.parametrize("cache,q", [(BF16, BF16), (E4M3, F32), (F16, F16)])
@pytest.mark.parametrize("window", [1, 31, 64, 200, 100000])
@pytest.mark.parametrize("sinks", [None, True])
def test_prompt_windows_and_sinks(dev, cache, q, window, sinks):
    new, past = [1, 300, 90], [700, 33, 0]
    prompt(dev, Cache(window, [a + b for a, b in zip(new, past)], 2, 128, 16, cache), new, 6, q, q, window=window,
           sinks=sinks, seed=window)


@pytest.mark.parametrize("cache,q", [(BF16, BF16), (E4M3, BF16), (F16, F32)])
@pytest.mark.parametrize("head_major", [False, True])
def test_prompt_unmapped_pages_and_slots(dev, cache, q, head_major):
    rows = [200, 33, 64, 500]
    c = Cache(5, rows, 3, 64, 16, cache, head_major=head_major,
              unmapped=[(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (3, 31)])
    prompt(dev, c, [150, 33, 5, 20], 6, q, q, seed=3)
    prompt(dev, c, [20, 33, 7], 6, q, q, seqs=[3, 1, 3], seed=4)


@pytest.mark.parametrize("cache,q", [(BF16, BF16), (E4M3, BF16), (F16, F32)])
@pytest.mark.parametrize("HD,page,window", [(64, 16, 0), (128, 16, 40), (80, 25, 0), (256, 64, 100)])
def test_prompt_infinities_and_nan_stay_with_the_queries_that_see_them(dev, cache, q, HD, page, window):
    """Elements of V that are infinite or NaN, and a row of K that is NaN, at positions in the middle of the prompt:
    queries before them and, with a window, queries far behind them are as if they were not there."""
    n, NH, NKH = 200, 6, 2
    c = Cache(HD, [n], NKH, HD, page, cache)
    nan, inf = float("nan"), float("inf")
    marks = [("v", 3, 0, 5, nan), ("v", 90, 1, 0, nan if cache == E4M3 else inf), ("v", 91, 1, 0, nan if cache == E4M3 else -inf),
             ("v", 150, 0, HD - 1, nan), ("k", 170, 1, 7, nan)]
    for name, s, h, d, x in marks:
        (c.k if name == "k" else c.v)[0][s, h, d] = x
        pool = c.pools[0 if name == "k" else 1]
        at = int(c.tables[0, s // page]), s % page, h, d
        if cache == E4M3:
            pool.view(torch.uint8)[at] = 0x7F
        else:
            pool[at] = x
    query = queries(2, n, NH, HD, q)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    got = dev.paged_attn_prompt(c.view(dev), query.cuda(), i32([0, n]), i32([n]), n, NH, window=window)
    got = got.double().cpu().view(n, NH, HD)
    t = torch.arange(n)
    see = t[None] <= t[:, None]
    if window:
        see &= t[None] > t[:, None] - window
    clean = Cache(HD, [n], NKH, HD, page, cache)
    for name, s, h, d, _ in marks:
        (clean.k if name == "k" else clean.v)[0][s, h, d] = 0.0
    o, mag, za, zq = attend(clean, 0, query.double().view(n, NH, HD), t, HD ** -0.5, window)
    bound = attend_bound(o, mag, za, zq, n, HD, cache, q, q)
    wrong = torch.zeros(n, NH, HD, dtype=torch.bool)
    for name, s, h, d, x in marks:
        heads = slice(h * NH // NKH, (h + 1) * NH // NKH)
        if name == "k":
            wrong[see[:, s], heads] = True
        else:
            wrong[:, heads, d] |= see[:, s, None]
    assert ((got - o).abs() <= bound)[~wrong].all()
    assert not torch.isfinite(got[wrong]).any()
    # one query per sequence: the same rows as the last query's
    last = dev.paged_attn_decode(c.view(dev), query[-1:].cuda(), i32([n]), n, NH, window=window).double().cpu().view(NH, HD)
    assert torch.equal(torch.isfinite(last), ~wrong[-1])
    assert ((last - o[-1]).abs() <= bound[-1])[~wrong[-1]].all()


def test_prompt_more_queries_than_rows(dev):
    """A length below the number of new tokens: the first queries lie before position 0 and give zeros."""
    c = Cache(6, [40], 2, 64, 16, BF16)
    prompt(dev, c, [50], 4, BF16, BF16, seed=1)


@pytest.mark.parametrize("cache,q", [(BF16, BF16), (F16, F32)])
def test_prompt_long(dev, cache, q):
    """Long enough that workgroups take several tiles of queries and the range of rows is cut."""
    prompt(dev, Cache(6, [2100, 4100], 1, 128, 64, cache), [2100, 6], 4, q, q, seed=1)


@pytest.mark.parametrize("cache,q", [(BF16, BF16), (F16, F32), (E4M3, F32)])
@pytest.mark.parametrize("scale,shrink", [(0.0, 1.0), (-0.2, 1.0), (0.125, 1e-30), (0.125, 0.0)])
def test_scales_and_tiny_queries(dev, cache, q, scale, shrink):
    """A scale of zero (the mean of the rows), a negative one, queries next to nothing and of zeros."""
    c = Cache(3, [130, 70], 2, 64, 16, cache)
    prompt(dev, c, [100, 3], 4, q, q, scale=scale, shrink=shrink, window=90, seed=5)
    if shrink == 1.0:
        decode(dev, c, [130, 70], 4, q, q, scale=scale, seed=5)


def test_tables_inside_a_wider_tensor(dev):
    c = Cache(5, [200, 33], 2, 64, 16, BF16)
    wide = torch.full((2, c.tables.shape[1] + 7), 9999, dtype=torch.int32)
    wide[:, 3:3 + c.tables.shape[1]] = c.tables
    t = wide.cuda()[:, 3:3 + c.tables.shape[1]]
    q = queries(4, 2, 8, 64, BF16)
    kv = c.view(dev)
    n = torch.tensor(c.rows, dtype=torch.int32).cuda()
    a = dev.paged_attn_decode(kv, q.cuda(), n, 200, 8)
    b = dev.paged_attn_decode(dev.paged_kv(kv._tensors[0], kv._tensors[1], t), q.cuda(), n, 200, 8)
    assert torch.equal(a, b)


def test_decode_is_the_prompt_of_one_token(dev):
    lens = [65, 300, 1]
    c = Cache(1, lens, 2, 64, 64, F16)
    prompt(dev, c, [1, 1, 1], 8, F32, F32, seed=2)
    decode(dev, c, lens, 8, F32, F32, seed=2)


# ------------------------------------------------------------------ how it is called
def test_repeated_and_captured(dev):
    """The same call twice gives the same bits; a captured pair of calls on one stream, replayed with new lengths and
    eager work between the replays, gives what eager calls give."""
    lens = [700, 65, 1]
    c = Cache(4, [700, 300, 9], 2, 64, 32, BF16)
    kv = c.view(dev)
    q = queries(1, 3, 8, 64, BF16).cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32).cuda()
    ws = dev.paged_attn_workspace(kv, 3, 3, 8, 700)
    out, out2 = torch.empty_like(q), torch.empty_like(q)

    def both():
        dev.paged_attn_decode(kv, q, n, 700, 8, out=out, ws=ws)
        dev.paged_attn_prompt(kv, q, starts, n, 700, 8, out=out2, ws=ws)

    both()
    first = out.clone(), out2.clone()
    both()
    assert torch.equal(out, first[0]) and torch.equal(out2, first[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        both()
    for new in ([700, 65, 1], [2, 300, 9], [699, 0, 5]):
        n.copy_(torch.tensor(new, dtype=torch.int32))
        both()
        want = out.clone(), out2.clone()
        out.zero_(), out2.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(out2, want[1])


def test_wrapper_refusals(dev):
    c = Cache(4, [70], 2, 64, 32, BF16)
    kv = c.view(dev)
    q = queries(1, 1, 8, 64, BF16).cuda()
    n = torch.tensor([70], dtype=torch.int32).cuda()
    for bad in (dict(q=q.cpu()), dict(q=q[:, :-64]), dict(lens=n.long()), dict(lens=n.repeat(2)), dict(NH=7), dict(q=q.half()),
                dict(sinks=torch.zeros(4, device="cuda")), dict(ws=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        a = dict(q=q, lens=n, max_len=70, NH=8) | bad
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            dev.paged_attn_decode(kv, **a)
    with pytest.raises(ValueError):
        dev.paged_kv(kv._tensors[0], kv._tensors[1][:, :16], kv._tensors[2])
    other = c.view(dev)
    other._device = 1                             # as a view made while another GPU was the current one
    with pytest.raises(ValueError):
        dev.paged_attn_decode(other, q, n, 70, 8)
    with pytest.raises(TypeError):
        dev.paged_kv(kv._tensors[0].double(), kv._tensors[1].double(), kv._tensors[2])
