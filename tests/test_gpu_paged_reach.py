"""Attention over a paged cache at the sizes where other kernels, splits and
joins take over: prompts in tiles of 256 rows, splits of prompts and decode with
windows and sinks, more splits than the join loads at once, 16 and more query
heads above head size 128, unmapped pages at every page size's kernel, split
calls captured and on two streams; and at the ends of its range: windows up to
2^31 - 1, infinities of V, a single row."""
import pytest
import torch

from mojollama_amd import kernels as K
from paged_ref import BF16, E4M3, F16, F32, Cache, attend, attend_bound

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return K.DeviceOps(K.load_kernels())


def i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def queries(seed, n, NH, HD, dtype):
    return (1.5 * torch.randn(n, NH * HD, generator=torch.Generator().manual_seed(seed))).to(dtype)


def some_sinks(NH, on):
    return 3 * torch.randn(NH, generator=torch.Generator().manual_seed(NH)) if on else None


def check(got, c, b, q, pos, NH, window, sinks, out, wrong=None):
    """Rows of one sequence; `wrong` marks the elements that see an infinity or a NaN."""
    HD = c.HD
    o, mag, za, zq = attend(c, b, q.double().view(len(q), NH, HD), pos, HD ** -0.5, window, sinks)
    got = got.double().cpu().view(o.shape)
    bound = attend_bound(o, mag, za, zq, c.rows[b], HD, c.dtype, q.dtype, out)
    ok = (got - o).abs() <= bound
    if wrong is not None:
        assert not torch.isfinite(got[wrong]).any()
        ok |= wrong
    assert ok.all(), (b, int((~ok).sum()), pos[(~ok).flatten(1).any(1)].tolist()[:9])


class Watched:
    """A workspace, and whether a call has written to it: only splits do."""

    def __init__(self, dev, kv, T, B, NH, max_len, window):
        self.ws = dev.paged_attn_workspace(kv, T, B, NH, max_len, window)
        self.ws.fill_(0xA5)

    def split(self):
        return bool((self.ws != 0xA5).any())


# ------------------------------------------------------------------ prompts in tiles of 256 rows
TILES = [(BF16, 64), (BF16, 80), (BF16, 128), (F16, 64), (F16, 128), (E4M3, 128), (E4M3, 64)]


@pytest.mark.parametrize("cache,HD", TILES)
@pytest.mark.parametrize("window,sinks", [(0, False), (300, True)])
def test_prompt_in_tiles_of_256_rows(dev, cache, HD, window, sinks):
    """tokens * heads of 65536 and more on pages of 64 rows: one long sequence and two short ones, a page of the first
    and one of the second unmapped, infinities and NaN in V and a NaN in K in the middle of the prompt."""
    NH, NKH, act = 32, 8, F16 if cache == F16 else BF16
    new, past = [2100, 70, 1], [0, 500, 64]
    rows, hole = [a + b for a, b in zip(new, past)], [(0, 11), (1, 3)]
    c, clean = (Cache(HD, rows, NKH, HD, 64, cache, unmapped=hole) for _ in range(2))
    e4m3 = cache == E4M3
    marks = [("v", 3, 0, 5, NAN), ("v", 900, 1, 0, NAN if e4m3 else INF), ("v", 901, 1, 0, NAN if e4m3 else -INF),
             ("v", 1500, 7, HD - 1, NAN), ("k", 1700, 2, 7, NAN)]
    for name, s, h, d, x in marks:
        pool = c.pools[0 if name == "k" else 1]
        at = int(c.tables[0, s // 64]), s % 64, h, d
        if e4m3:
            pool.view(torch.uint8)[at] = 0x7F
        else:
            pool[at] = x
        (clean.k if name == "k" else clean.v)[0][s, h, d] = 0.0
    T = sum(new)
    q, sk = queries(HD, T, NH, HD, act), some_sinks(NH, sinks)
    out = torch.full((T + 2, NH * HD), 7.0, dtype=act, device="cuda")
    qq = torch.cat([q, q[:2]]).cuda()
    starts = [0, new[0], new[0] + new[1], T]
    dev.paged_attn_prompt(c.view(dev), qq, i32(starts), i32(rows), max(rows), NH, window=window,
                          sinks=None if sk is None else sk.cuda(), out=out)
    assert (out[T:] == 7).all()
    # a tile of 256 rows is 64 tokens here
    at = torch.tensor([0, 1, 2, 3, 4, 63, 64, 65, 302, 303, 304, 703, 704, 705, 767, 768, 899, 900, 901, 902, 1003, 1004,
                       1199, 1200, 1201, 1499, 1500, 1501, 1699, 1700, 1701, 1800, 1801, 1999, 2000, 2047, 2048, 2098, 2099])
    s = torch.arange(rows[0])
    see = s[None] <= at[:, None]
    if window:
        see &= s[None] > at[:, None] - window
    wrong = torch.zeros(len(at), NH, HD, dtype=torch.bool)
    for name, row, h, d, _ in marks:
        heads = slice(4 * h, 4 * h + 4)
        if name == "k":
            wrong[see[:, row], heads] = True
        else:
            wrong[:, heads, d] |= see[:, row, None]
    check(out[at.cuda()], clean, 0, q[at], at, NH, window, sk, act, wrong)
    for b in (1, 2):
        check(out[starts[b]:starts[b + 1]], clean, b, q[starts[b]:starts[b + 1]], torch.arange(new[b]) + past[b], NH, window,
              sk, act)


# ------------------------------------------------------------------ splits
SPLIT = [(BF16, BF16), (F16, F32), (E4M3, BF16), (E4M3, F32)]


@pytest.mark.parametrize("cache,q", SPLIT)
@pytest.mark.parametrize("HD,page", [(64, 16), (128, 64), (128, 25), (256, 64)])
@pytest.mark.parametrize("window,sinks", [(0, False), (0, True), (1000, True), (1000, False)])
def test_prompt_splits(dev, cache, q, HD, page, window, sinks):
    """A few new tokens over thousands of rows."""
    NH, NKH, new = 8, 2, [6, 2, 0]
    rows = [4100, 700, 0]
    c = Cache(HD + page, rows, NKH, HD, page, cache, unmapped=[(0, 2000 // page), (0, 4050 // page)])
    x, sk = queries(HD, 8, NH, HD, q), some_sinks(NH, sinks)
    kv = c.view(dev)
    w = Watched(dev, kv, 8, 3, NH, 4100, window)
    out = dev.paged_attn_prompt(kv, x.cuda(), i32([0, 6, 8, 8]), i32(rows), 4100, NH, window=window,
                                sinks=None if sk is None else sk.cuda(), ws=w.ws)
    assert w.split()
    check(out[:6], c, 0, x[:6], torch.arange(4094, 4100), NH, window, sk, q)
    check(out[6:], c, 1, x[6:], torch.arange(698, 700), NH, window, sk, q)


@pytest.mark.parametrize("cache,q", SPLIT)
@pytest.mark.parametrize("HD,page", [(64, 16), (128, 64), (128, 25), (256, 64)])
@pytest.mark.parametrize("window,sinks", [(0, True), (1000, False), (1000, True), (2990, False)])
def test_decode_splits(dev, cache, q, HD, page, window, sinks):
    NH, NKH, rows = 8, 2, [3000, 0, 1001, 1, 2600]
    c = Cache(HD + page, rows, NKH, HD, page, cache, unmapped=[(0, 2500 // page), (4, 1700 // page)])
    x, sk = queries(HD, 5, NH, HD, q), some_sinks(NH, sinks)
    kv = c.view(dev)
    w = Watched(dev, kv, 5, 5, NH, 3000, window)
    out = dev.paged_attn_decode(kv, x.cuda(), i32(rows), 3000, NH, window=window, sinks=None if sk is None else sk.cuda(),
                                ws=w.ws)
    assert w.split()
    for b, n in enumerate(rows):
        check(out[b:b + 1], c, b, x[b:b + 1], torch.tensor([n - 1]), NH, window, sk, q)


@pytest.mark.parametrize("cache,q", [(BF16, BF16), (E4M3, F32)])
def test_decode_of_more_than_64_splits(dev, cache, q):
    """One kv head of one long sequence: 256 splits, beside a sequence that leaves most of them empty."""
    NH, rows = 4, [70000, 300]
    c = Cache(7, rows, 1, 64, 64, cache)
    x = queries(7, 2, NH, 64, q)
    kv = c.view(dev)
    w = Watched(dev, kv, 2, 2, NH, 70000, 0)
    out = dev.paged_attn_decode(kv, x.cuda(), i32(rows), 70000, NH, ws=w.ws)
    assert w.split()
    for b, n in enumerate(rows):
        check(out[b:b + 1], c, b, x[b:b + 1], torch.tensor([n - 1]), NH, 0, None, q)


# ------------------------------------------------------------------ many query heads a kv head
@pytest.mark.parametrize("cache,q", [(BF16, BF16), (F16, F16), (E4M3, BF16), (BF16, F32), (F16, F32), (E4M3, F32)])
@pytest.mark.parametrize("NH,NKH,HD", [(16, 1, 256), (20, 1, 256), (32, 2, 144), (64, 2, 128)])
def test_sixteen_and_more_heads_share_a_kv_head(dev, cache, q, NH, NKH, HD):
    rows = [1, 40, 900]
    c = Cache(NH + HD, rows, NKH, HD, 32, cache)
    x, kv = queries(HD, 3, NH, HD, q), c.view(dev)
    out = dev.paged_attn_decode(kv, x.cuda(), i32(rows), 900, NH)
    for b, n in enumerate(rows):
        check(out[b:b + 1], c, b, x[b:b + 1], torch.tensor([n - 1]), NH, 0, None, q)
    out = dev.paged_attn_decode(kv, x[:2].cuda(), i32(rows[:2]), 40, NH)          # whole, without a join
    for b, n in enumerate(rows[:2]):
        check(out[b:b + 1], c, b, x[b:b + 1], torch.tensor([n - 1]), NH, 0, None, q)


# ------------------------------------------------------------------ pages
@pytest.mark.parametrize("page", [16, 25, 48, 64, 128])
@pytest.mark.parametrize("cache,q", [(BF16, BF16), (E4M3, BF16), (F16, F32)])
@pytest.mark.parametrize("window", [0, 150])
def test_unmapped_pages_of_every_size(dev, page, cache, q, window):
    """The first, one in the middle and the last page of a sequence, and every page of another, are on no page."""
    NH, NKH, HD, rows = 6, 3, 64, [500, 120, 130]
    last = lambda n: (n - 1) // page  # noqa: E731
    holes = [(0, 0), (0, last(300)), (0, last(500))] + [(1, b) for b in range(last(120) + 1)]
    c = Cache(page, rows, NKH, HD, page, cache, unmapped=holes)
    kv, new = c.view(dev), [150, 120, 9]
    x = queries(page, sum(new), NH, HD, q)
    out = dev.paged_attn_prompt(kv, x.cuda(), i32([0, 150, 270, 279]), i32(rows), 500, NH, window=window)
    at = 0
    for b, n in enumerate(new):
        check(out[at:at + n], c, b, x[at:at + n], torch.arange(rows[b] - n, rows[b]), NH, window, None, q)
        at += n
    assert not out[150:270].any()
    out = dev.paged_attn_decode(kv, x[:3].cuda(), i32(rows), 500, NH, window=window)
    for b, n in enumerate(rows):
        check(out[b:b + 1], c, b, x[b:b + 1], torch.tensor([n - 1]), NH, window, None, q)


# ------------------------------------------------------------------ windows
@pytest.mark.parametrize("window", [40, 41, (1 << 30) + 1, (1 << 31) - 50, (1 << 31) - 1])
@pytest.mark.parametrize("cache,q", [(BF16, BF16), (F16, F32)])
def test_windows_without_an_end(dev, window, cache, q):
    """A window at or past the longest length is none, also where the first queries lie before position 0."""
    c = Cache(6, [40, 33], 2, 64, 16, cache)
    x, kv = queries(1, 83, 4, 64, q), c.view(dev)
    got = dev.paged_attn_prompt(kv, x.cuda(), i32([0, 50, 83]), i32([40, 33]), 40, 4, window=window)
    check(got[:50], c, 0, x[:50], torch.arange(-10, 40), 4, 0, None, q)
    check(got[50:], c, 1, x[50:], torch.arange(33), 4, 0, None, q)
    assert torch.equal(got, dev.paged_attn_prompt(kv, x.cuda(), i32([0, 50, 83]), i32([40, 33]), 40, 4))
    got = dev.paged_attn_decode(kv, x[:2].cuda(), i32([40, 33]), 40, 4, window=window)
    assert torch.equal(got, dev.paged_attn_decode(kv, x[:2].cuda(), i32([40, 33]), 40, 4))

# ------------------------------------------------------------------ infinities in V
@pytest.mark.parametrize("cache,q", [(BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("HD,page", [(64, 16), (128, 64), (80, 25), (256, 64)])
def test_infinities_of_one_sign_stay_infinite(dev, cache, q, HD, page):
    """An infinity of V in a row that a query sees makes that column infinite, not NaN: in a row of its own (weight 1), in
    rows that all queries of a tile see, and in steps where some do not; a column of both signs is NaN."""
    n, NH, NKH = 300, 4, 2
    c = Cache(HD, [n, 1], NKH, HD, page, cache)
    marks = [(0, 0, 0, 3, INF), (0, 40, 0, 7, -INF), (0, 250, 1, 1, INF), (0, 60, 1, 9, INF), (0, 61, 1, 9, -INF),
             (1, 0, 0, 2, -INF)]
    for b, s, h, d, x in marks:
        c.pools[1][int(c.tables[b, s // page]), s % page, h, d] = x
    kv, x = c.view(dev), queries(HD, n + 1, NH, HD, q) / 4                # no weight is so small that fp16 holds none of it
    got = dev.paged_attn_prompt(kv, x.cuda(), i32([0, n, n + 1]), i32([n, 1]), n, NH).float().cpu().view(n + 1, NH, HD)
    last = dev.paged_attn_decode(kv, x[n - 1:].cuda(), i32([n, 1]), n, NH).float().cpu().view(2, NH, HD)
    want = torch.zeros(n + 1, NH, HD)
    want[0:n, 0:2, 3], want[40:n, 0:2, 7], want[250:n, 2:, 1], want[60:n, 2:, 9] = INF, -INF, INF, INF
    want[61:n, 2:, 9], want[n, 0:2, 2] = NAN, -INF
    for y, w in ((got, want), (last, want[n - 1:])):
        assert torch.equal(torch.isnan(y), torch.isnan(w))
        assert torch.equal(torch.where(torch.isinf(y), y, 0), torch.where(torch.isinf(w), w, 0))


@pytest.mark.parametrize("cache,q", SPLIT + [(F16, F16), (BF16, F32)])
@pytest.mark.parametrize("HD", [64, 128, 256])
def test_a_row_of_all_the_weight_is_given_back(dev, cache, q, HD):
    """A query that sees one row: V's row, by a whole call and by a split one whose window leaves that row.  The weight
    w itself cancels between the sum and the product.  Its planes hold it to 2^-22 (fp16: 11 bits cut and 11 rounded;
    bf16's three to 2^-23), the product's two or three sums, the sum's factor, its reciprocal and the last product round
    once each in fp32: 6 * 2^-24 more, together below 2^-21.  bf16's two planes hold it to 2^-15.  A 16-bit output,
    which holds the row, is nearer to it than to its neighbours, 2^-9 or 2^-12 away, and exact."""
    rows, NKH, NH = [1, 2000], 2, 4
    c = Cache(HD, rows, NKH, HD, 16, cache)
    kv, x, v = c.view(dev), queries(HD, 3, NH, HD, q), torch.stack([c.v[0][0], c.v[1][1999]]).repeat_interleave(2, 1)
    tol = 2.0 ** -21 if q == F32 else 0.0
    calls = (dev.paged_attn_decode(kv, x[:2].cuda(), i32(rows), 2000, NH, window=1),
             dev.paged_attn_prompt(kv, x[:2].cuda(), i32([0, 1, 2]), i32(rows), 2000, NH, window=1),
             dev.paged_attn_decode(kv, x[:1].cuda(), i32([1]), 2000, NH))
    for out in calls:
        y = out.cpu().double().view(-1, NH, HD)
        assert ((y - v[:len(y)]).abs() <= tol * v[:len(y)].abs()).all()


# ------------------------------------------------------------------ how split calls are made
@pytest.fixture(scope="module")
def long(dev):
    c = Cache(4, [2000, 1300, 9], 2, 64, 32, BF16)
    return c, c.view(dev)


def test_split_calls_on_two_streams(dev, long):
    """Decode and a prompt of a few tokens, both split and joined, at once on two streams with a workspace each and
    different queries: what each gives alone."""
    c, kv = long
    lens, starts = i32(c.rows), i32([0, 4, 8, 9])
    qd = [queries(s, 3, 8, 64, BF16).cuda() for s in (1, 2)]
    qp = [queries(s, 9, 8, 64, BF16).cuda() for s in (3, 4)]

    def calls(i, ws):
        return (dev.paged_attn_decode(kv, qd[i], lens, 2000, 8, ws=ws),
                dev.paged_attn_prompt(kv, qp[i], starts, lens, 2000, 8, ws=ws))

    want = []
    for i in range(2):
        w = Watched(dev, kv, 9, 3, 8, 2000, 0)
        want.append(calls(i, w.ws))
        assert w.split()
    assert not torch.equal(want[0][0], want[1][0])
    streams, wss = [torch.cuda.Stream() for _ in range(2)], [Watched(dev, kv, 9, 3, 8, 2000, 0).ws for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(calls(i, wss[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in outs[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])


def test_split_calls_captured(dev, long):
    """Captured once at the longest lengths, replayed with others and with eager work between: two graphs that share a
    workspace on one stream."""
    c, kv = long
    lens, starts = i32(c.rows), i32([0, 4, 8, 9])
    qd, qp = queries(1, 3, 8, 64, BF16).cuda(), queries(2, 9, 8, 64, BF16).cuda()
    w = Watched(dev, kv, 9, 3, 8, 2000, 0)
    od, op = torch.empty_like(qd), torch.empty_like(qp)
    decode = lambda o, ws: dev.paged_attn_decode(kv, qd, lens, 2000, 8, out=o, ws=ws)  # noqa: E731
    prompt = lambda o, ws: dev.paged_attn_prompt(kv, qp, starts, lens, 2000, 8, out=o, ws=ws)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode(od, w.ws), prompt(op, w.ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert w.split()
    graphs = []
    for f, o in ((decode, od), (prompt, op)):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            f(o, w.ws)
    own = torch.empty_like(w.ws)
    for new in ([2000, 1300, 9], [4, 1000, 1], [1999, 0, 9], [700, 641, 8], [2000, 1300, 9]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        ed, ep = decode(torch.empty_like(qd), own), prompt(torch.empty_like(qp), own)
        od.zero_(), op.zero_()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(od, ed) and torch.equal(op, ep), new
        for b in range(3):
            check(ed[b:b + 1], c, b, qd[b:b + 1].cpu(), torch.tensor([new[b] - 1]), 8, 0, None, BF16)
