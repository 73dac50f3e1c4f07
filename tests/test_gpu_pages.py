"""Reserving, giving back, forking, compacting and copying pages on the device
against the same steps on Python lists: every table entry, count and byte."""
import random

import pytest
import torch

from mojollama_amd import kernels as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return K.DeviceOps(K.load_kernels())


class Pages:
    """The definition, on lists, beside the state on the GPU; the pools' contents follow page by page."""

    def __init__(self, dev, n_seqs, max_blocks, n_pages, page, shapes=((2, 48), (1, 16)), wide=0):
        self.dev, self.page, self.n_pages, self.max_blocks = dev, page, n_pages, max_blocks
        self.t = [[-1] * max_blocks for _ in range(n_seqs)]
        self.refs = [0] * n_pages
        g = torch.Generator().manual_seed(n_pages)
        self.pools = [torch.randint(0, 255, (layers, n_pages, size), generator=g).to(torch.uint8) for layers, size in shapes]
        self.g_tables = torch.full((n_seqs, max_blocks + wide), -1, dtype=torch.int32, device="cuda")
        self.g_refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        self.g_pools = [p.cuda() for p in self.pools]
        self.map = dev.page_map(self.g_tables[:, :max_blocks], self.g_refs, page)
        self.planes = dev.page_planes(self.g_pools)

    def i32(self, v):
        return torch.tensor(v, dtype=torch.int32).cuda()

    def ok(self, seq, n, done):
        return 0 <= seq < len(self.t) and 0 <= n <= self.max_blocks * self.page and seq not in done

    def reserve(self, seqs, lens):
        missing, done = 0, set()
        free = iter([p for p, r in enumerate(self.refs) if r == 0])
        for s, n in zip(seqs, lens):
            if not self.ok(s, n, done):
                missing += 1
                done.add(s)
                continue
            done.add(s)
            for b in range(-(-n // self.page)):
                if self.t[s][b] < 0:
                    page = next(free, None)
                    if page is None:
                        missing += 1
                        continue
                    self.t[s][b] = page
                    self.refs[page] = 1
        got = self.dev.pages_reserve(self.map, self.i32(seqs), self.i32(lens))
        assert int(got) == missing
        self.same()

    def free(self, seqs, lens=None):
        for i, s in enumerate(seqs):
            n = lens[i] if lens else 0
            if 0 <= s < len(self.t) and n >= 0:
                for b in range(-(-n // self.page), self.max_blocks):
                    if self.t[s][b] >= 0:
                        self.refs[self.t[s][b]] -= 1
                        self.t[s][b] = -1
        self.dev.pages_free(self.map, self.i32(seqs), self.i32(lens) if lens else None)
        self.same()

    def fork(self, parents, children, lens):
        missing, done = 0, set()
        was = [list(r) for r in self.t]
        free = [p for p, r in enumerate(self.refs) if r == 0]
        gone = []
        for p, c, n in zip(parents, children, lens):
            if not self.ok(c, n, done) or not 0 <= p < len(self.t):
                missing += 1
                done.add(c)
                continue
            done.add(c)
            if p == c:
                continue
            row = [-1] * self.max_blocks
            for b in range(n // self.page):
                row[b] = was[p][b]
                if row[b] >= 0:
                    self.refs[row[b]] += 1
            last = n // self.page
            if n % self.page and was[p][last] >= 0:
                if free:
                    row[last] = free.pop(0)
                    self.refs[row[last]] = 1
                    for x in self.pools:
                        x[:, row[last]] = x[:, was[p][last]]
                else:
                    missing += 1
            gone += [x for x in was[c] if x >= 0]
            self.t[c] = row
        for x in gone:
            self.refs[x] -= 1
        got = self.dev.pages_fork(self.map, self.planes, self.i32(parents), self.i32(children), self.i32(lens))
        assert int(got) == missing
        self.same()

    def compact(self):
        L = sum(r > 0 for r in self.refs)
        moves = dict(zip([p for p in range(L, self.n_pages) if self.refs[p]], [p for p in range(L) if not self.refs[p]]))
        for a, b in moves.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            for x in self.pools:
                x[:, b] = x[:, a]
        self.t = [[moves.get(p, p) for p in r] for r in self.t]
        assert int(self.dev.pages_compact(self.map, self.planes)) == L
        self.same()

    def same(self):
        assert self.g_tables[:, :self.max_blocks].tolist() == self.t
        assert (self.g_tables[:, self.max_blocks:] == -1).all()
        assert self.g_refs.tolist() == self.refs
        for a, b in zip(self.g_pools, self.pools):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("seed,shapes", [(0, ((2, 48), (1, 16))), (1, ((3, 17),)), (2, ((2, 40000), (2, 5))), (3, ())])
def test_a_pool_in_use(dev, seed, shapes):
    """Random requests: sequences grow, are cut, forked into others (some of them parents too), end, and the pool is
    compacted; now and then the pool runs out."""
    r = random.Random(seed)
    n_seqs, max_blocks, page = 7, 9, 4
    p = Pages(dev, n_seqs, max_blocks, 33, page, shapes, wide=seed)
    for _ in range(25):
        k = r.randint(1, n_seqs)
        what = r.choice(["reserve", "reserve", "free", "fork", "fork", "compact"])
        seqs = r.sample(range(n_seqs), k)
        lens = [r.randint(0, max_blocks * page) for _ in seqs]
        if what == "reserve":
            p.reserve(seqs, lens)
        elif what == "free":
            p.free(seqs[:2], None if r.random() < 0.5 else lens[:2])
        elif what == "fork":
            p.fork([r.randrange(n_seqs) for _ in seqs], seqs, lens)
        else:
            p.compact()


def test_requests_left_out(dev):
    p = Pages(dev, 4, 5, 20, 8)
    p.reserve([0, 9, 1, 0, -1, 2], [17, 8, 41, 40, 3, -1])
    p.fork([0, 0, 5, 0, 1, 0], [1, 1, 2, -3, 4, 3], [17, 9, 3, 4, 4, 41])
    p.free([0, 0, 7, -2, 1], [8, 0, 0, 0, -1])


@pytest.mark.parametrize("n_seqs,max_blocks,n_pages", [(1, 1, 1), (300, 40, 9000), (1500, 3, 5000), (3, 600, 1500)])
def test_large_pools(dev, n_seqs, max_blocks, n_pages):
    """More requests than a workgroup has threads, more blocks than a wave has lanes, more pages than one scan takes."""
    r = random.Random(n_seqs)
    p = Pages(dev, n_seqs, max_blocks, n_pages, 16, ((1, 32),))
    every = list(range(n_seqs))
    r.shuffle(every)
    p.reserve(every, [r.randint(0, max_blocks * 16) for _ in every])
    p.free(every[::3])
    p.compact()
    p.reserve(every[::3], [r.randint(0, max_blocks * 16) for _ in every[::3]])
    p.fork([r.choice(every) for _ in every[::2]], every[::2], [r.randint(0, max_blocks * 16) for _ in every[::2]])
    p.compact()


def test_copy(dev):
    for size, shift in ((64, 0), (40004, 0), (16400, 4)):
        base = torch.randint(0, 255, (2 * 12 * size + 16,), dtype=torch.uint8, device="cuda")
        pool = base[shift:shift + 2 * 12 * size].view(2, 12, size)
        want = pool.clone()
        src, dst = [0, 5, 0, 11, 3, 12], [2, 6, 7, -1, 1, 4]
        for a, b in zip(src, dst):
            if 0 <= a < 12 and 0 <= b < 12:
                want[:, b] = want[:, a]
        dev.pages_copy(dev.page_planes([pool]), 12, torch.tensor(src, dtype=torch.int32).cuda(),
                       torch.tensor(dst, dtype=torch.int32).cuda())
        assert torch.equal(pool, want)


def test_wrapper_refusals(dev):
    p = Pages(dev, 4, 5, 20, 8)
    one = p.i32([0])
    with pytest.raises(ValueError):
        dev.pages_reserve(p.map, one, p.i32([1, 2]))
    with pytest.raises(ValueError):
        dev.pages_fork(p.map, p.planes, one, one.long(), one)
    with pytest.raises(RuntimeError):
        dev.pages_reserve(p.map, one, one, ws=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        dev.pages_compact(p.map, dev.page_planes([torch.zeros(1, 19, 4, device="cuda")]))
    with pytest.raises(ValueError):
        dev.page_planes([torch.zeros(2, 20, 8, device="cuda")[:, :, ::2]])
    p.same()
