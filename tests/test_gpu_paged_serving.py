"""The operators over a paged cache as a server uses them together: pages
reserved, prompts turned, stored and attended, beams forked and decoded, ended
sequences given back and the pool compacted -- eagerly and as a captured step."""
import pytest
import torch

from mojollama_amd import kernels as K
from paged_ref import BF16, E4M3, F16, F32, attend_bound

pytestmark = pytest.mark.gpu
NH, NKH, HD, PAGE, BLOCKS, PAGES, LAYERS = 8, 2, 64, 16, 9, 40, 2


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return K.DeviceOps(K.load_kernels())


def i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


class Server:
    """Four slots, two layers; the same tokens' q, k, v for every layer, scaled."""

    def __init__(self, dev, dtype, act):
        self.dev, self.dtype, self.act = dev, dtype, act
        self.tables = torch.full((4, BLOCKS), -1, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(PAGES, dtype=torch.int32, device="cuda")
        self.map = dev.page_map(self.tables, self.refs, PAGE)
        nan = 0x7F if dtype == E4M3 else 0xFF
        size = 1 if dtype == E4M3 else 2
        raw = [torch.full((LAYERS, PAGES, PAGE, NKH, HD * size), nan, dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.pools = [r.view(dtype) for r in raw]
        self.exps = [torch.full((LAYERS, PAGES, NKH, PAGE), 255, dtype=torch.uint8, device="cuda") for _ in range(2)
                     ] if dtype == E4M3 else []
        self.planes = dev.page_planes(self.pools + self.exps)
        self.kv = [dev.paged_kv(*(p[i] for p in self.pools), self.tables, *(e[i] for e in self.exps)) for i in range(LAYERS)]
        self.rot = dev.rotary(HD, base=10000.0, scaling=K.ROPE_YARN, factor=4.0, ctx=64.0)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.ws = dev.pages_workspace(self.map, 4)

    def reserve(self, seqs, lens):
        self.dev.pages_reserve(self.map, seqs, lens, status=self.status, ws=self.ws)

    def append(self, layer, qkv, pos, seqs):
        a, b = NH * HD, NKH * HD
        q = torch.empty(len(qkv), a, dtype=self.act, device="cuda")
        self.dev.rotary_append(self.rot, qkv[:, :a], qkv[:, a:a + b], qkv[:, a + b:], pos, NH=NH, kv=self.kv[layer],
                               seqs=seqs, q_out=q)
        return q

    def rows(self, layer, seq, n):
        """What sequence seq's first n rows hold, in 64 bits."""
        t, s = self.tables[seq].cpu().long(), torch.arange(n)
        out = []
        for i, p in enumerate(self.pools):
            raw = p[layer].view(torch.uint8).cpu().view(self.dtype)
            x = raw.view(torch.uint8)[t[s // PAGE], s % PAGE].view(self.dtype).double()
            if self.exps:
                e = self.exps[i][layer].cpu()
                x = x * (2.0 ** (e[t[s // PAGE], :, s % PAGE].double() - 127))[..., None]
            out.append(x)
        return out

    def check(self, layer, seq, n, q, out):
        """Queries q [m] of the last m of n rows."""
        k, v = (x.repeat_interleave(NH // NKH, 1) for x in self.rows(layer, seq, n))
        q, out = (x.double().cpu().view(-1, NH, HD) for x in (q, out))
        m, scale = len(q), HD ** -0.5
        w = torch.einsum("nhd,shd->nhs", q, k) * scale
        w = w.masked_fill((torch.arange(n)[None] > torch.arange(m)[:, None] + n - m)[:, None], -float("inf"))
        w = torch.softmax(w, -1)
        o, mag = torch.einsum("nhs,shd->nhd", w, v), torch.einsum("nhs,shd->nhd", w, v.abs())
        za = float((torch.einsum("nhd,shd->nhs", q.abs(), k.abs()) * scale).max())
        zq = float((q.abs().amax(-1)[..., None] * k.abs().sum(-1).T[None] * scale).max())
        assert ((out - o).abs() <= attend_bound(o, mag, za, zq, n, HD, self.dtype, self.act, self.act)).all()


@pytest.mark.parametrize("dtype,act", [(BF16, BF16), (F16, F32), (E4M3, BF16), (E4M3, F32)])
def test_prompts_beams_and_compaction(dev, dtype, act):
    s = Server(dev, dtype, act)
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = lambda n: torch.randn(n, (NH + 2 * NKH) * HD, device="cuda", generator=g)  # noqa: E731
    # two prompts, 37 and 50 tokens, the second in two parts
    s.reserve(i32([0, 1]), i32([37, 30]))
    assert int(s.status) == 0
    x = tokens(67)
    pos, seqs = i32(list(range(37)) + list(range(30))), i32([0] * 37 + [1] * 30)
    for layer in range(LAYERS):
        q = s.append(layer, x * (1 + layer), pos, seqs)
        out = dev.paged_attn_prompt(s.kv[layer], q, i32([0, 37, 67]), i32([37, 30]), 37, NH, seqs=i32([0, 1]))
        s.check(layer, 0, 37, q[:37], out[:37])
        s.check(layer, 1, 30, q[37:], out[37:])
    s.reserve(i32([1]), i32([50]))
    x = tokens(20)
    for layer in range(LAYERS):
        q = s.append(layer, x, i32(list(range(30, 50))), i32([1] * 20))
        out = dev.paged_attn_prompt(s.kv[layer], q, i32([0, 20]), i32([50]), 50, NH, seqs=i32([1]))
        s.check(layer, 1, 50, q, out)
    # slots 2 and 3 go on from slot 0, each with a token of its own
    dev.pages_fork(s.map, s.planes, i32([0, 0]), i32([2, 3]), i32([37, 37]), status=s.status, ws=s.ws)
    assert int(s.status) == 0
    before = [s.rows(layer, 0, 37) for layer in range(LAYERS)]
    s.reserve(i32([0, 2, 3]), i32([38, 38, 38]))
    x = tokens(3)
    kept = []
    for layer in range(LAYERS):
        q = s.append(layer, x, i32([37, 37, 37]), i32([0, 2, 3]))
        out = dev.paged_attn_decode(s.kv[layer], q, i32([38, 38, 38]), 38, NH, seqs=i32([0, 2, 3]))
        for i, seq in enumerate([0, 2, 3]):
            s.check(layer, seq, 38, q[i:i + 1], out[i:i + 1])
            for a, b in zip(s.rows(layer, seq, 37), before[layer]):
                assert torch.equal(a, b)
        kept.append((q, out))
    # the second prompt ends, the rest moves to the front: the same answers, bit for bit
    dev.pages_free(s.map, i32([1]))
    live = int(dev.pages_compact(s.map, s.planes, status=s.status, ws=s.ws))
    assert live == int((s.refs > 0).sum()) and int((s.refs[live:] != 0).sum()) == 0
    for layer, (q, out) in enumerate(kept):
        again = dev.paged_attn_decode(s.kv[layer], q, i32([38, 38, 38]), 38, NH, seqs=i32([0, 2, 3]))
        assert torch.equal(again, out)


def test_captured_decode_steps(dev):
    """Reserve, append and decode of a step captured once and replayed with new tokens and lengths, against the same
    steps run eagerly on a second server, with eager work between the replays."""
    one, two = Server(dev, BF16, BF16), Server(dev, BF16, BF16)
    g = torch.Generator(device="cuda").manual_seed(2)
    seqs, lens, pos = i32([0, 2, 3]), i32([1, 1, 1]), i32([0, 0, 0])
    x = torch.randn(3, (NH + 2 * NKH) * HD, device="cuda", generator=g)
    ws = dev.paged_attn_workspace(one.kv[0], 3, 3, NH, BLOCKS * PAGE)
    q, out = torch.empty(3, NH * HD, dtype=BF16, device="cuda"), torch.empty(3, NH * HD, dtype=BF16, device="cuda")

    def step(s, q, out, ws):
        a, b = NH * HD, NKH * HD
        s.reserve(seqs, lens)
        dev.rotary_append(s.rot, x[:, :a], x[:, a:a + b], x[:, a + b:], pos, NH=NH, kv=s.kv[0], seqs=seqs, q_out=q)
        dev.paged_attn_decode(s.kv[0], q, lens, BLOCKS * PAGE, NH, seqs=seqs, out=out, ws=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(one, q, out, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(one, q, out, ws)
    q2, out2, ws2 = torch.empty_like(q), torch.empty_like(out), torch.empty_like(ws)
    for n in list(range(1, 40)) + [100, 144]:
        # at the jumps the rows between hold other tokens' k and v: the same in both
        for s in (one, two):
            s.reserve(seqs, i32([n, n, n]))
            if n > 40:
                for p in s.pools:
                    p.copy_(torch.nan_to_num(p, nan=0.5))
        x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        lens.fill_(n)
        pos.fill_(n - 1)
        torch.cuda.synchronize()
        graph.replay()
        step(two, q2, out2, ws2)
        torch.cuda.synchronize()
        assert torch.equal(out, out2) and torch.isfinite(out).all(), n
        assert torch.equal(one.tables, two.tables) and torch.equal(one.refs, two.refs)


def test_calls_on_two_streams(dev):
    """Two decode calls at once on two streams, with a workspace each."""
    s = Server(dev, BF16, BF16)
    s.reserve(i32([0, 1, 2, 3]), i32([144, 144, 100, 1]))
    for p in s.pools:
        p.copy_(torch.randn(p.shape, device="cuda").to(BF16))
    q = torch.randn(4, NH * HD, device="cuda").to(BF16)
    lens = i32([144, 130, 100, 1])
    want = dev.paged_attn_decode(s.kv[0], q, lens, 144, NH), dev.paged_attn_decode(s.kv[1], q, lens, 144, NH)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(q) for _ in range(2)]
    wss = [dev.paged_attn_workspace(s.kv[0], 4, 4, NH, 144) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                dev.paged_attn_decode(s.kv[i], q, lens, 144, NH, out=outs[i], ws=wss[i])
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
