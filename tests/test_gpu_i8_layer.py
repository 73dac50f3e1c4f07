"""Layers in 8-bit integers as a model runs them: norm, q/k/v product, rotary positions and attention over a paged
cache, quantised, output product, norm with the residual, gate and up product, silu, down product -- eagerly, captured
and replayed, and on two streams at once."""
import pytest
import torch

from mojollama_amd import kernels as K

pytestmark = pytest.mark.gpu
N, NH, NKH, HD, FF, EPS = 512, 8, 2, 64, 700, 1e-6
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    return K.DeviceOps()


class Layer:
    """Weights of one layer, and buffers for up to T tokens of B sequences."""

    def __init__(self, dev, seed, T, B):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
        self.dev, self.B = dev, B
        self.n1, self.n2 = (1 + 0.2 * r(N)).cuda(), (1 + 0.2 * r(N)).to(BF16).cuda()
        wide = (NH + 2 * NKH) * HD
        self.w = dict(qkv=dev.i8_weights((r(wide, N) * N ** -0.5).cuda()), o=dev.i8_weights((r(N, NH * HD) * N ** -0.5).to(BF16).cuda()),
                      gu=dev.i8_weights((r(2 * FF, N) * N ** -0.5).half().cuda()),
                      down=dev.i8_weights((r(N, FF) * FF ** -0.5).cuda()))
        self.bias = (0.1 * r(wide)).cuda()
        pool = lambda: torch.zeros((32, 16, NKH, HD), dtype=BF16, device="cuda")  # noqa: E731
        self.tables = torch.arange(8 * B, dtype=torch.int32, device="cuda").view(B, 8)
        self.kv = dev.paged_kv(pool(), pool(), self.tables)
        self.rot = dev.rotary(HD)
        self.ws = {k: dev.i8_gemm_workspace(w, T) for k, w in self.w.items()}

    def run(self, h, y, pos, seqs, starts, lens, max_len):
        """One pass over new tokens: h float32 [T, N] the residual stream (advanced in place), y the last layer's output."""
        d, steps = self.dev, {}
        q, s = d.i8_rms_norm(y, self.n1, EPS, res=h)
        steps["norm"] = (q, s, h.clone())
        qkv = d.i8_gemm(self.w["qkv"], q, s, bias=self.bias, ws=self.ws["qkv"])
        steps["qkv"] = (q, s, qkv)
        a, b = NH * HD, (NH + NKH) * HD
        q16 = torch.empty((len(h), a), dtype=BF16, device="cuda")
        d.rotary_append(self.rot, qkv[:, :a], qkv[:, a:b], qkv[:, b:], pos, NH=NH, kv=self.kv, seqs=seqs, q_out=q16)
        att = d.paged_attn_prompt(self.kv, q16, starts, lens, max_len, NH, out_dtype=BF16)
        q, s = d.i8_quantize(att)
        steps["attention"] = (att, q, s)
        o = d.i8_gemm(self.w["o"], q, s, ws=self.ws["o"])
        q, s = d.i8_rms_norm(o, self.n2, EPS, res=h)
        steps["norm2"] = (q, s, o, h.clone())
        gu = d.i8_gemm(self.w["gu"], q, s, out_dtype=torch.float16, ws=self.ws["gu"])
        q, s = d.i8_silu_mul(gu[:, :FF], gu[:, FF:])
        steps["silu"] = (gu, q, s)
        out = d.i8_gemm(self.w["down"], q, s, ws=self.ws["down"])
        steps["down"] = (q, s, out)
        return out, steps


def batch(lens, new, seed):
    g = torch.Generator().manual_seed(seed)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    T = starts[-1]
    pos = [p for n, m in zip(lens, new) for p in range(n - m, n)]
    seqs = [b for b, m in enumerate(new) for _ in range(m)]
    x = torch.randn((T, N), generator=g)
    return x.cuda(), (0.3 * torch.randn((T, N), generator=g)).to(BF16).cuda(), (i32(pos), i32(seqs), i32(starts), i32(lens), 128)


def product(q, s, W, bias=None):
    """Codes of the weights read back from the packed blocks [rows / 32][cols / 64][chunk][row][16]."""
    kb = (W.n_cols + 511) // 512 * 8
    w = W.packed.view(torch.int8).view(-1, kb, 4, 32, 16).permute(0, 3, 1, 2, 4).reshape(-1, kb * 64)[:W.n_rows, :W.n_cols]
    y = (q.cpu().double() @ w.cpu().double().T) * s.cpu().double()[:, None] * W.scale.cpu().double()
    return y if bias is None else y + bias.cpu().double()


def half_codes(y, q):
    """Codes are within half a step of the quotients (and fp32's roundings before)."""
    y = y.cpu().double()
    return (q.cpu().double() - 127 * y / y.abs().amax(1, keepdim=True)).abs().max() <= 0.5 + 127 * 2.0 ** -24 * 14


@pytest.mark.parametrize("lens,new", [([1, 1, 1], [1, 1, 1]), ([70, 33, 128], [70, 33, 128]), ([50, 20, 90], [1, 2, 40])])
def test_steps(dev, lens, new):
    """Every step against its formula on the step's own inputs."""
    L = Layer(dev, 1, 256, 3)
    h, y, args = batch(lens, new, 2)
    h0 = h.clone()
    out, st = L.run(h, y, *args)
    q, s, h1 = st["norm"]
    assert torch.equal(h1, h0 + y.float()) and half_codes(h1.double() * L.n1.double(), q)
    for (q, s, o), w, bias in ((st["qkv"], "qkv", L.bias), (st["down"], "down", None)):
        ref = product(q, s, L.w[w], bias)
        assert ((o.cpu().double() - ref).abs() <= 2.0 ** -8 * 1.001 * ref.abs() + 1e-5).all(), w
    att, q, s = st["attention"]
    assert half_codes(att, q)
    q, s, o, h2 = st["norm2"]
    assert torch.equal(h2, h1 + o.float()) and torch.equal(h, h2) and half_codes(h2.double() * L.n2.double(), q)
    gu, q, s = st["silu"]
    g = gu.double()
    assert half_codes(torch.nn.functional.silu(g[:, :FF]) * g[:, FF:], q)
    assert out.isfinite().all()


def test_near_unquantised(dev):
    """The whole chain of one token's feed-forward part against the same weights unquantised: each product is off by
    at most half a step of either side, which for normal rows of 512 is a few hundredths of the result's size."""
    L = Layer(dev, 3, 8, 1)
    g = torch.Generator().manual_seed(3)
    Layer_r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    n1, n2 = 1 + 0.2 * Layer_r(N), (1 + 0.2 * Layer_r(N)).to(BF16)   # the draws of Layer, in its order
    wide = (NH + 2 * NKH) * HD
    _, _ = Layer_r(wide, N), Layer_r(N, NH * HD)
    gu, down = (Layer_r(2 * FF, N) * N ** -0.5).half(), Layer_r(N, FF) * FF ** -0.5
    assert torch.equal(n1.cuda(), L.n1) and torch.equal(n2.cuda(), L.n2)
    h = torch.randn((4, N), generator=g)
    q, s = dev.i8_rms_norm(h.cuda(), L.n2, EPS)
    a = dev.i8_gemm(L.w["gu"], q, s, out_dtype=torch.float32)
    q, s = dev.i8_silu_mul(a[:, :FF], a[:, FF:])
    out = dev.i8_gemm(L.w["down"], q, s, out_dtype=torch.float32).cpu().double()
    x = h.double()
    x = x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * n2.double()
    z = x @ gu.double().T
    ref = (torch.nn.functional.silu(z[:, :FF]) * z[:, FF:]) @ down.double().T
    assert (out - ref).norm() <= 0.05 * ref.norm()


def test_captured(dev):
    """A captured layer, replayed with other inputs between eager work, gives the eager results; a second graph shares
    its workspaces."""
    L = Layer(dev, 4, 256, 3)
    cases = [batch([60, 40, 100], [60, 40, 100], s) for s in (5, 6, 7)]
    few = [batch([90, 90, 110], [1, 1, 1], s) for s in (8, 9, 10)]
    stream = torch.cuda.Stream()
    graphs = []
    for sets in (cases, few):
        h, y, args = (t.clone() if torch.is_tensor(t) else t for t in sets[0])
        with torch.cuda.stream(stream):
            L.run(h.clone(), y, *args)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            hh = h.clone()
            out, _ = L.run(hh, y, *args)
        graphs.append((graph, h, y, hh, out))
    for i in (0, 1, 2, 0):
        for sets, (graph, h, y, hh, out) in zip((cases, few), graphs):
            h0, y0, args = sets[i]
            h.copy_(h0)
            y.copy_(y0)
            graph.replay()
            torch.cuda.synchronize()
            got, gh = out.clone(), hh.clone()
            eh = h0.clone()
            want, _ = L.run(eh, y0, *args)
            assert torch.equal(got, want) and torch.equal(gh, eh)


def test_two_streams(dev):
    """Two layers at once on two streams, each with its own workspaces."""
    layers = [Layer(dev, s, 256, 3) for s in (11, 12)]
    sets = [batch([100, 37, 64], [100, 37, 64], s) for s in (13, 14)]
    want = [L.run(h.clone(), y, *args)[0] for L, (h, y, args) in zip(layers, sets)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(3):
        got = []
        for L, (h, y, args), st in zip(layers, sets, streams):
            with torch.cuda.stream(st):
                got.append(L.run(h.clone(), y, *args)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
