"""Plain 64-bit forms of the operators over a paged cache, on the CPU, and the
bounds that follow from how the kernels round."""
import math

import torch

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


class Cache:
    """Pools filled with rows of sequences of `rows` rows on scattered pages, everything else NaN (or, in 8 bits, the
    code of NaN), and the rows themselves in 64 bits, k[b], v[b]: [rows][NKH][HD]."""

    def __init__(self, seed, rows, NKH, HD, page, dtype, head_major=False, spare=3, wide=2, unmapped=()):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.NKH, self.HD, self.page, self.dtype = rows, NKH, HD, page, dtype
        need = [-(-n // page) for n in rows]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g)
        self.tables = torch.full((len(rows), max(need + [1]) + wide), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = order[at:at + n].int()
            at += n
        self.mapped = [torch.ones(n, dtype=torch.bool) for n in rows]
        shape = (self.n_pages, page, NKH, HD)
        pools, exps = [], []
        vals = []
        for _ in range(2):
            x = torch.randn(shape, generator=g)
            if dtype == E4M3:
                x = (x * 60).clamp(-448, 448).to(E4M3)
                e = torch.randint(118, 124, (self.n_pages, NKH, page), generator=g).to(torch.uint8)
                val = x.double() * (2.0 ** (e.double() - 127)).transpose(1, 2)[..., None]
            else:
                x, e = x.to(dtype), None
                val = x.double()
            vals.append(val)
            pools.append(x)
            exps.append(e)
        used = torch.zeros(self.n_pages, page, dtype=torch.bool)
        self.k, self.v = [], []
        for b, n in enumerate(rows):
            ids = self.tables[b, torch.arange(n) // page].long()
            used[ids, torch.arange(n) % page] = True
            self.k.append(vals[0][ids, torch.arange(n) % page])
            self.v.append(vals[1][ids, torch.arange(n) % page])
        for b, blk in unmapped:
            used[self.tables[b, blk].long()] = False
            self.tables[b, blk] = -1 if blk % 2 else self.n_pages + 5
            self.mapped[b][blk * page:(blk + 1) * page] = False
        for i, x in enumerate(pools):
            if dtype == E4M3:
                raw = x.view(torch.uint8).clone()
                raw[~used] = 0x7F
                pools[i] = raw.view(E4M3)
                exps[i].transpose(1, 2)[~used] = 255
            else:
                x[~used] = float("nan")
        self.pools, self.exps, self.head_major = pools, exps, head_major

    def view(self, dev):
        """The mllm_paged_kv over GPU copies."""
        cu = lambda t: None if t is None else t.cuda()  # noqa: E731
        pools = []
        for x in self.pools:
            raw = x.view(torch.uint8) if self.dtype == E4M3 else x
            if self.head_major:
                raw = raw.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
            else:
                raw = raw.cuda()
            pools.append(raw.view(E4M3) if self.dtype == E4M3 else raw)
        return dev.paged_kv(pools[0], pools[1], cu(self.tables), *(cu(e) for e in self.exps))


def attend(cache, b, q, pos, scale, window=0, sinks=None):
    """Queries q [n][NH][HD] (64 bits) of sequence b at positions pos [n]: (out, weighted |v|, largest scale * |q|.|k|,
    the same with every |q| at its row's largest)."""
    n, NH, HD = q.shape
    rep = NH // cache.NKH
    k, v, s = cache.k[b].clone(), cache.v[b].clone(), torch.arange(cache.rows[b])
    k[~cache.mapped[b]] = 0
    v[~cache.mapped[b]] = 0
    see = (s[None] <= pos[:, None]) & cache.mapped[b][None]
    if window:
        see &= s[None] > pos[:, None] - window
    k, v = (x.repeat_interleave(rep, 1) for x in (k, v))
    if not len(s):
        z = torch.zeros_like(q)
        return z, z, 0.0, 0.0
    w = torch.einsum("nhd,shd->nhs", q, k) * scale
    w = w.masked_fill(~see[:, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks.double()[None, :, None])
    top = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp(w - top)
    tot = w.sum(-1, keepdim=True)
    if sinks is not None:
        tot = tot + torch.exp(sinks.double()[None, :, None] - top)
    w = w / torch.where(tot == 0, 1.0, tot)
    o = torch.einsum("nhs,shd->nhd", w, v)
    o[~see.any(1)] = 0
    mag = torch.einsum("nhs,shd->nhd", w, v.abs())
    za = float((torch.einsum("nhd,shd->nhs", q.abs(), k.abs()) * abs(scale)).max())
    zq = float((q.abs().amax(-1)[..., None] * k.abs().sum(-1).T[None] * abs(scale)).max())
    return o, mag, za, zq


def attend_bound(o, mag, za, zq, S, HD, cache_dtype, q_dtype, out_dtype):
    """How far an output may be off.  Scores: an fp32 sum of HD products whose q keeps 22 bits of its row's largest
    element where it is split (2^-22 zq), and the argument of the exponential rounded once more; a score off by d moves
    a weight by a factor 1 + d and the normalised one by twice that (d is well below 1 here).  The two sums over S
    positions are fp32.  With 16-bit q and out each weight is rounded to the cache's 16-bit type, half a step."""
    u = 2.0 ** -24
    wide = q_dtype == F32 or out_dtype == F32
    half = torch.finfo(F16 if cache_dtype == F16 else BF16).eps / 2
    d = (HD + 8) * u * za + (2.0 ** -22 * zq if wide else 0.0) + 4 * u * za
    rel = 4 * d + 2 * (S + 64) * u + (2.0 ** -20 if wide else half)
    return mag * rel + o.abs() * torch.finfo(out_dtype).eps / 2 + 1e-30 + (2.0 ** -24 if out_dtype == F16 else 0.0)


def quantise_e4m3(x):
    """Rows x [..., HD] (64 bits) to e4m3: (codes' values, exponent), the exponent the least that brings the largest
    element to 448 or below."""
    m, k = torch.frexp(x.abs().amax(-1))
    e = torch.where(m == 0, 0, torch.where(m <= 0.875, k - 9, k - 8)).clamp(-100, 100)
    y = torch.ldexp(x, -e[..., None])
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448), e
