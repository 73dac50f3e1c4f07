"""Performance cases of the serving operators over a paged 16- or 8-bit KV cache.

  rotary   rotary positions on the q and k heads of T new tokens, q written out
           and k, v stored into their sequences' pages (DeviceOps.rotary_append)
  decode   attention of one new token per sequence over its cached rows
           (DeviceOps.paged_attn_decode)
  prompt   causal attention of each sequence's new tokens over its cached rows,
           the new ones among them (DeviceOps.paged_attn_prompt)
  fork     beams take over the state of other beams: whole pages shared, the
           last part-filled one copied (DeviceOps.pages_fork)
  compact  sequences end, the live pages move to the front of the pool, and new
           sequences get pages (DeviceOps.pages_free, pages_compact, pages_reserve)

A pool is [page][row][kv head][element]; an 8-bit (e4m3) pool has a power-of-two
scale per row and kv head, held as its biased exponent, [page][kv head][row].
"""
import math
import random

import numpy as np
import torch

own = False

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
TYPES = {"f32": F32, "f16": F16, "bf16": BF16, "e4m3": E4M3}


def listed():
    return [
        # one decode step of a small batch: the fp32 output of the q/k/v products, 64/8 heads of 64
        dict(name="rotary_decode_8", kind="rotary", T=8, B=8, NH=64, NKH=8, HD=64, rot=64, layout="half",
             scaling="yarn", inp="f32", out="bf16", cache="bf16", page=64, far=3000, mix=1),
        # the prompt of one sequence, 32/8 heads of 128, in 16 bits throughout
        dict(name="rotary_prompt_4096", kind="rotary", T=4096, B=1, NH=32, NKH=8, HD=128, rot=128, layout="half",
             scaling="bands", inp="bf16", out="bf16", cache="bf16", page=64, far=0, mix=2),
        # several prompts of odd lengths far into a long context: neighbouring pairs in half of each head, an
        # 8-bit cache on 16-row pages
        dict(name="rotary_ragged_e4m3", kind="rotary", T=1333, B=7, NH=16, NKH=4, HD=96, rot=48, layout="pairs",
             scaling="linear", inp="f32", out="f32", cache="e4m3", page=16, far=90000, mix=3),
        # the smallest call: one sequence early in its generation, fp32 in and out (TinyLlama heads)
        dict(name="decode_1x300", kind="decode", B=1, NH=32, NKH=4, HD=64, lo=300, hi=300, page=64, cache="f16",
             q="f32", out="f32", window=0, sinks=False, mix=4),
        # a small batch of unequal lengths, attention sinks (64/8 heads of 64)
        dict(name="decode_8x4096", kind="decode", B=8, NH=64, NKH=8, HD=64, lo=2048, hi=4096, page=64, cache="bf16",
             q="bf16", out="bf16", window=0, sinks=True, mix=5),
        # batched serving from an 8-bit cache: 48 sequences of up to 9000 rows (32/8 heads of 128)
        dict(name="decode_48x9000_e4m3", kind="decode", B=48, NH=32, NKH=8, HD=128, lo=1, hi=9000, page=32,
             cache="e4m3", q="bf16", out="bf16", window=0, sinks=False, mix=6),
        # one sequence in a long context (32/4 heads of 128)
        dict(name="decode_1x131072", kind="decode", B=1, NH=32, NKH=4, HD=128, lo=131072, hi=131072, page=64,
             cache="bf16", q="bf16", out="bf16", window=0, sinks=False, mix=7),
        # drafted tokens of eight sequences checked against long caches (64/8 heads of 64), fp32 in and out
        dict(name="prompt_draft_8x5", kind="prompt", B=8, NH=64, NKH=8, HD=64, new_lo=3, new_hi=5, past_lo=1500,
             past_hi=4000, page=64, cache="bf16", q="f32", out="f32", window=0, sinks=True, mix=8),
        # several prompts, some continued, with a sliding window, odd lengths (16/4 heads of 96)
        dict(name="prompt_ragged_window", kind="prompt", B=6, NH=16, NKH=4, HD=96, new_lo=1, new_hi=1100, past_lo=0,
             past_hi=1500, page=16, cache="f16", q="f16", out="f16", window=512, sinks=False, mix=9),
        # one long prompt (32/8 heads of 128)
        dict(name="prompt_1x6011", kind="prompt", B=1, NH=32, NKH=8, HD=128, new_lo=6011, new_hi=6011, past_lo=0,
             past_hi=0, page=64, cache="bf16", q="bf16", out="bf16", window=0, sinks=False, mix=10),
        # beam search, four prompts of four beams, in a model of 24 layers (8 kv heads of 64)
        dict(name="fork_4x4", kind="fork", G=4, W=4, length=1000, layers=24, NKH=8, HD=64, page=64, cache="bf16",
             mix=11),
        # half of a pool's sequences end and as many begin, 16 layers (4 kv heads of 128, 8 bits)
        dict(name="compact_24", kind="compact", B=24, lo=100, hi=900, layers=16, NKH=4, HD=128, page=32,
             cache="e4m3", mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "decode", "decode", "decode", "prompt", "prompt", "prompt", "fork",
                       "compact"])
    NKH = rng.choice([1, 2, 3, 4, 8])
    NH = NKH * rng.choice([1, 2, 4, 7, 8])
    HD = rng.choice([64, 64, 80, 96, 128, 128, 256])
    page = rng.choice([16, 32, 64, 64, 100, 128])
    mix = rng.randrange(1 << 20)
    cache = rng.choice(["bf16", "bf16", "f16", "e4m3"])
    act = "f16" if cache == "f16" else "bf16"
    if kind == "rotary":
        T = _log(rng, 1, min(4096, 25000000 // ((NH + 2 * NKH) * HD)))
        return dict(kind=kind, T=T, B=rng.randint(1, min(T, 16)), NH=NH, NKH=NKH, HD=HD,
                    rot=16 * rng.randint(1, HD // 16), layout=rng.choice(["half", "pairs"]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]), inp=rng.choice(["f32", act]),
                    out=rng.choice(["f32", act]), cache=cache, page=page, far=rng.choice([0, 1000, 120000]), mix=mix)
    if kind == "decode":
        B = _log(rng, 1, 48)
        return dict(kind=kind, B=B, NH=NH, NKH=NKH, HD=HD, lo=1,
                    hi=_log(rng, 1, min(100000, 60000000 // (B * NKH * HD))), page=page, cache=cache,
                    q=(t := rng.choice(["f32", act, act])), out=t, window=rng.choice([0, 0, 0, 128, 1000]),
                    sinks=rng.random() < 0.4, mix=mix)
    if kind == "prompt":
        pairs = 6e10 / (NH * HD)                        # of a query and a cached row, at most
        hi = _log(rng, 1, int(min(4000, math.sqrt(pairs))))
        B = rng.randint(1, max(1, min(12, 4000 // hi, int(pairs / hi ** 2))))
        past = max(1, min(4000, int(pairs / (B * hi) - hi / 2)))
        return dict(kind=kind, B=B, NH=NH, NKH=NKH, HD=HD, new_lo=1, new_hi=hi, past_lo=0,
                    past_hi=rng.choice([0, _log(rng, 1, past)]), page=page, cache=cache,
                    q=(t := rng.choice(["f32", act, act])), out=t, window=rng.choice([0, 0, 0, 128, 1000]),
                    sinks=rng.random() < 0.4, mix=mix)
    layers = rng.randint(1, 12)
    NKH, HD = rng.choice([(2, 64), (4, 128), (8, 64), (3, 80)])
    if kind == "fork":
        return dict(kind=kind, G=_log(rng, 1, 12), W=rng.randint(2, 8), length=_log(rng, 1, 3000), layers=layers,
                    NKH=NKH, HD=HD, page=page, cache=cache, mix=mix)
    return dict(kind=kind, B=2 * rng.randint(1, 12), lo=1, hi=_log(rng, 20, 900), layers=layers, NKH=NKH, HD=HD,
                page=page, cache=cache, mix=mix)


# ------------------------------------------------------------------ what a case fixes besides its fields
def _lens(case):
    """Cached rows of each sequence of a decode case."""
    r = random.Random(case["mix"])
    return [case["hi"]] + [_log(r, case["lo"], case["hi"]) for _ in range(case["B"] - 1)]


def _prompt_lens(case):
    """(new tokens, cached rows before them) of each sequence of a prompt case."""
    r = random.Random(case["mix"])
    new = [case["new_hi"]] + [_log(r, case["new_lo"], case["new_hi"]) for _ in range(case["B"] - 1)]
    return new, [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["B"])]


def _rotary_tokens(case):
    """(sequence, position) of each token: T tokens over B sequences, each a run of positions from its start."""
    r = random.Random(case["mix"])
    cuts = sorted(r.sample(range(1, case["T"]), case["B"] - 1)) if case["B"] > 1 else []
    n = [b - a for a, b in zip([0] + cuts, cuts + [case["T"]])]
    start = [r.randint(case["far"], 2 * case["far"]) for _ in n]
    return [b for b, k in enumerate(n) for _ in range(k)], [start[b] + i for b, k in enumerate(n) for i in range(k)]


def _parents(case):
    """Fork case: the beam of the same group that each beam goes on from (about two in five stay)."""
    r = random.Random(case["mix"])
    return [g * case["W"] + (w if r.random() < 0.3 else r.randrange(case["W"]))
            for g in range(case["G"]) for w in range(case["W"])]


def _blocks(n, page):
    return -(-n // page)


def _freqs(case):
    """Radians per position of the r/2 pairs and the factor on q and k, in 64 bits."""
    r, base, f, ctx = case["rot"], 150000.0, 32.0, 4096.0
    j = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    w = base ** (-2 * j / r)
    kind = case["scaling"]
    if kind == "linear":
        return w / f, 1.0
    if kind == "ntk":
        return (base * f ** (r / max(r - 2, 1))) ** (-2 * j / r), 1.0
    if kind == "yarn":
        lo, hi = (r * math.log(ctx / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
        ramp = ((j - lo) / (hi - lo if hi > lo else 0.001)).clamp(0, 1)
        return w / f * ramp + w * (1 - ramp), 0.1 * math.log(f) + 1
    if kind == "bands":
        s = ((ctx * w / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return w / f * (1 - s) + w * s, 1.0
    return w, 1.0


# ------------------------------------------------------------------ inputs
def _randn(g, shape, dtype):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def _pool(g, shape, cache):
    """A pool of rows, and with e4m3 the biased exponents of their scales; made layer by layer to bound memory."""
    if cache != "e4m3":
        return _randn(g, shape, TYPES[cache]), None
    p, r, h, d = shape
    exp = torch.randint(119, 123, (p, h, r), device="cuda", generator=g).to(torch.uint8)
    return (_randn(g, shape, F32) * 60).to(E4M3), exp


def _tables(case, rows, spare=3):
    """Pages in scattered order for sequences of `rows` rows: (tables, pages in the pool)."""
    page = case["page"]
    need = [_blocks(n, page) for n in rows]
    n = sum(need) + spare
    order = torch.randperm(n, generator=torch.Generator().manual_seed(case["mix"])).to(torch.int32)
    t = torch.full((len(rows), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        t[b, :k] = order[at:at + k]
        at += k
    return t.cuda(), n


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + 17) & 0x7FFFFFFFFFFFFFF)
    s = dict(case=case)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["kind"] in ("fork", "compact"):
        _prepare_pages(case, g, s, i32)
    elif case["kind"] == "rotary":
        seq, pos = _rotary_tokens(case)
        page, heads = case["page"], case["NH"] + 2 * case["NKH"]
        blocks = sorted({(b, p // page) for b, p in zip(seq, pos)})
        t = torch.full((case["B"], max(b for _, b in blocks) + 1), -1, dtype=torch.int32)
        n = len(blocks) + 2
        order = torch.randperm(n, generator=torch.Generator().manual_seed(case["mix"]))
        for i, (b, k) in enumerate(blocks):
            t[b, k] = int(order[i])
        s.update(tables=t.cuda(), seq=i32(seq), pos=i32(pos),
                 qkv=_randn(g, (case["T"], heads * case["HD"]), TYPES[case["inp"]]),
                 q_out=torch.zeros((case["T"], case["NH"] * case["HD"]), dtype=TYPES[case["out"]], device="cuda"))
        for x in ("k", "v"):
            s[x], s[x + "_exp"] = _pool(g, (n, page, case["NKH"], case["HD"]), case["cache"])
        s["freqs"], s["mscale"] = _freqs(case)
    else:
        if case["kind"] == "decode":
            lens = _lens(case)
            tokens = case["B"]
        else:
            new, past = _prompt_lens(case)
            lens, tokens = [a + b for a, b in zip(new, past)], sum(new)
            s["starts"] = i32([0] + list(np.cumsum(new)))
            s["max_new"] = max(new)
        s["tables"], n = _tables(case, lens)
        s["lens"], s["max_len"] = i32(lens), max(lens)
        for x in ("k", "v"):
            s[x], s[x + "_exp"] = _pool(g, (n, case["page"], case["NKH"], case["HD"]), case["cache"])
        s["q"] = (1.5 * torch.randn((tokens, case["NH"] * case["HD"]), device="cuda", generator=g)).to(TYPES[case["q"]])
        s["sinks"] = torch.randn(case["NH"], device="cuda", generator=g) if case["sinks"] else None
        s["out"] = torch.empty((tokens, case["NH"] * case["HD"]), dtype=TYPES[case["out"]], device="cuda")
    if own:
        _handles(s)
    return s


def _prepare_pages(case, g, s, i32):
    page = case["page"]
    if case["kind"] == "fork":
        # every group's beams share their whole pages; each has its last, part-filled page for itself
        full, part, W = case["length"] // page, case["length"] % page != 0, case["W"]
        n = case["G"] * (full + 2 * W * part) + 4
        t = torch.full((case["G"] * W, full + 2), -1, dtype=torch.int32)
        refs = torch.zeros(n, dtype=torch.int32)
        order = torch.randperm(n, generator=torch.Generator().manual_seed(case["mix"])).to(torch.int32)
        at = 0
        for i in range(case["G"]):
            rows = slice(i * W, i * W + W)
            t[rows, :full] = order[at:at + full]
            refs[order[at:at + full].long()] = W
            at += full
            if part:
                t[rows, full] = order[at:at + W]
                refs[order[at:at + W].long()] = 1
                at += W
        s.update(tables=t.cuda(), refs=refs.cuda(), parents=i32(_parents(case)), children=i32(list(range(len(t)))),
                 lens=i32([case["length"]] * len(t)))
    else:
        # two halves of sequences, the first on the lower pages: each pass one half ends and comes back
        lens = _lens(case)
        need = [_blocks(x, page) for x in lens]
        n = sum(need) + 2
        t = torch.full((case["B"], max(need)), -1, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            t[b, :k] = torch.arange(at, at + k, dtype=torch.int32)
            at += k
        refs = torch.zeros(n, dtype=torch.int32)
        refs[:at] = 1
        half = [list(range(case["B"] // 2)), list(range(case["B"] // 2, case["B"]))]
        s.update(tables=t.cuda(), refs=refs.cuda(), halves=[i32(h) for h in half],
                 lens=[i32([lens[b] for b in h]) for h in half], turn=0)
    # [layer][page]...: the pages of all layers go together
    for x in ("k", "v"):
        both = [_pool(g, (n, page, case["NKH"], case["HD"]), case["cache"]) for _ in range(case["layers"])]
        s[x] = torch.stack([b[0].view(torch.uint8) if case["cache"] == "e4m3" else b[0] for b in both])
        if case["cache"] == "e4m3":
            s[x] = s[x].view(E4M3)
        s[x + "_exp"] = torch.stack([b[1] for b in both]) if case["cache"] == "e4m3" else None


def _handles(s):
    """What a program on the framework keeps beside its tensors: views, the rotary plan, workspaces."""
    from mojollama_amd import kernels as K
    c = s["case"]
    dev = s["dev"] = K.DeviceOps()
    if c["kind"] in ("fork", "compact"):
        s["map"] = dev.page_map(s["tables"], s["refs"], c["page"])
        s["planes"] = dev.page_planes([x for x in (s["k"], s["v"], s["k_exp"], s["v_exp"]) if x is not None])
        s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["ws"] = dev.pages_workspace(s["map"], len(s["tables"]))
        return
    s["kv"] = dev.paged_kv(s["k"], s["v"], s["tables"], k_exp=s["k_exp"], v_exp=s["v_exp"])
    if c["kind"] == "rotary":
        kind = dict(none=K.ROPE_NONE, linear=K.ROPE_LINEAR, ntk=K.ROPE_NTK, yarn=K.ROPE_YARN, bands=K.ROPE_BANDS)
        s["rot"] = dev.rotary(c["rot"], layout=K.ROPE_HALF if c["layout"] == "half" else K.ROPE_PAIRS,
                              base=150000.0, scaling=kind[c["scaling"]], factor=32.0, ctx=4096.0)
        a, b = c["NH"] * c["HD"], c["NKH"] * c["HD"]
        s["parts"] = s["qkv"][:, :a], s["qkv"][:, a:a + b], s["qkv"][:, a + b:]
    elif c["kind"] == "decode":
        s["ws"] = dev.paged_attn_workspace(s["kv"], c["B"], c["B"], c["NH"], s["max_len"], c["window"])
    else:
        s["ws"] = dev.paged_attn_workspace(s["kv"], len(s["q"]), c["B"], c["NH"], s["max_len"], c["window"])


# ------------------------------------------------------------------ one pass
def run(s):
    return {"rotary": _rotary, "decode": _attend, "prompt": _attend, "fork": _fork, "compact": _compact}[
        s["case"]["kind"]](s)


def _pools(s):
    return [s[x] for x in ("k", "v", "k_exp", "v_exp") if s[x] is not None]


def _rotary(s):
    c = s["case"]
    if own:
        q, k, v = s["parts"]
        s["dev"].rotary_append(s["rot"], q, k, v, s["pos"], NH=c["NH"], kv=s["kv"], seqs=s["seq"], q_out=s["q_out"])
        return [s["q_out"]] + _pools(s)
    NH, NKH, HD, r, page = c["NH"], c["NKH"], c["HD"], c["rot"], c["page"]
    # values held in 8 bits are rounded from 64: a code or scale next to a border is the same however it is summed
    wide = torch.float64 if c["cache"] == "e4m3" else F32
    a = s["pos"].double()[:, None] * s["freqs"]
    cos, sin = (f(a) * s["mscale"] for f in (torch.cos, torch.sin))
    x = s["qkv"].view(c["T"], NH + 2 * NKH, HD)
    rotated = []
    for y, w in ((x[:, :NH], F32), (x[:, NH:NH + NKH], wide)):
        y, co, si = y.to(w), cos.to(w)[:, None], sin.to(w)[:, None]
        if c["layout"] == "half":
            p, q = y[..., :r // 2], y[..., r // 2:r]
            z = torch.cat([p * co - q * si, q * co + p * si], -1)
        else:
            p, q = y[..., 0:r:2], y[..., 1:r:2]
            z = torch.stack([p * co - q * si, q * co + p * si], -1).flatten(-2)
        rotated.append(torch.cat([z, y[..., r:]], -1))
    s["q_out"].copy_(rotated[0].reshape(c["T"], -1))
    pos = s["pos"].long()
    at, row = s["tables"][s["seq"].long(), pos // page].long(), pos % page
    _store(s, "k", at, row, rotated[1])
    _store(s, "v", at, row, x[:, NH + NKH:].to(wide))
    return [s["q_out"]] + _pools(s)


def _store(s, name, at, row, x):
    pool = s[name]
    if s["case"]["cache"] != "e4m3":
        pool[at, row] = x.to(pool.dtype)
        return
    m, k = torch.frexp(x.abs().amax(-1))                # the largest is m 2^k, 448 is 0.875 2^9
    e = torch.where(m == 0, 0, torch.where(m <= 0.875, k - 9, k - 8)).clamp(-100, 100)
    y = torch.ldexp(x, -e[..., None])
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    y = (torch.round(y / step) * step).clamp(-448, 448).float().to(E4M3)
    pool.view(torch.uint8)[at, row] = y.view(torch.uint8)
    s[name + "_exp"][at[:, None], torch.arange(x.shape[1], device=x.device), row[:, None]] = (e + 127).to(torch.uint8)


def _cached(s, name, ids, row):
    x = s[name][ids, row] if s["case"]["cache"] != "e4m3" else s[name].view(torch.uint8)[ids, row].view(E4M3)
    x = x.float()                                       # [B][S][NKH][HD]
    if s[name + "_exp"] is not None:
        x = x * torch.exp2(s[name + "_exp"].permute(0, 2, 1)[ids, row].float() - 127)[..., None]
    return x.transpose(1, 2)


def _attend(s):
    c = s["case"]
    scale = 1 / math.sqrt(c["HD"])
    if own:
        if c["kind"] == "decode":
            s["dev"].paged_attn_decode(s["kv"], s["q"], s["lens"], s["max_len"], c["NH"], scale=scale,
                                       window=c["window"], sinks=s["sinks"], out=s["out"], ws=s["ws"])
        else:
            s["dev"].paged_attn_prompt(s["kv"], s["q"], s["starts"], s["lens"], s["max_len"], c["NH"], scale=scale,
                                       window=c["window"], sinks=s["sinks"], out=s["out"], ws=s["ws"])
        return s["out"]
    B, NH, NKH, HD, page = c["B"], c["NH"], c["NKH"], c["HD"], c["page"]
    G, S = NH // NKH, s["max_len"]
    pos = torch.arange(S, device="cuda")
    ids, row = s["tables"].long()[:, pos // page].clamp(min=0), (pos % page).expand(B, S)
    k, v = _cached(s, "k", ids, row), _cached(s, "v", ids, row)              # [B][NKH][S][HD]
    # queries padded to the longest sequence's: n of them, query i of sequence b at its position `at`
    lens = s["lens"].long()
    if c["kind"] == "decode":
        n, token, real, at = 1, torch.arange(B, device="cuda")[:, None], None, lens[:, None] - 1
    else:
        n, first = s["max_new"], s["starts"].long()
        i, new = torch.arange(n, device="cuda"), first[1:] - first[:-1]
        real = i < new[:, None]
        token = (first[:-1, None] + i).clamp(max=len(s["q"]) - 1)
        at = (lens - new)[:, None] + i
    q = s["q"][token].float().view(B, n, NKH, G, HD).permute(0, 2, 3, 1, 4).reshape(B, NKH, G * n, HD)
    w = (torch.matmul(q, k.transpose(2, 3).contiguous()) * scale).view(B, NKH, G, n, S)
    seen = (pos <= at[..., None]) & (pos < lens[:, None, None])
    if c["window"]:
        seen &= pos > at[..., None] - c["window"]
    w.masked_fill_(~seen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(NKH, G, 1, 1)
        top = torch.maximum(top, sink)
    top = top.clamp(min=-3e38)
    w = torch.exp(w - top)
    total = w.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    v = torch.where((pos < lens[:, None])[:, None, :, None], v, torch.zeros((), device="cuda"))
    o = torch.matmul(w.view(B, NKH, G * n, S), v).view(B, NKH, G, n, HD) / torch.where(total == 0, 1, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, NH * HD)
    s["out"].copy_(o[:, 0] if real is None else o[real])
    return s["out"]


def _fork(s):
    c = s["case"]
    if own:
        s["dev"].pages_fork(s["map"], s["planes"], s["parents"], s["children"], s["lens"], status=s["status"],
                            ws=s["ws"])
        return [s["tables"], s["refs"]] + _pools(s)
    tables, refs = s["tables"], s["refs"]
    parent, child, lens = s["parents"].long(), s["children"].long(), s["lens"].long()
    on = parent != child
    parent, child, lens = parent[on], child[on], lens[on]
    blk = torch.arange(tables.shape[1], device="cuda")
    full = (lens // c["page"])[:, None]
    rows = torch.where(blk < full, tables[parent], -1)
    part = lens % c["page"] != 0
    src = tables[parent[part], full[part, 0]].long()
    dst = torch.nonzero(refs == 0)[:len(src), 0]
    rows[part, full[part, 0]] = dst.int()
    one = torch.ones((), dtype=torch.int32, device="cuda")
    gone = tables[child].long()
    refs.index_add_(0, rows[rows >= 0].long(), one.expand(int((rows >= 0).sum())))
    refs.index_add_(0, gone[gone >= 0], -one.expand(int((gone >= 0).sum())))
    tables[child] = rows
    _move(s, src, dst)
    return [tables, refs] + _pools(s)


def _move(s, src, dst):
    for x in _pools(s):
        x = x.view(torch.uint8) if x.dtype == E4M3 else x
        x[:, dst] = x[:, src]


def _compact(s):
    c = s["case"]
    turn = s["turn"]
    s["turn"] = 1 - turn
    seqs, lens = s["halves"][turn], s["lens"][turn]
    if own:
        s["dev"].pages_free(s["map"], seqs)
        s["dev"].pages_compact(s["map"], s["planes"], status=s["status"], ws=s["ws"])
        s["dev"].pages_reserve(s["map"], seqs, lens, status=s["status"], ws=s["ws"])
        return [s["tables"], s["refs"]] + _pools(s)
    tables, refs = s["tables"], s["refs"]
    one = torch.ones((), dtype=torch.int32, device="cuda")
    gone = tables[seqs.long()].long()
    refs.index_add_(0, gone[gone >= 0], -one.expand(int((gone >= 0).sum())))
    tables[seqs.long()] = -1
    live = refs > 0
    n = int(live.sum())
    src = torch.nonzero(live[n:])[:, 0] + n
    dst = torch.nonzero(~live[:n])[:, 0]
    to = torch.arange(len(refs), dtype=torch.int32, device="cuda")
    to[src] = dst.int()
    tables.copy_(torch.where(tables >= 0, to[tables.clamp(min=0).long()], -1))
    refs[dst] = refs[src]
    refs[src] = 0
    _move(s, src, dst)
    want = torch.arange(tables.shape[1], device="cuda") < ((lens.long() + c["page"] - 1) // c["page"])[:, None]
    rows = tables[seqs.long()]
    want &= rows < 0
    got = torch.nonzero(refs == 0)[:int(want.sum()), 0]
    rows[want] = got.int()
    tables[seqs.long()] = rows
    refs[got] = 1
    return [tables, refs] + _pools(s)


# ------------------------------------------------------------------ what a pass cannot do without
def _size(name):
    return {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}[name]


def _row_bytes(case):
    """One cached row of K or of V, all kv heads."""
    return case["NKH"] * (case["HD"] * _size(case["cache"]) + (case["cache"] == "e4m3"))


def work(case):
    if case["kind"] == "rotary":
        n = case["NH"] + 2 * case["NKH"]
        b = case["T"] * (n * case["HD"] * _size(case["inp"]) + case["NH"] * case["HD"] * _size(case["out"])
                         + 2 * _row_bytes(case) + 8)
        return {"bytes": b, "flops": 3 * case["T"] * (case["NH"] + case["NKH"]) * case["rot"]}
    if case["kind"] in ("decode", "prompt"):
        if case["kind"] == "decode":
            new, past = [1] * case["B"], [n - 1 for n in _lens(case)]
        else:
            new, past = _prompt_lens(case)
        w = case["window"] or 1 << 40
        rows = sum(min(p + n, w + n - 1) for n, p in zip(new, past))
        # query i of a sequence sees min(past + i + 1, window) rows
        pairs = sum(int(np.minimum(p + 1 + np.arange(n), w).sum()) for n, p in zip(new, past))
        b = 2 * rows * _row_bytes(case) + sum(new) * case["NH"] * case["HD"] * (_size(case["q"]) + _size(case["out"]))
        return {"bytes": b, "flops": 4 * pairs * case["NH"] * case["HD"]}
    page_bytes = 2 * case["layers"] * case["page"] * _row_bytes(case)
    if case["kind"] == "fork":
        moved = sum(p != i for i, p in enumerate(_parents(case))) if case["length"] % case["page"] else 0
        tables = case["G"] * case["W"] * _blocks(case["length"], case["page"]) * 8
        return {"bytes": 2 * moved * page_bytes + tables, "flops": 0}
    need = [_blocks(n, case["page"]) for n in _lens(case)]
    # the half that goes on lies above the other's pages (in every second pass the other way round): what lies
    # past the number of live pages moves
    a, b = sum(need[:len(need) // 2]), sum(need[len(need) // 2:])
    return {"bytes": 2 * min(a, b) * page_bytes + 8 * sum(need), "flops": 0}


# ------------------------------------------------------------------ the same from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(dict(case), seed)
    return {"rotary": _exact_rotary, "decode": _exact_attend, "prompt": _exact_attend, "fork": _exact_fork,
            "compact": _exact_compact}[case["kind"]](case, s)


def _values(x):
    return x.float().double()


def _exact_rotary(case, s):
    """Each pair as a complex number times e^(i angle)."""
    NH, NKH, HD, r = case["NH"], case["NKH"], case["HD"], case["rot"]
    seq, pos = _rotary_tokens(case)
    x = _values(s["qkv"]).view(case["T"], NH + 2 * NKH, HD)
    turn = torch.polar(torch.full((), s["mscale"], dtype=torch.float64, device="cuda").expand(case["T"], r // 2),
                       torch.outer(torch.tensor(pos, dtype=torch.float64, device="cuda"), s["freqs"]))[:, None]
    head = x[:, :NH + NKH, :r]
    if case["layout"] == "half":
        z = torch.complex(head[..., :r // 2].contiguous(), head[..., r // 2:].contiguous()) * turn
        x[:, :NH + NKH, :r] = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(head.reshape(case["T"], NH + NKH, r // 2, 2).contiguous()) * turn
        x[:, :NH + NKH, :r] = torch.view_as_real(z).flatten(-2)
    out = [x[:, :NH].reshape(case["T"], -1)]
    table = s["tables"].cpu().numpy()
    at = torch.tensor([int(table[b, p // case["page"]]) * case["page"] + p % case["page"] for b, p in zip(seq, pos)],
                      device="cuda")
    exps = []
    for name, y in (("k", x[:, NH:NH + NKH]), ("v", x[:, NH + NKH:])):
        pool = _values(s[name])
        flat = pool.view(-1, NKH, HD)
        if case["cache"] == "e4m3":
            # the least power of two that brings the row's largest element to 448 or below
            e = torch.ceil(torch.log2(y.abs().amax(-1) / 448))
            y = y / torch.exp2(e)[..., None]
            # the values that e4m3 holds, in the order of their codes
            grid = torch.tensor([m * 2.0 ** (q - 3) for q in range(-6, 9) for m in range(0 if q == -6 else 8, 16)
                                 if m * 2.0 ** (q - 3) <= 448], dtype=torch.float64, device="cuda")
            i = torch.searchsorted(grid, y.abs()).clamp(1, len(grid) - 1)
            lo, hi = grid[i - 1], grid[i]
            up = (hi - y.abs() < y.abs() - lo) | ((hi - y.abs() == y.abs() - lo) & (i % 2 == 0))
            y = torch.sign(y) * torch.where(up, hi, lo)
            b = s[name + "_exp"].permute(0, 2, 1).reshape(-1, NKH).clone()
            b[at] = (e + 127).to(torch.uint8)
            exps.append(b.view(pool.shape[0], case["page"], NKH).permute(0, 2, 1).contiguous())
        flat[at] = y
        out.append(pool)
    return out + exps


def _exact_attend(case, s):
    """Sequence by sequence, its rows gathered and every score formed in 64 bits."""
    NH, NKH, HD, page = case["NH"], case["NKH"], case["HD"], case["page"]
    if case["kind"] == "decode":
        past, new = [n - 1 for n in _lens(case)], [1] * case["B"]
    else:
        new, past = _prompt_lens(case)
    out = torch.zeros((sum(new), NH, HD), dtype=torch.float64, device="cuda")
    t0 = 0
    for b, (n, p) in enumerate(zip(new, past)):
        pages = s["tables"][b, :_blocks(n + p, page)].long()
        kv = []
        for x in ("k", "v"):
            rows = s[x].view(torch.uint8)[pages].view(s[x].dtype) if case["cache"] == "e4m3" else s[x][pages]
            rows = _values(rows)
            if s[x + "_exp"] is not None:
                rows = rows * (2.0 ** (s[x + "_exp"][pages].double() - 127)).transpose(1, 2)[..., None]
            kv.append(rows.reshape(-1, NKH, HD)[:n + p])
        q = _values(s["q"][t0:t0 + n]).view(n, NH, HD)
        i = torch.arange(n, device="cuda")[:, None] + p
        j = torch.arange(n + p, device="cuda")[None]
        off = (j > i) | ((i - j >= case["window"]) if case["window"] else (j < 0))
        for h in range(NH):
            w = q[:, h] @ kv[0][:, h // (NH // NKH)].T / math.sqrt(HD)
            w[off] = -math.inf
            if s["sinks"] is not None:
                w = torch.cat([w, s["sinks"][h].double().expand(n, 1)], 1)
            out[t0:t0 + n, h] = torch.softmax(w, 1)[:, :n + p] @ kv[1][:, h // (NH // NKH)]
        t0 += n
    return out.view(sum(new), NH * HD)


def _exact_fork(case, s):
    """Beam by beam, with lists."""
    t, refs, page, n = s["tables"].tolist(), s["refs"].tolist(), case["page"], case["length"]
    was, free, moves = [list(r) for r in t], [p for p, r in enumerate(refs) if r == 0], []
    for i, p in enumerate(_parents(case)):
        if p == i:
            continue
        row = [-1] * len(t[i])
        for b in range(n // page):
            row[b] = was[p][b]
            refs[row[b]] += 1
        if n % page:
            row[n // page] = free.pop(0)
            refs[row[n // page]] += 1
            moves.append((was[p][n // page], row[n // page]))
        for x in was[i]:
            if x >= 0:
                refs[x] -= 1
        t[i] = row
    return _moved(s, t, refs, moves)


def _moved(s, t, refs, moves):
    src, dst = ([m[i] for m in moves] for i in (0, 1))
    out = [torch.tensor(t), torch.tensor(refs)]
    for x in _pools(s):
        y = x if x.dtype == torch.uint8 else x.float()
        y[:, dst] = y[:, src].clone()
        out.append(y)
    return out


def _exact_compact(case, s):
    t, refs, page = s["tables"].tolist(), s["refs"].tolist(), case["page"]
    lens, gone = _lens(case), range(case["B"] // 2)
    for b in gone:
        for x in t[b]:
            if x >= 0:
                refs[x] -= 1
        t[b] = [-1] * len(t[b])
    n = sum(r > 0 for r in refs)
    moves = list(zip([p for p in range(n, len(refs)) if refs[p] > 0], [p for p in range(n) if refs[p] == 0]))
    to = dict(moves)
    for a, b in moves:
        refs[b], refs[a] = refs[a], 0
    t = [[to.get(x, x) for x in row] for row in t]
    for b in gone:
        for k in range(_blocks(lens[b], page)):
            t[b][k] = refs.index(0)
            refs[t[b][k]] = 1
    return _moved(s, t, refs, moves)
