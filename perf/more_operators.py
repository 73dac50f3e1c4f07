"""Performance cases of layers whose weights and activations are 8-bit integers, with a scale for
each weight row (output channel) and each token.

  quantize  T rows to 8-bit integers, and back to the values these stand for
            (DeviceOps.i8_quantize, i8_dequant)
  norm      residual addition and root-mean-square norm of T rows, into 8-bit integers
            (DeviceOps.i8_rms_norm, i8_dequant)
  silu      silu(gate) * up of T rows, into 8-bit integers (DeviceOps.i8_silu_mul, i8_dequant)
  gemm      the matrix product of T such rows with such weights (DeviceOps.i8_gemm)

Row t of a quantised matrix stands for scale[t] * q[t][i], with scale[t] = max |x[t]| / 127 and
q[t][i] = x[t][i] * (127 / max |x[t]|), rounded to the nearest integer, ties to even.  What is held
in 8 bits is returned as the values it stands for, in 16 bits.
"""
import math

import torch

own = False

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}
EPS = 1e-6


def listed():
    return [
        # one decode step of a small batch, the fp32 rows of a width that the framework's tests use
        dict(name="quantize_decode_8", kind="quantize", T=8, n=2048, type="f32", pad=0),
        # the attention output of a long prompt, in front of the output product
        dict(name="quantize_prompt_4096", kind="quantize", T=4096, n=4096, type="bf16", pad=0),
        # odd rows out of a wider buffer: neither their width nor their stride is a multiple of 16 bytes
        dict(name="quantize_ragged_1333", kind="quantize", T=1333, n=2881, type="f16", pad=6),
        # one token's residual stream held in fp32, the last product's output in 16 bits
        dict(name="norm_decode_1", kind="norm", T=1, n=2880, type="bf16", res="f32", w="f32"),
        # a long prompt, everything in 16 bits
        dict(name="norm_prompt_8192", kind="norm", T=8192, n=4096, type="bf16", res="bf16", w="bf16"),
        # the gate and up halves of one product's output, a batch of decoding sequences
        dict(name="silu_decode_16", kind="silu", T=16, n=5632, type="bf16"),
        # the same for a long prompt
        dict(name="silu_prompt_4096", kind="silu", T=4096, n=11264, type="bf16"),
        # one token against the gate or up matrix of a small model, fp32 out
        dict(name="gemm_decode_1", kind="gemm", T=1, rows=5632, cols=2048, out="f32", bias=False),
        # a batch of decoding sequences against a square matrix with bias
        dict(name="gemm_decode_16", kind="gemm", T=16, rows=4096, cols=4096, out="bf16", bias=True),
        # more sequences, drafts or short prompts: gate and up in one matrix
        dict(name="gemm_batch_96", kind="gemm", T=96, rows=11264, cols=2048, out="bf16", bias=False),
        # odd sizes in every direction
        dict(name="gemm_ragged_1021", kind="gemm", T=1021, rows=2883, cols=2881, out="f16", bias=True),
        # a long prompt against a large matrix
        dict(name="gemm_prompt_8192", kind="gemm", T=8192, rows=8192, cols=8192, out="bf16", bias=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "norm", "silu", "gemm", "gemm", "gemm"])
    if kind == "gemm":
        while True:
            T, rows, cols = _log(rng, 1, 8192), _log(rng, 16, 32768), _log(rng, 33, 16384)
            if T * rows * cols <= 8192 ** 3 and rows * cols <= 1 << 28 and T * rows <= 1 << 27:
                break
        return dict(kind=kind, T=T, rows=rows, cols=cols, out=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    bias=rng.random() < 0.4)
    while True:
        T, n = _log(rng, 1, 8192), _log(rng, 8, 16384)
        if T * n <= 4096 * 11264:
            break
    c = dict(kind=kind, T=T, n=n, type=rng.choice(["bf16", "bf16", "f16", "f32"]))
    if kind == "quantize":
        c["pad"] = rng.choice([0, 0, 1, 8, 64])
    if kind == "norm":
        c["res"] = rng.choice([c["type"], "f32", "none"])
        c["w"] = rng.choice(["f32", c["type"]])
    return c


# ------------------------------------------------------------------ inputs
def _rows(g, T, n, kind):
    """Activations as layers see them: normal, some channels a good deal larger, tokens of different size."""
    x = torch.randn((T, n), device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn((T, 1), device="cuda", generator=g))
    x *= 1.0 + 11.0 * (torch.rand(n, device="cuda", generator=g) < 0.01)
    return x.to(TYPES[kind])


def _codes(g, T, n):
    """8-bit integers of normal values under the scale of their largest, about four deviations."""
    return (torch.randn((T, n), device="cuda", generator=g) * 31.0).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}
    kind, T = case["kind"], case["T"]
    if kind == "gemm":
        rows, cols = case["rows"], case["cols"]
        wide = (cols + 15) // 16 * 16                     # rows at multiples of 16 bytes
        s["x"] = torch.zeros((T, wide), dtype=torch.int8, device="cuda")[:, :cols]
        s["x"].copy_(_codes(g, T, cols))
        s["x_scale"] = torch.exp(0.5 * torch.randn(T, device="cuda", generator=g)) * 4.0 / 127.0
        s["w"] = _codes(g, rows, cols)
        s["w_scale"] = torch.exp(0.3 * torch.randn(rows, device="cuda", generator=g)) * 4.0 / 127.0 / math.sqrt(cols)
        s["bias"] = torch.randn(rows, device="cuda", generator=g) if case["bias"] else None
        s["out"] = torch.empty((T, rows), dtype=TYPES[case["out"]], device="cuda")
    else:
        n = case["n"]
        if kind == "quantize":
            s["x"] = _rows(g, T, n + case["pad"], case["type"])[:, case["pad"]:]
        elif kind == "norm":
            s["x"] = _rows(g, T, n, case["type"])
            s["res"] = None if case["res"] == "none" else _rows(g, T, n, case["res"])
            s["res_out"] = None if case["res"] == "none" else torch.empty_like(s["res"])
            s["w"] = (1.0 + 0.2 * torch.randn(n, device="cuda", generator=g)).to(TYPES[case["w"]])
        else:
            s["x"] = _rows(g, T, 2 * n, case["type"])     # gate, then up
        s["q"] = torch.empty((T, (n + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :n]
        s["scale"] = torch.empty(T, device="cuda")
        s["out"] = torch.empty((T, n), dtype=F16 if case["type"] == "f16" else BF16, device="cuda")
    if own:
        from mojollama_amd import kernels as K
        s["dev"] = K.DeviceOps()
        if kind == "gemm":
            s["weights"] = s["dev"].i8_weights(s["w"], s["w_scale"])
            s["ws"] = s["dev"].i8_gemm_workspace(s["weights"], T)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return {"quantize": _quantize, "norm": _norm, "silu": _silu, "gemm": _gemm}[s["case"]["kind"]](s)


def _to_codes(s, x):
    """(values, largest): the rows of x in 8-bit steps of their largest element, as multiples of one step."""
    most = x.abs().amax(-1, keepdim=True)
    inv = torch.where(most > 0, 127.0 / most, 0.0)
    return torch.round(x * inv), most


def _quantize(s):
    if own:
        s["dev"].i8_quantize(s["x"], q=s["q"], scale=s["scale"])
        s["dev"].i8_dequant(s["q"], s["scale"], out=s["out"])
        return [s["out"], s["scale"]]
    q, most = _to_codes(s, s["x"].float())
    scale = most / 127.0
    return [(q * scale).to(s["out"].dtype), scale[:, 0]]


def _norm(s):
    res = s["res"]
    if own:
        s["dev"].i8_rms_norm(s["x"], s["w"], EPS, res=res, res_out=s["res_out"], q=s["q"], scale=s["scale"])
        s["dev"].i8_dequant(s["q"], s["scale"], out=s["out"])
        return [s["out"], s["scale"]] + ([] if res is None else [s["res_out"]])
    h = s["x"] if res is None else (s["x"].float() + res.float()).to(res.dtype)
    v = h.float()
    q, most = _to_codes(s, v * s["w"].float())           # the norm's factor is one number per row: it is in the scale
    scale = most * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) / 127.0
    return [(q * scale).to(s["out"].dtype), scale[:, 0]] + ([] if res is None else [h])


def _silu(s):
    n = s["case"]["n"]
    gate, up = s["x"][:, :n], s["x"][:, n:]
    if own:
        s["dev"].i8_silu_mul(gate, up, q=s["q"], scale=s["scale"])
        s["dev"].i8_dequant(s["q"], s["scale"], out=s["out"])
        return [s["out"], s["scale"]]
    gate = gate.float()
    q, most = _to_codes(s, gate / (1.0 + torch.exp(-gate)) * up.float())
    scale = most / 127.0
    return [(q * scale).to(s["out"].dtype), scale[:, 0]]


def _gemm(s):
    if own:
        return [s["dev"].i8_gemm(s["weights"], s["x"], s["x_scale"], bias=s["bias"], out=s["out"], ws=s["ws"])]
    y = (s["x"].float() @ s["w"].float().T) * s["x_scale"][:, None] * s["w_scale"]
    return [(y if s["bias"] is None else y + s["bias"]).to(s["out"].dtype)]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "none": 0}
    T = case["T"]
    if case["kind"] == "gemm":
        rows, cols = case["rows"], case["cols"]
        return {"bytes": T * cols + rows * cols + T * rows * size[case["out"]] + 4 * T + 4 * rows * (1 + case["bias"]),
                "flops": 2 * T * rows * cols}
    n = case["n"]
    out = 3 * T * n + 4 * T                                # the codes, the values they stand for, the scales
    if case["kind"] == "quantize":
        return {"bytes": T * n * size[case["type"]] + out, "flops": 4 * T * n}
    if case["kind"] == "norm":
        return {"bytes": T * n * (size[case["type"]] + 2 * size[case["res"]]) + n * size[case["w"]] + out, "flops": 8 * T * n}
    return {"bytes": 2 * T * n * size[case["type"]] + out, "flops": 9 * T * n}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f64 = lambda t: t.to(torch.float64)  # noqa: E731
    if case["kind"] == "gemm":
        out = torch.empty((case["T"], case["rows"]), dtype=torch.float64, device="cuda")
        x = f64(s["x"])
        for r in range(0, case["rows"], 4096):             # every sum of products is a whole number below 2^53
            at = slice(r, r + 4096)
            out[:, at] = torch.matmul(x, f64(s["w"][at]).transpose(0, 1).contiguous())
            out[:, at] *= f64(s["x_scale"])[:, None] * f64(s["w_scale"][at])[None, :]
            if case["bias"]:
                out[:, at] += f64(s["bias"][at])
        return [out]
    x = f64(s["x"])
    more = []
    if case["kind"] == "silu":
        gate, up = x.split(case["n"], dim=1)
        y = gate * torch.sigmoid(gate) * up
    elif case["kind"] == "norm":
        if s["res"] is not None:
            more = [x + f64(s["res"])]
            x = f64(more[0].to(s["res"].dtype))            # the norm is of the stored sum
        y = x / torch.sqrt((x ** 2).sum(1, keepdim=True) / case["n"] + EPS) * f64(s["w"])
    else:
        y = x
    top = torch.maximum(y.max(1).values, -y.min(1).values)
    step = torch.where(top > 0, top / 127, torch.ones_like(top))[:, None]
    return [torch.round(y / step) * step, top / 127] + more
