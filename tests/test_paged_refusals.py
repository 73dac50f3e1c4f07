"""What the operators over a paged cache refuse, before any launch, and the
frequencies of rotary positions (host code; no GPU)."""
import ctypes
import math

import pytest

from mojollama_amd import kernels as K

P = 4096   # an address that is checked and never read


@pytest.fixture(scope="module")
def so():
    import os
    if not os.path.exists(K.LIB_PATH):
        K.build()
    return K.load_kernels()


def kv(**change):
    v = K.PagedKV(K.T_BF16, 2, 64, 10, 16, P, P, None, None, 16 * 128, 128, 64, P, 3, 4, 4)
    for name, x in change.items():
        setattr(v, name, x)
    return v


BAD_KV = [dict(type=K.T_F32), dict(type=7), dict(type=K.T_E4M3), dict(head_dim=72), dict(head_dim=0), dict(head_dim=272),
          dict(n_kv_head=0), dict(page_size=0), dict(n_pages=0), dict(n_seqs=0), dict(max_blocks=0), dict(table_ld=3),
          dict(k=None), dict(v=P + 8), dict(row_stride=132), dict(page_stride=-16), dict(head_stride=4), dict(tables=None)]


def decode(so, v, **c):
    a = dict(q_type=K.T_BF16, q=P, q_ld=512, seqs=None, lens=P, max_len=60, B=3, NH=8, scale=0.1, window=0, out_type=K.T_BF16, out=P,
             out_ld=512, ws=P, n=1 << 40) | c
    return so.mllm_paged_attn_decode(v, a["q_type"], a["q"], a["q_ld"], a["seqs"], a["lens"], a["max_len"], a["B"], a["NH"],
                                     a["scale"], a["window"], None, a["out_type"], a["out"], a["out_ld"], a["ws"], a["n"], None)


def prompt(so, v, **c):
    a = dict(q_type=K.T_BF16, q=P, q_ld=512, seqs=None, starts=P, lens=P, max_len=60, T=9, B=3, NH=8, scale=0.1, window=0,
             out_type=K.T_BF16, out=P, out_ld=512, ws=P, n=1 << 40) | c
    return so.mllm_paged_attn_prompt(v, a["q_type"], a["q"], a["q_ld"], a["seqs"], a["starts"], a["lens"], a["max_len"],
                                     a["T"], a["B"], a["NH"], a["scale"], a["window"], None, a["out_type"], a["out"], a["out_ld"],
                                     a["ws"], a["n"], None)


@pytest.mark.parametrize("change", BAD_KV)
def test_views(so, change):
    v = kv(**change)
    assert decode(so, v) == -1 and prompt(so, v) == -1
    assert so.mllm_paged_attn_workspace_size(v, 3, 3, 8, 60, 0) == -1
    rot = K.Rotary(0, 0, None, 1.0)
    assert so.mllm_rotary_append(rot, K.T_F32, None, 0, P, 128, P, 128, P, 3, 0, v.n_kv_head, v.head_dim, K.T_F32, None, 0,
                                 None, 0, v, None, None, None) == -1
    assert so.mllm_last_error().startswith(b"mllm_rotary_append")


@pytest.mark.parametrize("c", [dict(q_type=K.T_F16), dict(out_type=K.T_F16), dict(q_type=K.T_E4M3), dict(q=None),
                               dict(out=None), dict(lens=None), dict(q=P + 2), dict(q_ld=504), dict(q_ld=516), dict(out_ld=500),
                               dict(NH=9), dict(NH=0), dict(B=-1), dict(B=4), dict(max_len=-1),
                               dict(max_len=(1 << 30) + 1), dict(window=-1), dict(scale=float("nan")),
                               dict(scale=float("inf")), dict(ws=None),
                               dict(n=0)])
def test_attention(so, c):
    assert decode(so, kv(), **c) == -1 and so.mllm_last_error().startswith(b"mllm_paged_attn_decode")
    assert prompt(so, kv(), **c) == -1 and so.mllm_last_error().startswith(b"mllm_paged_attn_prompt")


def test_attention_of_nothing(so):
    """No sequences or no tokens: nothing is launched."""
    assert decode(so, kv(), B=0) == 0
    assert prompt(so, kv(), T=0) == 0
    assert prompt(so, kv(), starts=None) == -1 and prompt(so, kv(), T=-1) == -1


@pytest.mark.parametrize("cache", [K.T_BF16, K.T_F16])
def test_workspace_never_decreases(so, cache):
    """A workspace for a length, number of sequences and of tokens serves every smaller call."""
    for NKH, NH, HD in ((8, 64, 64), (1, 1, 16), (4, 28, 128), (2, 6, 256)):
        v = kv(type=cache, n_kv_head=NKH, head_dim=HD, page_stride=16 * NKH * HD, row_stride=NKH * HD, head_stride=HD)
        f = lambda T, B, n, w: so.mllm_paged_attn_workspace_size(v, T, B, NH, n, w)  # noqa: E731
        for w in (0, 100):
            for B in (1, 3, 64):
                sizes = [f(B, B, n, w) for n in (0, 1, 64, 65, 1000, 4097, 100000, 1 << 22, 1 << 30)]
                assert sizes == sorted(sizes) and sizes[0] > 0
            for n in (1, 5000):
                sizes = [f(B, B, n, w) for B in range(1, 700, 7)]
                assert sizes == sorted(sizes)
                sizes = [f(T, min(T, 3), n, w) for T in range(1, 3000, 11)]
                assert sizes == sorted(sizes)
                sizes = [f(200, B, n, w) for B in range(1, 200)]
                assert sizes == sorted(sizes)


def rotary(so, **c):
    a = dict(layout=0, rope_dim=64, freqs=P, it=K.T_F32, q=P, q_ld=512, k=P, k_ld=128, v=P, v_ld=128, pos=P, T=3, NH=8, NKH=2,
             HD=64, ot=K.T_BF16, qo=P, qo_ld=512, ko=None, ko_ld=0, kv=kv(), seqs=None) | c
    rot = K.Rotary(a["layout"], a["rope_dim"], a["freqs"], 1.0)
    return so.mllm_rotary_append(rot, a["it"], a["q"], a["q_ld"], a["k"], a["k_ld"], a["v"], a["v_ld"], a["pos"], a["T"], a["NH"],
                                 a["NKH"], a["HD"], a["ot"], a["qo"], a["qo_ld"], a["ko"], a["ko_ld"], a["kv"], a["seqs"],
                                 None, None)


@pytest.mark.parametrize("c", [dict(layout=2), dict(rope_dim=63), dict(rope_dim=66), dict(rope_dim=-2), dict(freqs=None),
                               dict(it=K.T_E4M3), dict(ot=K.T_E4M3), dict(q_ld=511), dict(qo_ld=511), dict(k_ld=127),
                               dict(v_ld=127), dict(pos=None), dict(T=-1), dict(T=4), dict(HD=72), dict(NH=0), dict(NKH=3),
                               dict(qo=None), dict(k=None), dict(v=None), dict(kv=None), dict(ko=P, ko_ld=100),
                               dict(q=P, qo=P), dict(q=P, qo=P, ot=K.T_F32, qo_ld=520)])
def test_rotary(so, c):
    base = dict(qo=2 * P)
    assert rotary(so, **(base | c)) == -1 and so.mllm_last_error().startswith(b"mllm_rotary_append")


def test_rotary_of_nothing(so):
    assert rotary(so, T=0, qo=2 * P) == 0
    assert rotary(so, q=None, k=None, v=None, kv=None) == 0


def pages(so):
    return K.PageMap(P, 4, 5, 5, P, 20, 8), (K.PagePlane * 1)(K.PagePlane(P, 64, 1280, 2))


@pytest.mark.parametrize("c", [dict(tables=None), dict(refs=None), dict(n_seqs=0), dict(max_blocks=0), dict(table_ld=4),
                               dict(n_pages=0), dict(page_size=0)])
def test_page_maps(so, c):
    m, planes = pages(so)
    for name, x in c.items():
        setattr(m, name, x)
    big = 1 << 30
    assert so.mllm_pages_workspace_size(m, 3) == -1
    assert so.mllm_pages_reserve(m, 1, P, P, P, P, big, None) == -1
    assert so.mllm_pages_free(m, 1, P, None, None) == -1
    assert so.mllm_pages_fork(m, planes, 1, 1, P, P, P, P, P, big, None) == -1
    assert so.mllm_pages_compact(m, planes, 1, P, P, big, None) == -1


def test_page_calls(so):
    m, planes = pages(so)
    big = 1 << 30
    for bad in ((-1, P, P, P, P, big), (1, None, P, P, P, big), (1, P, None, P, P, big), (1, P, P, None, P, big),
                (1, P, P, P, None, big), (1, P, P, P, P, 64)):
        assert so.mllm_pages_reserve(m, *bad, None) == -1
    assert so.mllm_pages_free(m, 1, None, None, None) == -1 and so.mllm_pages_free(m, -1, P, None, None) == -1
    assert so.mllm_pages_free(m, 0, None, None, None) == 0
    for bad in ((1, None, P, P, P, P, big), (1, P, None, P, P, P, big), (1, P, P, None, P, P, big), (1, P, P, P, None, P, big),
                (70000, P, P, P, P, P, big), (1, P, P, P, P, P, 64)):
        assert so.mllm_pages_fork(m, planes, 1, *bad, None) == -1
    assert so.mllm_pages_fork(m, planes, 9, 1, P, P, P, P, P, big, None) == -1
    assert so.mllm_pages_compact(m, planes, 1, None, P, big, None) == -1
    for name, x in (("base", None), ("page_bytes", 0), ("n_layers", 0), ("layer_bytes", 1279)):
        p = (K.PagePlane * 1)(K.PagePlane(P, 64, 1280, 2))
        setattr(p[0], name, x)
        assert so.mllm_pages_copy(p, 1, 20, 1, P, P, None) == -1
        assert so.mllm_pages_compact(m, p, 1, P, P, big, None) == -1
    assert so.mllm_pages_copy(planes, 1, 20, 1, None, P, None) == -1
    assert so.mllm_pages_copy(planes, 1, 20, 0, None, None, None) == 0


# ------------------------------------------------------------------ frequencies
def freqs(so, scaling, r, base=10000.0, factor=8.0, ctx=2048.0, fast=0.0, slow=0.0):
    f, m = (ctypes.c_double * (r // 2))(), ctypes.c_float()
    assert so.mllm_rotary_freqs(scaling, r, base, factor, ctx, fast, slow, f, ctypes.byref(m)) == 0
    return list(f), m.value


@pytest.mark.parametrize("r,base", [(64, 10000.0), (128, 500000.0), (2, 10000.0), (20, 150000.0)])
def test_frequencies(so, r, base):
    plain = [base ** (-2 * j / r) for j in range(r // 2)]
    close = lambda a, b: all(abs(x - y) <= 1e-14 * abs(y) for x, y in zip(a, b)) and len(a) == len(b)  # noqa: E731
    f, m = freqs(so, K.ROPE_NONE, r, base)
    assert close(f, plain) and m == 1.0
    assert close(freqs(so, K.ROPE_LINEAR, r, base)[0], [w / 8 for w in plain])
    if r > 2:
        f, _ = freqs(so, K.ROPE_NTK, r, base)
        # the first pair keeps its frequency, the last one's is divided by the factor
        assert f[0] == 1.0 and math.isclose(f[-1], plain[-1] / 8, rel_tol=1e-12)
    f, m = freqs(so, K.ROPE_YARN, r, base)
    assert math.isclose(m, 0.1 * math.log(8) + 1, rel_tol=1e-6)
    for x, w in zip(f, plain):
        turns = 2048 * w / (2 * math.pi)
        assert w / 8 * (1 - 1e-12) <= x <= w
        if turns < 0.9 and w < 0.5:      # one pair's step below beta_slow: the ramp's end is rounded to whole pairs
            j = plain.index(w)
            if j >= math.ceil(r * math.log(2048 / (2 * math.pi)) / (2 * math.log(base))):
                assert math.isclose(x, w / 8, rel_tol=1e-12)
    f, m = freqs(so, K.ROPE_BANDS, r, base)
    for x, w in zip(f, plain):
        s = min(max((2048 * w / (2 * math.pi) - 1) / 3, 0), 1)
        assert math.isclose(x, w / 8 * (1 - s) + w * s, rel_tol=1e-12)
    assert m == 1.0


@pytest.mark.parametrize("a", [(0, 3, 1e4, 1, 1), (0, 258, 1e4, 1, 1), (5, 64, 1e4, 1, 1), (-1, 64, 1e4, 1, 1), (0, 64, 1, 1, 1),
                               (1, 64, 1e4, 0, 1), (3, 64, 1e4, 8, 0), (2, 2, 1e4, 8, 1)])
def test_frequency_refusals(so, a):
    f, m = (ctypes.c_double * 200)(), ctypes.c_float()
    assert so.mllm_rotary_freqs(a[0], a[1], a[2], a[3], a[4], 0.0, 0.0, f, ctypes.byref(m)) == -1
    assert so.mllm_rotary_freqs(3, 64, 1e4, 8.0, 2048.0, 1.0, 2.0, f, ctypes.byref(m)) == -1
