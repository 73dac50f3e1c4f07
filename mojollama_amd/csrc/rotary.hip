// rotary.hip — rotary positions of new tokens' q and k heads, and the store of
// k and v into a paged 16- or 8-bit cache.
#include <math.h>
#include <type_traits>
#include "paged.h"

namespace {

struct rot_args {
    const void *q, *k, *v;
    long q_ld, k_ld, v_ld, qo_ld, ko_ld;
    void *q_out, *k_out;
    const double *freqs;
    float mscale;
    int layout, r, in_type, out_type;
    bool in_wide, out_wide;       // every head's rows are multiples of 16 bytes
    const int *pos, *seqs, *rows;
    int T, NH, NKH, HD;
    bool store;
    mllm_paged_kv kv;
};

// Element e (8 of them from 8u on) of a head after rotation, in T = float or double.  The
// pair's other element is read again from global memory (it is in L1): a lane then needs no
// other lane's registers whatever the rotated width is.
template <class T>
__device__ __forceinline__ void rotate8(const rot_args &a, const void *p, long at, int e0, const T *cs, T (&o)[8])
{
    float x[8];
    load8(p, at + e0, a.in_type, a.in_wide, x);
    const int r = a.r, h = r >> 1;
    if (e0 >= r) {
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = (T)x[i];
        return;
    }
    const T *c = cs, *s = cs + h;
    if (a.layout == MLLM_ROPE_PAIRS) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const int j = (e0 + i) >> 1;
            const bool in = e0 + i < r;
            const T co = in ? c[j] : (T)1, si = in ? s[j] : (T)0;
            o[i] = (T)x[i] * co - (T)x[i + 1] * si;
            o[i + 1] = (T)x[i + 1] * co + (T)x[i] * si;
            if (!in) { o[i] = (T)x[i]; o[i + 1] = (T)x[i + 1]; }
        }
        return;
    }
    float y[8];
    if (h % 8 == 0) {
        load8(p, at + (e0 < h ? e0 + h : e0 - h), a.in_type, a.in_wide, y);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int e = e0 + i;
            const long m = at + (e >= r ? e : e < h ? e + h : e - h);
            y[i] = a.in_type == MLLM_F32 ? ((const float *)p)[m]
                 : a.in_type == MLLM_BF16 ? (float)((const __bf16 *)p)[m] : (float)((const _Float16 *)p)[m];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int e = e0 + i;
        const bool lo = e < h;
        if (e >= r) {
            o[i] = (T)x[i];
        } else {
            const int j = lo ? e : e - h;
            o[i] = lo ? (T)x[i] * c[j] - (T)y[i] * s[j] : (T)x[i] * c[j] + (T)y[i] * s[j];
        }
    }
}

// x rounded to odd in fp32: a second rounding to at most 22 bits then gives what one rounding from
// 64 bits gives.
__device__ __forceinline__ float to_odd(double x)
{
    float f = (float)x;
    if ((double)f != x && f - f == 0.0f) {
        uint32_t b = __float_as_uint(f);
        if (fabs((double)f) > fabs(x)) b -= 1;
        f = __uint_as_float(b | 1);
    }
    return f;
}

// A row of LPR lanes, eight elements each, into an E4M3 cache.
__device__ __forceinline__ void store_e4m3(uint8_t *dst, uint8_t *exp, const double (&x)[8], int u, int lpr, int HD)
{
    double m = 0.0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        m = fmax(m, fabs(x[i]));
        bad |= !(fabs(x[i]) < INFINITY);
    }
    for (int d = lpr >> 1; d > 0; d >>= 1) {
        m = fmax(m, __shfl_xor(m, d, 64));
        bad |= (bool)__shfl_xor((int)bad, d, 64);
    }
    int e = 0;
    if (!bad && m > 0.0) {
        const double f = frexp(m, &e);          // m = f 2^e, 448 = 0.875 * 2^9
        e = f <= 0.875 ? e - 9 : e - 8;
        e = e < -100 ? -100 : e > 100 ? 100 : e;
    }
    if (8 * u >= HD) return;
    const double inv = ldexp(1.0, -e);
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float f = to_odd(x[4 * h + i] * inv);         // infinite where x leaves fp32's range
            const float g = f > 448.0f ? 448.0f : f < -448.0f ? -448.0f : f;
            y[i] = fabs(x[4 * h + i]) < INFINITY ? g : NAN;
        }
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
    }
    *(uint2 *)(dst + 8 * u) = make_uint2(w[0], w[1]);
    if (u == 0) *exp = (uint8_t)(e + 127);
}

// One token per workgroup: its cosines and sines are formed once and serve all heads from LDS, and the rows
// pass through registers once.  Bound by memory in large calls (4096 tokens, 32/8 heads of 128 in 16 bits: 22.9 us,
// 4.4 TB/s), by the launch in small ones (8 tokens: 6 us, of which the chain position - angle - LDS is half).
// A head's row is LPR lanes (a power of two) of eight elements.
// q heads, then k heads, then v heads.
// PAST: stores go past the caches.
template <bool E4M3, bool PAST>
__global__ __launch_bounds__(256) void k_rotary(rot_args a, int lpr_log)
{
    using T = typename std::conditional<E4M3, double, float>::type;
    __shared__ float cs[256];
    __shared__ double csd[E4M3 ? 256 : 1];
    const int t = blockIdx.x, h = a.r >> 1;
    const int pos = a.pos[t];
    if (pos < 0) return;
    for (int j = threadIdx.x; j < h; j += 256) {
        // whole turns are taken off in 64 bits: far positions keep their angle
        const double turns = (double)pos * a.freqs[j] * 0.15915494309189533577;
        const double f = 2.0 * (turns - rint(turns));
        if constexpr (E4M3) {
            double s, c;
            sincospi(f, &s, &c);
            csd[j] = c * a.mscale;
            csd[h + j] = s * a.mscale;
            cs[j] = (float)csd[j];
            cs[h + j] = (float)csd[h + j];
        } else {
            float s, c;
            sincospif((float)f, &s, &c);
            cs[j] = c * a.mscale;
            cs[h + j] = s * a.mscale;
        }
    }
    __syncthreads();
    const int lpr = 1 << lpr_log, u = threadIdx.x & (lpr - 1), HD = a.HD;
    const int nq = a.q ? a.NH : 0, nk = a.k ? a.NKH : 0, n = nq + (a.store ? 2 : 1) * nk;
    int page = -1, row = 0;
    if (a.store) {
        const int seq = a.seqs ? a.seqs[t] : t;
        row = a.rows ? a.rows[t] : pos;
        if (seq >= 0 && seq < a.kv.n_seqs && row >= 0) page = pk_page(a.kv, seq, row);
    }
    for (int i = threadIdx.x >> lpr_log; i < n; i += 256 >> lpr_log) {
        const int e0 = 8 * u;
        const bool real = e0 < HD;            // HD / 8 is no power of two: the last lanes of a row idle
        const int kind = i < nq ? 0 : i < nq + nk ? 1 : 2, j = kind == 0 ? i : kind == 1 ? i - nq : i - nq - nk;
        const long at = kind == 0 ? t * a.q_ld + (long)j * HD : kind == 1 ? t * a.k_ld + (long)j * HD
                                                                        : t * a.v_ld + (long)j * HD;
        if (kind == 0) {
            if (!real) continue;
            float o[8];
            rotate8<float>(a, a.q, at, e0, cs, o);
            store8<PAST>(a.q_out, t * a.qo_ld + (long)j * HD + e0, a.out_type, a.out_wide, o);
            continue;
        }
        T o[8] = {};
        if (real) {
            if (kind == 1) {
                if constexpr (E4M3) rotate8<T>(a, a.k, at, e0, csd, o);
                else rotate8<T>(a, a.k, at, e0, cs, o);
            } else {
                float x[8];
                load8(a.v, at + e0, a.in_type, a.in_wide, x);
#pragma unroll
                for (int c = 0; c < 8; c++) o[c] = (T)x[c];
            }
        }
        if (kind == 1 && a.k_out && real) {
            float f[8];
#pragma unroll
            for (int c = 0; c < 8; c++) f[c] = (float)o[c];
            store8<PAST>(a.k_out, t * a.ko_ld + (long)j * HD + e0, a.out_type, a.out_wide, f);
        }
        if (page < 0) continue;               // the whole workgroup
        const long to = page * a.kv.page_stride + row * a.kv.row_stride + j * a.kv.head_stride;
        void *base = kind == 1 ? a.kv.k : a.kv.v;
        if constexpr (E4M3) {
            uint8_t *exp = (kind == 1 ? a.kv.k_exp : a.kv.v_exp) + ((long)page * a.NKH + j) * a.kv.page_size + row;
            store_e4m3((uint8_t *)base + to, exp, o, u, lpr, HD);
        } else if (real) {
            store8<PAST>(base, to + e0, a.kv.type, true, o);
        }
    }
}

} // namespace

extern "C" {

MLLM_API int mllm_rotary_freqs(int scaling, int rope_dim, double base, double factor, double ctx, double beta_fast,
                               double beta_slow, double *freqs, float *mscale)
{
    const int r = rope_dim;
    if (r < 0 || r % 2 || r > 256 || (r && !freqs) || !mscale || scaling < MLLM_ROPE_NONE || scaling > MLLM_ROPE_BANDS ||
        !(base > 1.0) || (scaling != MLLM_ROPE_NONE && !(factor > 0.0)) ||
        (scaling >= MLLM_ROPE_YARN && !(ctx > 0.0)) || (scaling == MLLM_ROPE_NTK && r == 2))
        return pk_fail("mllm_rotary_freqs", "rope_dim is even and at most 256 (above 2 for NTK), base above 1, factor and "
                                            "ctx positive where the scaling uses them");
    if (beta_fast <= 0.0) beta_fast = scaling == MLLM_ROPE_YARN ? 32.0 : 4.0;
    if (beta_slow <= 0.0) beta_slow = 1.0;
    if (scaling >= MLLM_ROPE_YARN && !(beta_fast > beta_slow))
        return pk_fail("mllm_rotary_freqs", "beta_fast is above beta_slow");
    *mscale = 1.0f;
    const double two_pi = 6.283185307179586476925286766559;
    double lo = 0.0, hi = 0.0;
    if (scaling == MLLM_ROPE_NTK) base *= pow(factor, (double)r / (r - 2));
    if (scaling == MLLM_ROPE_YARN) {
        // the pair that turns beta times in ctx positions: base^(-2j/r) ctx = 2 pi beta
        lo = floor(r * log(ctx / (beta_fast * two_pi)) / (2.0 * log(base)));
        hi = ceil(r * log(ctx / (beta_slow * two_pi)) / (2.0 * log(base)));
        lo = lo < 0.0 ? 0.0 : lo;
        hi = hi > r - 1 ? r - 1 : hi;
        if (factor > 1.0) *mscale = (float)(0.1 * log(factor) + 1.0);
    }
    for (int j = 0; j < r / 2; j++) {
        const double w = pow(base, -2.0 * j / r);
        double s = 0.0;                        // 0: as it is, 1: divided by factor
        if (scaling == MLLM_ROPE_LINEAR) s = 1.0;
        if (scaling == MLLM_ROPE_YARN) s = (j - lo) / (hi > lo ? hi - lo : 0.001);
        if (scaling == MLLM_ROPE_BANDS) s = 1.0 - (ctx * w / two_pi - beta_slow) / (beta_fast - beta_slow);
        s = s < 0.0 ? 0.0 : s > 1.0 ? 1.0 : s;
        freqs[j] = s == 0.0 ? w : w / factor * s + w * (1.0 - s);
    }
    return 0;
}

MLLM_API int mllm_rotary_append(const mllm_rotary *rot, int in_type, const void *q, long q_ld, const void *k, long k_ld,
                                const void *v, long v_ld, const int *pos, int T, int NH, int NKH, int HD, int out_type,
                                void *q_out, long q_out_ld, void *k_out, long k_out_ld, const mllm_paged_kv *kv,
                                const int *seqs, const int *rows, void *stream)
{
    const char *who = "mllm_rotary_append";
    auto real = [](int t) { return t == MLLM_F32 || t == MLLM_F16 || t == MLLM_BF16; };
    if (!rot || !pos || T < 0 || HD <= 0 || HD > 256 || HD % 16 || !real(in_type) || !real(out_type))
        return pk_fail(who, "head_dim is a multiple of 16 up to 256, the types F32, F16 or BF16");
    if (rot->rope_dim < 0 || rot->rope_dim % 2 || rot->rope_dim > HD || (rot->rope_dim && !rot->freqs) ||
        (rot->layout != MLLM_ROPE_HALF && rot->layout != MLLM_ROPE_PAIRS))
        return pk_fail(who, "rope_dim is even and at most head_dim, with freqs, layout HALF or PAIRS");
    if (q && (!q_out || NH <= 0 || q_ld < (long)NH * HD || q_out_ld < (long)NH * HD))
        return pk_fail(who, "q needs q_out, NH and row strides of at least NH * HD");
    if (k && (NKH <= 0 || k_ld < (long)NKH * HD || (k_out && k_out_ld < (long)NKH * HD)))
        return pk_fail(who, "k needs NKH and row strides of at least NKH * HD");
    if (kv) {
        if (const char *why = pk_refusal(kv)) return pk_fail(who, why);
        if (!k || !v || kv->n_kv_head != NKH || kv->head_dim != HD || v_ld < (long)NKH * HD)
            return pk_fail(who, "a cache takes k and v of its own heads and head_dim, v_ld at least NKH * HD");
        if (!seqs && T > kv->n_seqs) return pk_fail(who, "without seqs, T is at most the cache's n_seqs");
    } else if (k && !k_out) {
        return pk_fail(who, "k without a cache needs k_out");
    }
    if (q && q == q_out && (in_type != out_type || q_ld != q_out_ld))
        return pk_fail(who, "q_out may be q only in its type and stride");
    if (k && k == k_out && (in_type != out_type || k_ld != k_out_ld))
        return pk_fail(who, "k_out may be k only in its type and stride");
    if (!T || (!q && !k)) return 0;
    rot_args a{};
    a.q = q; a.k = k; a.v = v; a.q_ld = q_ld; a.k_ld = k_ld; a.v_ld = v_ld; a.qo_ld = q_out_ld; a.ko_ld = k_out_ld;
    a.q_out = q_out; a.k_out = k_out; a.freqs = rot->freqs; a.mscale = rot->mscale; a.layout = rot->layout;
    a.r = rot->rope_dim; a.in_type = in_type; a.out_type = out_type; a.pos = pos; a.seqs = seqs; a.rows = rows;
    a.T = T; a.NH = NH; a.NKH = NKH; a.HD = HD; a.store = kv != nullptr;
    if (kv) a.kv = *kv;
    const long ib = pk_size(in_type), ob = pk_size(out_type);
    auto al = [](const void *p, long ld, long b) { return !p || !(((uintptr_t)p | (uintptr_t)(ld * b)) & 15); };
    a.in_wide = al(q, q_ld, ib) && al(k, k_ld, ib) && (!kv || al(v, v_ld, ib));
    a.out_wide = al(q ? q_out : nullptr, q_out_ld, ob) && al(k ? k_out : nullptr, k_out_ld, ob);
    // What is written past the size of the L2s is not read from there again: stores past them leave the reads
    // their lines (4096 tokens, 32/8 heads of 128 in 16 bits, 101 MB in all: 31.6 -> 23.9 us).  Below it the next
    // kernel finds q and the new rows in L2.
    const long bytes = T * ((long)(q ? NH : 0) * HD * ob + (k ? 2l * NKH * HD * 2 : 0));
    const bool past = bytes > 32l << 20;
    int lpr_log = 1;
    while ((8 << lpr_log) < HD) lpr_log++;
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(T), dim3(256), 0, st, a, lpr_log); };
    if (kv && kv->type == MLLM_E4M3) past ? go(k_rotary<true, true>) : go(k_rotary<true, false>);
    else past ? go(k_rotary<false, true>) : go(k_rotary<false, false>);
    return hipGetLastError() == hipSuccess ? 0 : pk_fail(who, "the launch failed");
}

} // extern "C"
