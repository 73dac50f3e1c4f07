// i8_rows.hip — rows into 8-bit integers with a scale each: as they are, after the residual addition and
// root-mean-square norm, and after silu(gate) * up; back to values; and weights into the packed layout.
//
// y[i] of a row, its largest |y| and (norm) the sum of squares are formed in one pass over memory and stay
// in registers; the codes are rounded from there: memory is read and written once, which is what bounds
// these kernels where there are many rows (norm of 8192 x 4096 with residual, 16 bits: 45 to 47 us in a loop of launches,
// 5.0 to 5.2 TB/s, 50 in a profiler's trace; silu of 4096 x 11264: 50 to 55 us, 4.2 to 4.7 TB/s, 57 in the trace, its
// exponentials beside it; the card copies 4 GiB at 4.7).  Rows wider than 16384 elements take one workgroup a CU, whose
// barrier nothing hides (silu of 4096 x 18944: 111 us, 3.5 TB/s).  A few rows take the launch and one memory round trip (3
// to 5 us).  The norm's factor 1 / sqrt(mean + eps) is one number per row: it enters the scale alone, and the codes do not
// wait for it.  A row of a norm whose products w h, squares or values would leave fp32 though y does not is formed again in
// 64 bits, behind the rest (far_norm).
#include <algorithm>
#include <type_traits>
#include "i8.h"

namespace {

// N bytes from an address of any alignment (the hardware's unaligned access).
template <int N> struct raw { uint32_t w[N / 4]; };
template <int N> __device__ __forceinline__ raw<N> ld_any(const void *p)
{
    raw<N> r;
    __builtin_memcpy(&r, p, N);
    return r;
}

// Eight consecutive elements, W bytes each, as they lie in memory; those from `left` on are zeros.
template <int W> __device__ __forceinline__ raw<8 * W> ld8(const void *p, long at, int left)
{
    if (left >= 8) return ld_any<8 * W>((const char *)p + at * W);
    raw<8 * W> r{};
    for (int i = 0; i < left; i++) {
        if constexpr (W == 4) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j == i) r.w[j] = ((const uint32_t *)p)[at + i];
        } else {
            const uint32_t h = ((const uint16_t *)p)[at + i];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j == i) r.w[j >> 1] |= h << (16 * (j & 1));
        }
    }
    return r;
}
constexpr int size_of(int type) { return type == MLLM_F32 ? 4 : 2; }
template <int TYPE> using raw8 = raw<8 * size_of(TYPE)>;
template <int TYPE> __device__ __forceinline__ void to_f32(const raw8<TYPE> &r, float (&x)[8])
{
    if constexpr (TYPE == MLLM_F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __uint_as_float(r.w[i]);
    } else if constexpr (TYPE == MLLM_BF16) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(r.w[i] << 16);
            x[2 * i + 1] = __uint_as_float(r.w[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f16x2 v = __builtin_bit_cast(f16x2, r.w[i]);
            x[2 * i] = (float)v.x;
            x[2 * i + 1] = (float)v.y;
        }
    }
}
template <int TYPE> __device__ __forceinline__ raw8<TYPE> from_f32(const float (&x)[8])
{
    raw8<TYPE> r;
    if constexpr (TYPE == MLLM_F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) r.w[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) r.w[i] = pack2<TYPE>(x[2 * i], x[2 * i + 1]);
    }
    return r;
}
template <int W> __device__ __forceinline__ void st8(void *p, long at, int left, const raw<8 * W> &r)
{
    if (left >= 8) {
        __builtin_memcpy((char *)p + at * W, &r, 8 * W);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < left) {
            if constexpr (W == 4) ((uint32_t *)p)[at + i] = r.w[i];
            else ((uint16_t *)p)[at + i] = (uint16_t)(r.w[i >> 1] >> (16 * (i & 1)));
        }
}

// The largest |y|, gathered as bits: of the positive numbers as signed, of the negative as unsigned integers (one
// instruction for two elements each, and infinities and NaNs come out on top).
struct top {
    int pos = 0;
    uint32_t neg = 0;
    __device__ __forceinline__ void add(const float (&y)[8])
    {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            pos = max(max(pos, __float_as_int(y[i])), __float_as_int(y[i + 1]));
            neg = max(max(neg, __float_as_uint(y[i])), __float_as_uint(y[i + 1]));
        }
    }
    __device__ __forceinline__ uint32_t get() const { return max((uint32_t)pos, neg >> 31 ? neg & 0x7FFFFFFFu : 0u); }
};

// The step of a row: m is the largest |y| as fp32 bits, above or at those of infinity where the row holds an
// infinity or a NaN.  Codes are rint(y * pre * inv), inv = 127 * (1 / (most * pre)); the power of two pre keeps
// the reciprocal a normal number at either end of fp32.
struct row_step { float pre, inv, most; bool bad; };
__device__ __forceinline__ row_step step_of(uint32_t m)
{
    row_step s;
    s.bad = m >= 0x7F800000u;
    s.most = __uint_as_float(m);
    s.pre = s.most < 0x1p-100f ? 0x1p64f : s.most > 0x1p100f ? 0x1p-64f : 1.0f;
    s.inv = s.bad || m == 0 ? 0.0f : 1.0f / (s.most * s.pre) * 127.0f;
    return s;
}
// The nearest integer of f, |f| <= 127, is the low byte of f + 1.5 * 2^23 (ties to even, as the sum rounds).
__device__ __forceinline__ uint32_t four(float a, float b, float c, float d)
{
#pragma clang fp contract(off)
    constexpr float M = 12582912.0f;
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(b + M), __float_as_uint(a + M), 0x0C0C0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(d + M), __float_as_uint(c + M), 0x04000C0Cu);
    return lo | hi;
}
__device__ __forceinline__ uint2 codes(const float (&y)[8], const row_step &s)
{
#pragma clang fp contract(off)                               // the product rounds before the sum that makes it whole
    if (s.bad) return make_uint2(0, 0);
    float f[8];
    if (s.pre != 1.0f) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = y[i] * s.pre * s.inv;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = y[i] * s.inv;
    }
    return make_uint2(four(f[0], f[1], f[2], f[3]), four(f[4], f[5], f[6], f[7]));
}

// One of them, pre in y already.
__device__ __forceinline__ int8_t code(float y, float inv)
{
#pragma clang fp contract(off)
    return (int8_t)(__float_as_uint(y * inv + 12582912.0f) & 255);
}

// g / d, 1 <= d <= 2^100: the reciprocal with one Newton step, the quotient with its remainder taken back (the rounded
// quotient but for about one in a million, there its neighbour), in six instructions for the ten of a division that
// serves every number.
__device__ __forceinline__ float quotient(float g, float d)
{
    float r = __builtin_amdgcn_rcpf(d);
    r = fmaf(fmaf(-d, r, 1.0f), r, r);
    const float q = g * r;
    return fmaf(fmaf(-d, q, g), r, q);
}

enum { QUANTIZE, NORM, NORM_RES, SILU };

struct row_args {
    const void *x, *res, *w;       // SILU: gate, up
    void *res_out;
    long x_ld, res_ld, res_out_ld, q_ld;
    int8_t *q;
    float *scale;
    float eps;
    int w_type, T, n;
    long kb;                       // packed weights: blocks along K (q then is the packed matrix)
    int n_pad, T_pad;
};

template <int TYPE> __device__ __forceinline__ void times(const void *w, int e, int left, float (&y)[8])
{
    float f[8];
    to_f32<TYPE>(ld8<size_of(TYPE)>(w, e, left), f);
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] *= f[i];
}
__device__ __forceinline__ void weigh(const row_args &a, int e, int left, float (&y)[8])
{
    if (a.w_type == MLLM_F32) times<MLLM_F32>(a.w, e, left, y);
    else if (a.w_type == MLLM_BF16) times<MLLM_BF16>(a.w, e, left, y);
    else times<MLLM_F16>(a.w, e, left, y);
}

// y of elements e .. e + 7 of row t; sq gains the squares of h, bits the bits of h.
template <int KIND, int XT, int RT>
__device__ __forceinline__ void form(const row_args &a, const raw8<XT> &xr, const raw8<RT> &rr, int e, long t, int left,
                                     bool store, float (&y)[8], float &sq, uint32_t &bits)
{
    to_f32<XT>(xr, y);
    if constexpr (KIND == SILU) {
        float u[8], g[8], least = 0.0f;
        to_f32<RT>(rr, u);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            g[i] = y[i];
            least = fminf(least, g[i]);
            y[i] = quotient(g[i], 1.0f + expf(-g[i]));
        }
        // far below zero, where e^-g goes out of the quotient's reach, 1 + e^-g is e^-g: g h u h with h = e^(g / 2), in this
        // order, so that nothing leaves fp32 that the result does not
        if (__any(least < -69.0f)) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float h = expf(0.5f * g[i]);
                y[i] = g[i] < -69.0f ? g[i] * h * u[i] : y[i];
                u[i] = g[i] < -69.0f ? h : u[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] *= u[i];
    }
    if constexpr (KIND == NORM_RES) {
        float r[8];
        to_f32<RT>(rr, r);
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] += r[i];
        const raw8<RT> h = from_f32<RT>(y);
        if (store) st8<size_of(RT)>(a.res_out, t * a.res_out_ld + e, left, h);
        to_f32<RT>(h, y);
        // of the words as they are stored: four to a vector of 16-bit elements
#pragma unroll
        for (int i = 0; i < 2 * size_of(RT); i++) bits |= h.w[i];
    }
    if constexpr (KIND == NORM || KIND == NORM_RES) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            sq = fmaf(y[i], y[i], sq);
            if constexpr (KIND == NORM) bits |= __float_as_uint(y[i]);
        }
        weigh(a, e, left, y);
    }
}

template <int KIND, int XT, int RT>
__device__ __forceinline__ void load(const row_args &a, long t, int e, int left, raw8<XT> &x, raw8<RT> &r)
{
    x = ld8<size_of(XT)>(a.x, t * a.x_ld + e, left);
    if constexpr (KIND == NORM_RES || KIND == SILU) r = ld8<size_of(RT)>(a.res, t * a.res_ld + e, left);
}

// What a norm keeps in fp32 for a row: its largest |w h| (bits m) with room below and above for the smaller ones, for the
// factor and for y, and the mean square, beside eps.
__device__ __forceinline__ bool near_one(uint32_t m, float mean, float eps)
{
    return m >= __float_as_uint(0x1p-100f) && m < __float_as_uint(0x1p77f) && mean < 0x1p100f &&
           (mean >= 0x1p-100f || eps >= 0x1p-100f);
}

__device__ __forceinline__ float element(const void *p, int type, long at)
{
    if (type == MLLM_F32) return ((const float *)p)[at];
    return type == MLLM_BF16 ? __uint_as_float((uint32_t)((const uint16_t *)p)[at] << 16) : (float)((const _Float16 *)p)[at];
}

// f(e, h, w h) of the elements of a lane, one by one (few registers beside the row's), in 64 bits, where they are exact
// and in range.  h is the stored sum where there is one (x or res may be where it went): this lane's own.
template <int KIND, int XT, int RT, class F> __device__ __forceinline__ void far_each(const row_args &a, long t, int at, int L, F &&f)
{
    for (int b = 8 * at; b < a.n; b += 8 * L)
#pragma unroll 1
        for (int e = b; e < min(b + 8, a.n); e++) {
            const double h = KIND == NORM_RES ? element(a.res_out, RT, t * a.res_out_ld + e) : element(a.x, XT, t * a.x_ld + e);
            f(e, h, h * element(a.w, a.w_type, e));
        }
}

// A norm's row that is neither near_one nor of zeros.  The codes are those of w h times a power of two that takes the
// largest to between 1 and 2: of the same steps in fp32 as elsewhere, with nothing out of range.
template <int KIND, int XT, int RT>
__device__ void far_norm(const row_args &a, int per_wave)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = per_wave ? 1 : blockDim.x >> 6;
    const int L = per_wave ? 64 : blockDim.x, at = per_wave ? lane : threadIdx.x;
    const long t = per_wave ? i8_block() * (blockDim.x >> 6) + wave : i8_block();
    double most = 0.0, sum = 0.0;
    far_each<KIND, XT, RT>(a, t, at, L, [&](int, double h, double y) {
        sum += h * h;
        most = fmax(most, fabs(y) < INFINITY ? fabs(y) : INFINITY);                  // a NaN is as bad
    });
    for (int d = 32; d > 0; d >>= 1) {
        sum += __shfl_xor(sum, d, 64);
        most = fmax(most, __shfl_xor(most, d, 64));
    }
    if (waves > 1) {
        __shared__ double sums[16], mosts[16];
        if (lane == 0) {
            sums[wave] = sum;
            mosts[wave] = most;
        }
        __syncthreads();
        sum = most = 0.0;
        for (int i = 0; i < waves; i++) {
            sum += sums[i];
            most = fmax(most, mosts[i]);
        }
    }
    const double y_most = most == 0.0 ? 0.0 : most / sqrt(sum / a.n + (double)a.eps);
    const bool bad = !((float)y_most < INFINITY), none = bad || most == 0.0;
    if (at == 0) a.scale[t] = bad ? NAN : (float)(y_most / 127.0);
    const double pre = none ? 0.0 : ldexp(1.0, -ilogb(most));
    const float inv = none ? 0.0f : 1.0f / (float)(most * pre) * 127.0f;
    far_each<KIND, XT, RT>(a, t, at, L, [&](int e, double, double y) {
        a.q[t * a.q_ld + e] = none ? 0 : code((float)(y * pre), inv);
    });
}

// A row over L = blockDim.x lanes (PER_WAVE: a row per wave).  NV vectors of eight elements a lane stay in
// registers; longer rows are formed again for their codes.  PACK: codes go to the packed weight layout.
template <int KIND, int XT, int RT, int NV, bool PACK>
__global__ __launch_bounds__(NV > 4 ? 256 : 1024) void k_i8_rows(row_args a, int per_wave)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int L = per_wave ? 64 : blockDim.x, at = per_wave ? lane : threadIdx.x;
    const long t = per_wave ? i8_block() * waves + wave : i8_block();
    if (t >= (PACK ? a.T_pad : a.T)) return;             // a whole wave, or the whole workgroup
    const bool real = !PACK || t < a.T;
    float y[NV][8];
    raw8<XT> x[NV];
    raw8<RT> r[NV];
    float sq = 0.0f;
    uint32_t bits = 0;
    top mm;
    if (real) {
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int e = 8 * (v * L + at);
            if (e < a.n) load<KIND, XT, RT>(a, t, e, a.n - e, x[v], r[v]);
        }
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int e = 8 * (v * L + at);
#pragma unroll
            for (int i = 0; i < 8; i++) y[v][i] = 0.0f;
            if (e < a.n) form<KIND, XT, RT>(a, x[v], r[v], e, t, a.n - e, true, y[v], sq, bits);
            mm.add(y[v]);
        }
        for (int e = 8 * (NV * L + at); e < a.n; e += 8 * L) {
            float z[8];
            load<KIND, XT, RT>(a, t, e, a.n - e, x[0], r[0]);
            form<KIND, XT, RT>(a, x[0], r[0], e, t, a.n - e, true, z, sq, bits);
            mm.add(z);
        }
    }
    uint32_t m = mm.get();
    for (int d = 32; d > 0; d >>= 1) {
        m = max(m, (uint32_t)__shfl_xor((int)m, d, 64));
        if constexpr (KIND == NORM || KIND == NORM_RES) sq += __shfl_xor(sq, d, 64);
    }
    if (!per_wave && waves > 1) {
        __shared__ uint32_t ms[16];
        __shared__ float qs[16];
        if (lane == 0) {
            ms[wave] = m;
            qs[wave] = sq;
        }
        __syncthreads();
        m = 0;
        sq = 0.0f;
        for (int i = 0; i < waves; i++) {
            m = max(m, ms[i]);
            sq += qs[i];
        }
    }
    const row_step s = step_of(__builtin_amdgcn_readfirstlane(m));
    float step = s.most / 127.0f;
    // The row is not for fp32.  (Its type decides how the row's branch is compiled, and so the registers of all that is
    // before: a norm with residual of 8192 x 4096 takes 52 us with int, 47 with bool; of 2048 x 16384 56 with bool, 55
    // with int; one without of 4096 x 8192 32.8 with bool, 30 with int.)
    std::conditional_t<KIND == NORM || NV == 8, int, bool> away = false;
    if constexpr (KIND == NORM || KIND == NORM_RES) {
        const float mean = sq / (float)a.n;
        away = !near_one(m, mean, a.eps);
        if (m == 0) {                                    // padding, unless it is 0 in fp32 only
            away = __any((bits & (KIND == NORM || RT == MLLM_F32 ? 0x7FFFFFFFu : 0x7FFF7FFFu)) != 0);
            if (!per_wave && waves > 1) away = __syncthreads_or(away);
        }
        away = __builtin_amdgcn_readfirstlane(away);     // one branch for the row
        step = s.most * (1.0f / sqrtf(mean + a.eps)) / 127.0f;
    }
    if (at == 0 && real) a.scale[t] = s.bad ? NAN : m == 0 ? 0.0f : step;
    const int n = PACK ? a.n_pad : a.n;
    auto put = [&](int e, const float (&z)[8]) {
        const uint2 c = codes(z, s);
        if constexpr (PACK) {
            *(uint2 *)(a.q + i8_at(a.kb, (int)t, e)) = c;
        } else {
            int8_t *p = a.q + t * a.q_ld + e;
            if (a.n - e >= 8) {
                __builtin_memcpy(p, &c, 8);
            } else {
                for (int i = 0; i < a.n - e; i++) p[i] = (int8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
            }
        }
    };
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int e = 8 * (v * L + at);
        if (!real) {
#pragma unroll
            for (int i = 0; i < 8; i++) y[v][i] = 0.0f;
        }
        if (e < n) put(e, y[v]);
    }
    for (int e = 8 * (NV * L + at); e < n; e += 8 * L) {
        float z[8] = {}, no = 0.0f;
        if (real && e < a.n) {
            if constexpr (KIND == NORM_RES) {            // the stored sum: x or res may be where it went
                to_f32<RT>(ld8<size_of(RT)>(a.res_out, t * a.res_out_ld + e, a.n - e), z);
                weigh(a, e, a.n - e, z);
            } else {
                load<KIND, XT, RT>(a, t, e, a.n - e, x[0], r[0]);
                form<KIND, XT, RT>(a, x[0], r[0], e, t, a.n - e, false, z, no, bits);
            }
        }
        put(e, z);
    }
    // behind all else, where the row's registers are free: its lanes write over their codes
    if constexpr (KIND == NORM || KIND == NORM_RES)
        if (away) far_norm<KIND, XT, RT>(a, per_wave);
}

template <int KIND, int XT, int RT, bool PACK> void go_rows(const row_args &a, hipStream_t st)
{
    const int rows = PACK ? a.T_pad : a.T, n = PACK ? a.n_pad : a.n;
    const int vecs = (n + 7) / 8;
    // A wave a row where it is short (many rows of 1024: 5.6 us for 4096 of them, 7.6 with a workgroup each).  Many
    // rows: workgroups of 256 lanes, or 512 where a vector is 32 bytes, which leave several to a CU to hide each
    // other's barrier (silu of 4096 x 11264: 53 us, 75 with 1024).  Few: a lane for each vector.
    const bool many = rows >= 256;
    const int per_wave = vecs <= (rows >= 1024 ? 128 : 64);
    const int threads = per_wave || vecs <= 256 ? 256
                      : many && vecs <= 2048    ? (size_of(XT) + size_of(RT) > 4 ? 512 : 256)
                                                : vecs <= 512 ? 512 : 1024;
    const int grid = per_wave ? (rows + 3) / 4 : rows;
    const int nv = per_wave ? (vecs + 63) / 64 : (vecs + threads - 1) / threads;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, i8_grid(grid), dim3(threads), 0, st, a, per_wave); };
    if (nv <= 1) go(k_i8_rows<KIND, XT, RT, 1, PACK>);
    else if (nv == 2) go(k_i8_rows<KIND, XT, RT, 2, PACK>);
    else if (nv <= 4 || threads > 256) go(k_i8_rows<KIND, XT, RT, 4, PACK>);
    else if (nv <= 6) go(k_i8_rows<KIND, XT, RT, 6, PACK>);
    else go(k_i8_rows<KIND, XT, RT, 8, PACK>);
}

// Integers into the packed layout: a lane moves 16 of them.
__global__ __launch_bounds__(256) void k_i8_pack(const int8_t *w, long w_ld, int n_rows, int n_cols, long kb, int8_t *packed)
{
    const int u = blockIdx.y * 256 + threadIdx.x;        // chunk of 16 columns
    const int r = (int)i8_block();
    if (u >= kb * 4 || r >= (n_rows + 31) / 32 * 32) return;
    raw<16> c{};
    if (r < n_rows) {
        const int8_t *p = w + r * w_ld + 16l * u;
        if (16 * u + 16 <= n_cols) c = ld_any<16>(p);
        else
            for (int i = 0; i < n_cols - 16 * u; i++) c.w[i >> 2] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
    }
    __builtin_memcpy(packed + i8_at(kb, r, 16 * u), &c, 16);
}

// Back to values: 2^lpr_log lanes a row, eight codes of each of four vectors a lane (four loads under way; 8192 x 4096
// to 16 bits: 21 to 22 us, 4.5 to 4.7 TB/s).
template <int TYPE>
__global__ __launch_bounds__(256) void k_i8_dequant(const int8_t *q, long q_ld, const float *scale, int T, int n, void *out,
                                                    long out_ld, int lpr_log)
{
    const long t = i8_block() * (256 >> lpr_log) + (threadIdx.x >> lpr_log);
    if (t >= T) return;
    const int lpr = 1 << lpr_log, lane = threadIdx.x & (lpr - 1);
    const float s = scale[t];
    for (long v = (long)blockIdx.y * 4 * lpr + lane; 8 * v < n; v += (long)gridDim.y * 4 * lpr) {
        raw<8> c[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int e = (int)(8 * (v + k * lpr)), left = n - e;
            const int8_t *p = q + t * q_ld + e;
            if (left >= 8) c[k] = ld_any<8>(p);
            else {
                c[k] = raw<8>{};
#pragma unroll
                for (int i = 0; i < 7; i++)
                    if (i < left) c[k].w[i >> 2] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int e = (int)(8 * (v + k * lpr)), left = n - e;
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = (float)(int8_t)(c[k].w[i >> 2] >> (8 * (i & 3))) * s;
            if (left > 0) st8<size_of(TYPE)>(out, t * out_ld + e, left, from_f32<TYPE>(y));
        }
    }
}

// f of the type as a constant.
template <int T> using type_is = std::integral_constant<int, T>;
template <class F> void by_type(int type, F &&f)
{
    type == MLLM_F32 ? f(type_is<MLLM_F32>{}) : type == MLLM_BF16 ? f(type_is<MLLM_BF16>{}) : f(type_is<MLLM_F16>{});
}

const char *rows_refusal(int type, const void *x, long x_ld, int T, int n, const void *q, long q_ld, const float *scale)
{
    if (!i8_real(type)) return "the type is F32, F16 or BF16";
    if (T < 0 || T > 1 << 30 || n <= 0 || n > 1 << 30) return "T is not negative, n positive, both at most 2^30";
    if (x_ld < n || q_ld < n) return "rows lie at least n elements apart";
    if (T && (!x || !q || !scale)) return "x, q and scale are given";
    return nullptr;
}

int done(const char *who) { return hipGetLastError() == hipSuccess ? 0 : pk_fail(who, "the launch failed"); }

} // namespace

extern "C" {

MLLM_API int mllm_i8_quantize(int type, const void *x, long x_ld, int T, int n, int8_t *q, long q_ld, float *scale,
                              void *stream)
{
    const char *who = "mllm_i8_quantize";
    if (const char *why = rows_refusal(type, x, x_ld, T, n, q, q_ld, scale)) return pk_fail(who, why);
    if (!T) return 0;
    row_args a{};
    a.x = x; a.x_ld = x_ld; a.q = q; a.q_ld = q_ld; a.scale = scale; a.T = T; a.n = n;
    hipStream_t st = (hipStream_t)stream;
    by_type(type, [&](auto x) { go_rows<QUANTIZE, x, x, false>(a, st); });
    return done(who);
}

MLLM_API int mllm_i8_dequant(const int8_t *q, long q_ld, const float *scale, int T, int n, int type, void *out,
                             long out_ld, void *stream)
{
    const char *who = "mllm_i8_dequant";
    if (const char *why = rows_refusal(type, out, out_ld, T, n, q, q_ld, scale)) return pk_fail(who, why);
    if (!T) return 0;
    const int vecs = (n + 7) / 8;
    int lpr_log = 2;
    while (lpr_log < 8 && 1 << lpr_log < vecs) lpr_log++;
    const int rows = 256 >> lpr_log, grid_y = std::min((vecs + (4 << lpr_log) - 1) / (4 << lpr_log), 1 << 14);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, i8_grid(((long)T + rows - 1) / rows, grid_y), dim3(256), 0, (hipStream_t)stream, q,
                           q_ld, scale, T, n, out, out_ld, lpr_log);
    };
    type == MLLM_F32 ? go(k_i8_dequant<MLLM_F32>) : type == MLLM_BF16 ? go(k_i8_dequant<MLLM_BF16>) : go(k_i8_dequant<MLLM_F16>);
    return done(who);
}

MLLM_API int mllm_i8_rms_norm(int type, const void *x, long x_ld, int res_type, const void *res, long res_ld,
                              void *res_out, long res_out_ld, int w_type, const void *w, float eps, int T, int n,
                              int8_t *q, long q_ld, float *scale, void *stream)
{
    const char *who = "mllm_i8_rms_norm";
    if (const char *why = rows_refusal(type, x, x_ld, T, n, q, q_ld, scale)) return pk_fail(who, why);
    if (!i8_real(w_type) || (T && !w)) return pk_fail(who, "w is given, in F32, F16 or BF16");
    if (!(eps >= 0.0f) || eps > 3.402823466e38f) return pk_fail(who, "eps is finite and not negative");
    if (res) {
        if (!i8_real(res_type)) return pk_fail(who, "the type of res is F32, F16 or BF16");
        if (!res_out || res_ld < n || res_out_ld < n) return pk_fail(who, "res needs res_out, and rows at least n elements apart");
        if (res_out == res && res_out_ld != res_ld) return pk_fail(who, "res_out may be res only in its stride");
        if (res_out == x && (res_type != type || res_out_ld != x_ld))
            return pk_fail(who, "res_out may be x only in its type and stride");
    }
    if (!T) return 0;
    row_args a{};
    a.x = x; a.x_ld = x_ld; a.res = res; a.res_ld = res_ld; a.res_out = res_out; a.res_out_ld = res_out_ld; a.w = w;
    a.eps = eps; a.q = q; a.q_ld = q_ld; a.scale = scale; a.w_type = w_type;
    a.T = T; a.n = n;
    hipStream_t st = (hipStream_t)stream;
    by_type(type, [&](auto x) {
        if (!res) go_rows<NORM, x, x, false>(a, st);
        else by_type(res_type, [&](auto r) { go_rows<NORM_RES, x, r, false>(a, st); });
    });
    return done(who);
}

MLLM_API int mllm_i8_silu_mul(int type, const void *gate, long gate_ld, const void *up, long up_ld, int T, int n,
                              int8_t *q, long q_ld, float *scale, void *stream)
{
    const char *who = "mllm_i8_silu_mul";
    if (const char *why = rows_refusal(type, gate, gate_ld, T, n, q, q_ld, scale)) return pk_fail(who, why);
    if (up_ld < n || (T && !up)) return pk_fail(who, "up is given, its rows at least n elements apart");
    if (!T) return 0;
    row_args a{};
    a.x = gate; a.x_ld = gate_ld; a.res = up; a.res_ld = up_ld; a.q = q; a.q_ld = q_ld; a.scale = scale;
    a.T = T; a.n = n;
    hipStream_t st = (hipStream_t)stream;
    by_type(type, [&](auto x) { go_rows<SILU, x, x, false>(a, st); });
    return done(who);
}

MLLM_API long mllm_i8_packed_size(int n_rows, int n_cols)
{
    if (n_rows <= 0 || n_cols <= 0 || n_cols > kI8MaxCols || n_rows > 1 << 30) return -1;
    return i8_rblocks(n_rows) * i8_kblocks(n_cols) * 2048;
}

MLLM_API int mllm_i8_pack(int type, const void *w, long w_ld, int n_rows, int n_cols, void *packed, float *scale,
                          void *stream)
{
    const char *who = "mllm_i8_pack";
    if (mllm_i8_packed_size(n_rows, n_cols) < 0) return pk_fail(who, "n_rows is positive, n_cols from 1 to 131071");
    if (type != MLLM_I8 && !i8_real(type)) return pk_fail(who, "the type is F32, F16, BF16 or I8");
    if (!w || !packed || ((uintptr_t)packed & 15) || w_ld < n_cols || (type != MLLM_I8 && !scale))
        return pk_fail(who, "w, packed (16-byte aligned) and scale are given, rows at least n_cols apart");
    const long kb = i8_kblocks(n_cols);
    const int rows = (int)i8_rblocks(n_rows) * 32;
    hipStream_t st = (hipStream_t)stream;
    if (type == MLLM_I8) {
        hipLaunchKernelGGL(k_i8_pack, i8_grid(rows, (unsigned)((kb * 4 + 255) / 256)), dim3(256), 0, st, (const int8_t *)w, w_ld,
                           n_rows, n_cols, kb, (int8_t *)packed);
        return done(who);
    }
    row_args a{};
    a.x = w; a.x_ld = w_ld; a.q = (int8_t *)packed; a.scale = scale; a.T = n_rows; a.n = n_cols; a.kb = kb;
    a.T_pad = rows; a.n_pad = (int)kb * 64;
    by_type(type, [&](auto x) { go_rows<QUANTIZE, x, x, true>(a, st); });
    return done(who);
}

} // extern "C"
