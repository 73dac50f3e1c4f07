// pattn.hip — attention of new tokens over a paged 16- or 8-bit KV cache: its checks, the choice of splits
// and tiles, and the join of split rows.  The kernels are in pattn_decode.h and pattn_prompt.h.
#include <math.h>
#include <algorithm>
#include "pattn.h"

namespace {

const char *pa_refusal(const mllm_paged_kv *kv, int q_type, const void *q, long q_ld, const int *lens, int max_len, int T,
                       int B, int NH, float scale, int window, int out_type, void *out, long out_ld)
{
    if (const char *why = pk_refusal(kv)) return why;
    if (T < 0 || B < 0 || max_len < 0 || NH <= 0 || NH % kv->n_kv_head || window < 0)
        return "NH is a multiple of n_kv_head, counts and window are not negative";
    if ((long)T * NH > 1 << 30 || NH > 65535 || B > 65535 || max_len > 1 << 30)
        return "at most 2^30 queries times heads, 65535 heads and sequences, max_len 2^30";
    if ((T && (!q || !out)) || (B && !lens)) return "q, lens and out are needed";
    if (!(fabsf(scale) < INFINITY)) return "scale is finite";
    const int own = kv->type == MLLM_F16 ? MLLM_F16 : MLLM_BF16;
    if ((q_type != MLLM_F32 && q_type != own) || (out_type != MLLM_F32 && out_type != own))
        return "q and out are F32 or the cache's type (BF16 for E4M3)";
    if (q_ld < (long)NH * kv->head_dim || out_ld < (long)NH * kv->head_dim) return "row strides are at least NH * head_dim";
    if ((((uintptr_t)q | (uintptr_t)(q_ld * pk_size(q_type))) | ((uintptr_t)out | (uintptr_t)(out_ld * pk_size(out_type)))) & 15)
        return "the rows of q and out are multiples of 16 bytes";
    return nullptr;
}

// The splits of a query's rows joined: their sums under one maximum.  One row (query and head) and up
// to 64 columns per workgroup: 16 threads cover the columns, the 16 groups of so many take every 16th
// split, four loads in flight each.
__global__ __launch_bounds__(256) void k_pa_join(pa_args a)
{
    __shared__ float wt[256], red[2][4];
    __shared__ __attribute__((aligned(16))) float acc[256 * 4];
    const int h = blockIdx.y, t = blockIdx.x, tid = threadIdx.x, HD = a.kv.head_dim;
    if (a.starts && (t < a.starts[0] || t >= a.starts[a.B])) return;
    const long row = (long)t * a.NH + h;
    const int gi = tid >> 4, d = 64 * blockIdx.z + 4 * (tid & 15), dc = min(d, HD - 4);
    const float *part = a.part + row * a.splits * HD + dc;
    float2 ml = make_float2(kLowest, 0.0f);
    if (tid < a.splits) ml = *(const float2 *)(a.stat + (row * a.splits + tid) * 2);
    float4 x[4];
#pragma unroll
    for (int u = 0; u < 4; u++) x[u] = *(const float4 *)(part + (long)min(gi + 16 * u, a.splits - 1) * HD);
    float m = ml.x;
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
    if (!(tid & 63)) red[0][tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float f = ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - m);
    wt[tid] = f;
    float l = f * ml.y;
    for (int k = 32; k; k >>= 1) l += __shfl_xor(l, k, 64);
    if (!(tid & 63)) red[1][tid >> 6] = l;
    __syncthreads();
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s = gi; s < a.splits; s += 64) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const float c = s + 16 * u < a.splits ? wt[s + 16 * u] : 0.0f;
            if (c != 0.0f) {                         // an empty split's sums are not written (NaN's are: c is NaN)
                y.x = fmaf(c, x[u].x, y.x); y.y = fmaf(c, x[u].y, y.y); y.z = fmaf(c, x[u].z, y.z); y.w = fmaf(c, x[u].w, y.w);
            }
        }
        if (s + 64 < a.splits)
#pragma unroll
            for (int u = 0; u < 4; u++) x[u] = *(const float4 *)(part + (long)min(s + 64 + 16 * u, a.splits - 1) * HD);
    }
    *(float4 *)(acc + 4 * tid) = y;
    __syncthreads();
    if (gi || d >= HD) return;
#pragma unroll
    for (int s = 1; s < 16; s++) {
        const float4 z = *(const float4 *)(acc + 4 * (tid + 16 * s));
        y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
    }
    pa_finish(a, h, t, d, m, l, y);
}

constexpr int kMaxSplits = 256, kMinRows = 256;      // rows of a split at least
// Splits are made until a launch has so many workgroups: then all partial sums together are at most those of
// kPartRows rows (16 of a workgroup's in decode, 128 in a prompt's) and one of each row.
constexpr long kPartRows = 65536, kDecodeWG = kPartRows / 16, kPromptWG = kPartRows / 128;

// Rows that a query can see, as far as the host knows.
long seen(int max_len, int window) { return window > 0 ? std::min<long>(max_len, (long)window + 31) : max_len; }

long up(long a, long b) { return (a + b - 1) / b; }

// Splits of a launch of `wgs` workgroups that would each take all of n rows: until there are `target`.
int pa_splits(long wgs, long n, long target)
{
    return (int)std::max<long>(1, std::min({up(target, wgs), up(n, kMinRows), (long)kMaxSplits}));
}

// In decode, of 1024 rows where the launch is large (unequal lengths then share the GPU evenly, and the sums
// stay small), down to 256 until every CU has a workgroup; up to 640 rows whole, which saves the join.
// 256 / 512 / 1024 rows: one sequence of 2000 rows, 4 kv heads, 8.2 / 9.6 / 12.4 us, of 131072 60.8 / 60.6 /
// 58.7, eight of 2048 to 4096, 8 kv heads, 18.3 / 19.2 / 16.5, 48 of up to 9000 42.0 / 42.5 / 43.1; one of 300
// rows whole / split 5.8 / 8.1, of 500 6.7 / 8.2, of 700 8.0 / 8.2.
int pa_splits_decode(long wgs, long n)
{
    if (n <= 640) return 1;
    const long fill = std::min(up(n, kMinRows), up(256, wgs));
    return (int)std::min({std::max(std::min(up(n, 1024), up(kDecodeWG, wgs)), fill), (long)kMaxSplits});
}

void pa_divisor(pa_args &a)
{
    // s / d = s * m >> (31 + l) for s < 2^31, with l = ceil(log2 d), m = floor(2^(31 + l) / d) + 1 (Granlund
    // and Montgomery); m is below 2^32
    const uint64_t d = (uint64_t)a.kv.page_size;
    int l = 0;
    while ((1ull << l) < d) l++;
    a.div_mul = (unsigned)(((1ull << (31 + l)) / d) + 1);
    a.div_sh = 31 + l;
}

// The partial sums' places; false where the workspace does not hold them.
bool pa_partials(pa_args &a, void *ws, long ws_bytes)
{
    if (a.splits == 1) return true;
    const long n = (long)a.T * a.NH * a.splits, stat = (n * 2 + 3) / 4 * 4;
    a.stat = (float *)ws;
    a.part = a.stat + stat;
    return 4 * (stat + n * a.kv.head_dim) <= ws_bytes;
}

int pa_launch(const char *who, pa_args &a, void *ws, long ws_bytes, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    // every position is below max_len: such a window masks nothing, and the kernels' sums with it stay in 32 bits
    if (a.window >= a.max_len) a.window = 0;
    pa_divisor(a);
    a.rep = a.NH / a.kv.n_kv_head;
    const bool wide = a.q_type == MLLM_F32 || a.out_type == MLLM_F32;
    const int es = pk_size(a.kv.type);
    // pages of a multiple of 16 rows: a tile's rows lie in one page (and four exponents in a word)
    const bool uniform = a.kv.page_size % 16 == 0 && a.kv.row_stride * 16 * es < 0x7FFFFFFF &&
                         (es == 2 || !(((uintptr_t)a.kv.k_exp | (uintptr_t)a.kv.v_exp) & 3));
    if (!a.starts) {
        a.groups = (a.rep + 15) / 16;
        const long n = seen(a.max_len, a.window);
        a.splits = pa_splits_decode((long)a.B * a.kv.n_kv_head * a.groups, n);
        a.chunk = (int)(std::max<long>(1, (n + 128l * a.splits - 1) / (128l * a.splits)) * 128);
        a.splits = (int)std::max<long>(1, (n + a.chunk - 1) / a.chunk);
        if (!pa_partials(a, ws, ws_bytes)) return pk_fail(who, "workspace below what the splits take");
        if (a.kv.type == MLLM_F16) pa_decode_f16(a, wide, uniform, st);
        else if (a.kv.type == MLLM_BF16) pa_decode_bf16(a, wide, uniform, st);
        else pa_decode_e4m3(a, wide, uniform, st);
    } else {
        const long rows = (long)a.T * a.rep, n = a.window > 0 ? std::min<long>(a.window + 320l, a.max_len) : a.max_len;
        const int hdb = a.kv.head_dim <= 64 ? 64 : a.kv.head_dim <= 128 ? 128 : 256;
        a.groups = pa_row_groups(a.kv.type, wide, hdb);
        // tiles of 256 rows, half the traffic from L2, where they fill the GPU (6011 tokens, 32/8 heads of 128:
        // 418 us, of 128 rows 452; below a workgroup per CU they leave CUs without work)
        const bool large = a.groups == 4 && pa_halves(a.kv.type, wide, hdb) == 2 && uniform && a.kv.page_size % 64 == 0 &&
                           rows / 256 * a.kv.n_kv_head >= 256;
        if (large) a.groups = 8;
        a.tiles = (int)(rows / (32 * a.groups) + std::min(a.T, a.B));
        // no more than keep the partial sums, written and read again, below the rows of K and V that they save
        // time on: prompts of 1 to 1100 tokens over up to 2600 rows, window 512, 16/4 heads of 96, split
        // to fill the GPU / whole 99 / 33 us; 3 to 5 tokens over 1500 to 4000 rows, 64/8 heads of 64, seven / whole
        // 29 / 123 us
        const long most = n * a.B * a.kv.n_kv_head * es / (4l * a.T * a.NH);
        a.splits = large ? 1 : (int)std::max<long>(1, std::min<long>(most, pa_splits((long)a.tiles * a.kv.n_kv_head, n, kPromptWG)));
        a.chunk = a.splits == 1 ? 1 << 30 : (int)((n + 64l * a.splits - 1) / (64l * a.splits) * 64);
        if (a.splits > 1) a.splits = (int)((n + a.chunk - 1) / a.chunk);
        if (!pa_partials(a, ws, ws_bytes)) return pk_fail(who, "workspace below what the splits take");
        auto go = a.kv.type == MLLM_F16 ? wide ? pa_prompt_wide_f16 : pa_prompt_f16
                : a.kv.type == MLLM_BF16 ? wide ? pa_prompt_wide_bf16 : pa_prompt_bf16
                                         : wide ? pa_prompt_wide_e4m3 : pa_prompt_e4m3;
        go(a, uniform, st);
    }
    if (a.splits > 1) hipLaunchKernelGGL(k_pa_join, dim3(a.T, a.NH, (a.kv.head_dim + 63) / 64), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : pk_fail(who, "the launch failed");
}

} // namespace

extern "C" {

MLLM_API long mllm_paged_attn_workspace_size(const mllm_paged_kv *kv, int T, int B, int NH, int max_len, int window)
{
    if (pk_refusal(kv) || T < 0 || B < 0 || NH <= 0 || NH % kv->n_kv_head || max_len < 0 || window < 0) return -1;
    // rows (query and head) times splits: each row has at most its range's, all rows together kPartRows and
    // one each; both grow with every size, so a workspace serves smaller calls
    const long rows = (long)T * NH, n = window > 0 ? std::min<long>(max_len, window + 320l) : max_len;
    const long most = std::max<long>(1, std::min<long>((n + kMinRows - 1) / kMinRows, kMaxSplits));
    return 4 * (std::min(rows * most, kPartRows + rows) * (kv->head_dim + 2) + 64);
}

MLLM_API int mllm_paged_attn_decode(const mllm_paged_kv *kv, int q_type, const void *q, long q_ld, const int *seqs,
                                    const int *lens, int max_len, int B, int NH, float scale, int window,
                                    const float *sinks, int out_type, void *out, long out_ld, void *workspace,
                                    long ws_bytes, void *stream)
{
    const char *who = "mllm_paged_attn_decode";
    if (const char *why = pa_refusal(kv, q_type, q, q_ld, lens, max_len, B, B, NH, scale, window, out_type, out, out_ld))
        return pk_fail(who, why);
    if (!seqs && B > kv->n_seqs) return pk_fail(who, "without seqs, B is at most the cache's n_seqs");
    if (!workspace || ws_bytes < mllm_paged_attn_workspace_size(kv, B, B, NH, max_len, window))
        return pk_fail(who, "workspace below mllm_paged_attn_workspace_size");
    if (!B) return 0;
    pa_args a{q, out, q_ld, out_ld, q_type, out_type, *kv, seqs, nullptr, lens, max_len, B, B, NH, window, scale, sinks};
    return pa_launch(who, a, workspace, ws_bytes, stream);
}

MLLM_API int mllm_paged_attn_prompt(const mllm_paged_kv *kv, int q_type, const void *q, long q_ld, const int *seqs,
                                    const int *starts, const int *lens, int max_len, int T, int B, int NH, float scale,
                                    int window, const float *sinks, int out_type, void *out, long out_ld,
                                    void *workspace, long ws_bytes, void *stream)
{
    const char *who = "mllm_paged_attn_prompt";
    if (const char *why = pa_refusal(kv, q_type, q, q_ld, lens, max_len, T, B, NH, scale, window, out_type, out, out_ld))
        return pk_fail(who, why);
    if (!starts) return pk_fail(who, "starts is needed");
    if (!seqs && B > kv->n_seqs) return pk_fail(who, "without seqs, B is at most the cache's n_seqs");
    if (!workspace || ws_bytes < mllm_paged_attn_workspace_size(kv, T, B, NH, max_len, window))
        return pk_fail(who, "workspace below mllm_paged_attn_workspace_size");
    if (!T || !B) return 0;
    pa_args a{q, out, q_ld, out_ld, q_type, out_type, *kv, seqs, starts, lens, max_len, T, B, NH, window, scale, sinks};
    return pa_launch(who, a, workspace, ws_bytes, stream);
}

} // extern "C"
