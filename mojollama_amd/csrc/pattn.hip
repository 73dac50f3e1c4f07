// pattn.hip — attention of new tokens over a paged 16- or 8-bit KV cache.
#include <math.h>
#include "paged.h"

namespace {

struct pa_args {
    const void *q;
    void *out;
    long q_ld, out_ld;
    int q_type, out_type;
    mllm_paged_kv kv;
    const int *seqs, *starts, *lens;
    int max_len, T, B, NH, window;
    float scale;
    const float *sinks;
};

// One workgroup per query and head: 256 positions at a time, a score per thread, the running maximum
// and sum, then an element of the output per thread.
__global__ __launch_bounds__(256) void k_pattn(pa_args a)
{
    __shared__ float qs[256], ws[256], red[8];
    __shared__ long at[256];
    __shared__ float vs[256];
    const int h = blockIdx.y, t = blockIdx.x, tid = threadIdx.x, HD = a.kv.head_dim, j = h / (a.NH / a.kv.n_kv_head);
    int b = t, p = 0;
    if (a.starts) {
        for (b = 0; b < a.B && a.starts[b + 1] <= t; b++) {}
        if (b == a.B || t < a.starts[0]) return;
        p = t - a.starts[b + 1];
    } else {
        p = -1;
    }
    const int seq = a.seqs ? a.seqs[b] : b;
    int len = a.lens[b] < a.max_len ? a.lens[b] : a.max_len;
    if (seq < 0 || seq >= a.kv.n_seqs) len = 0;
    p += len;
    const int lo = a.window > 0 && p >= a.window ? p - a.window + 1 : 0;
    if (tid < HD) {
        const long o = t * a.q_ld + (long)h * HD + tid;
        qs[tid] = a.q_type == MLLM_F32 ? ((const float *)a.q)[o]
                : a.q_type == MLLM_BF16 ? (float)((const __bf16 *)a.q)[o] : (float)((const _Float16 *)a.q)[o];
    }
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int s0 = lo; s0 <= p; s0 += 256) {
        __syncthreads();
        int r = s0 + tid;
        long row = -1;
        float z = -INFINITY, vsc = 1.0f;
        if (r <= p) {
            const int page = pk_page(a.kv, seq, r);
            if (page >= 0) row = page * a.kv.page_stride + r * a.kv.row_stride + j * a.kv.head_stride;
            if (row >= 0) {
                float dot = 0.0f, ksc = 1.0f;
                if (a.kv.type == MLLM_E4M3) {
                    const long e = ((long)page * a.kv.n_kv_head + j) * a.kv.page_size + r;
                    ksc = ldexpf(1.0f, a.kv.k_exp[e] - 127);
                    vsc = ldexpf(1.0f, a.kv.v_exp[e] - 127);
                }
                for (int d = 0; d < HD; d++) {
                    float k;
                    if (a.kv.type == MLLM_E4M3) k = __builtin_amdgcn_cvt_f32_fp8(((const uint8_t *)a.kv.k)[row + d], 0) * ksc;
                    else if (a.kv.type == MLLM_BF16) k = (float)((const __bf16 *)a.kv.k)[row + d];
                    else k = (float)((const _Float16 *)a.kv.k)[row + d];
                    dot = fmaf(qs[d], k, dot);
                }
                z = dot * a.scale;
            }
        }
        at[tid] = row;
        vs[tid] = vsc;
        ws[tid] = z;
        __syncthreads();
        float mm = m;
        for (int i = 0; i < 256; i++) mm = fmaxf(mm, ws[i]);
        const float base = mm == -INFINITY ? 0.0f : mm, f = expf(m - base);
        __syncthreads();
        ws[tid] = row < 0 ? 0.0f : expf(z - base);
        __syncthreads();
        l *= f;
        o *= f;
        m = mm;
        for (int i = 0; i < 256; i++) {
            if (at[i] < 0) continue;
            l += ws[i];
            if (tid < HD) {
                float v;
                const long x = at[i] + tid;
                if (a.kv.type == MLLM_E4M3) v = __builtin_amdgcn_cvt_f32_fp8(((const uint8_t *)a.kv.v)[x], 0) * vs[i];
                else if (a.kv.type == MLLM_BF16) v = (float)((const __bf16 *)a.kv.v)[x];
                else v = (float)((const _Float16 *)a.kv.v)[x];
                o = fmaf(ws[i], v, o);
            }
        }
    }
    if (a.sinks && l != 0.0f) {
        const float s = a.sinks[h], mm = fmaxf(m, s), f = expf(m - mm);
        o *= f;
        l = l * f + expf(s - mm);
    }
    if (tid < HD) {
        const float y = l == 0.0f ? 0.0f : o / l;
        const long x = t * a.out_ld + (long)h * HD + tid;
        if (a.out_type == MLLM_F32) ((float *)a.out)[x] = y;
        else if (a.out_type == MLLM_BF16) ((__bf16 *)a.out)[x] = (__bf16)y;
        else ((_Float16 *)a.out)[x] = (_Float16)y;
    }
}

const char *pa_refusal(const mllm_paged_kv *kv, int q_type, const void *q, long q_ld, const int *lens, int max_len, int T,
                       int B, int NH, int window, int out_type, void *out, long out_ld)
{
    if (const char *why = pk_refusal(kv)) return why;
    if (T < 0 || B < 0 || max_len < 0 || NH <= 0 || NH % kv->n_kv_head || window < 0)
        return "NH is a multiple of n_kv_head, counts and window are not negative";
    if ((long)T * NH > 1 << 30 || NH > 65535) return "at most 2^30 queries times heads, 65535 heads";
    if ((T && (!q || !out)) || (B && !lens)) return "q, lens and out are needed";
    const int own = kv->type == MLLM_F16 ? MLLM_F16 : MLLM_BF16;
    if ((q_type != MLLM_F32 && q_type != own) || (out_type != MLLM_F32 && out_type != own))
        return "q and out are F32 or the cache's type (BF16 for E4M3)";
    if (q_ld < (long)NH * kv->head_dim || out_ld < (long)NH * kv->head_dim) return "row strides are at least NH * head_dim";
    if ((((uintptr_t)q | (uintptr_t)(q_ld * pk_size(q_type))) | ((uintptr_t)out | (uintptr_t)(out_ld * pk_size(out_type)))) & 15)
        return "the rows of q and out are multiples of 16 bytes";
    return nullptr;
}

int pa_launch(const char *who, pa_args &a, void *stream)
{
    hipLaunchKernelGGL(k_pattn, dim3(a.T, a.NH), dim3(256), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? 0 : pk_fail(who, "the launch failed");
}

} // namespace

extern "C" {

MLLM_API long mllm_paged_attn_workspace_size(const mllm_paged_kv *kv, int T, int B, int NH, int max_len, int window)
{
    if (pk_refusal(kv) || T < 0 || B < 0 || NH <= 0 || NH % kv->n_kv_head || max_len < 0 || window < 0) return -1;
    return 256;
}

MLLM_API int mllm_paged_attn_decode(const mllm_paged_kv *kv, int q_type, const void *q, long q_ld, const int *seqs,
                                    const int *lens, int max_len, int B, int NH, float scale, int window,
                                    const float *sinks, int out_type, void *out, long out_ld, void *workspace,
                                    long ws_bytes, void *stream)
{
    const char *who = "mllm_paged_attn_decode";
    if (const char *why = pa_refusal(kv, q_type, q, q_ld, lens, max_len, B, B, NH, window, out_type, out, out_ld))
        return pk_fail(who, why);
    if (!seqs && B > kv->n_seqs) return pk_fail(who, "without seqs, B is at most the cache's n_seqs");
    if (!workspace || ws_bytes < mllm_paged_attn_workspace_size(kv, B, B, NH, max_len, window))
        return pk_fail(who, "workspace below mllm_paged_attn_workspace_size");
    if (!B) return 0;
    pa_args a{q, out, q_ld, out_ld, q_type, out_type, *kv, seqs, nullptr, lens, max_len, B, B, NH, window, scale, sinks};
    return pa_launch(who, a, stream);
}

MLLM_API int mllm_paged_attn_prompt(const mllm_paged_kv *kv, int q_type, const void *q, long q_ld, const int *seqs,
                                    const int *starts, const int *lens, int max_len, int T, int B, int NH, float scale,
                                    int window, const float *sinks, int out_type, void *out, long out_ld,
                                    void *workspace, long ws_bytes, void *stream)
{
    const char *who = "mllm_paged_attn_prompt";
    if (const char *why = pa_refusal(kv, q_type, q, q_ld, lens, max_len, T, B, NH, window, out_type, out, out_ld))
        return pk_fail(who, why);
    if (!starts) return pk_fail(who, "starts is needed");
    if (!seqs && B > kv->n_seqs) return pk_fail(who, "without seqs, B is at most the cache's n_seqs");
    if (!workspace || ws_bytes < mllm_paged_attn_workspace_size(kv, T, B, NH, max_len, window))
        return pk_fail(who, "workspace below mllm_paged_attn_workspace_size");
    if (!T || !B) return 0;
    pa_args a{q, out, q_ld, out_ld, q_type, out_type, *kv, seqs, starts, lens, max_len, T, B, NH, window, scale, sinks};
    return pa_launch(who, a, stream);
}

} // extern "C"
