// i8_gemm.hip — the product of 8-bit integer rows with packed 8-bit integer weights (i8.h), scales per
// token and per weight row.
//
// out[t][r] = (sum_k x[t][k] w[r][k]) * xs[t] * ws[r] + bias[r]; the sums are whole numbers below 2^31 and
// exact in any order, so K may be split freely and the result does not depend on how.
#include "i8.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

struct gemm_args {
    const int8_t *w, *x;
    const float *ws, *xs, *bias;
    void *out;
    long x_ld, out_ld, kb;
    int T, R, K, type;
};

__device__ __forceinline__ float value(int acc, float xs, float ws) { return (float)acc * xs * ws; }

// A wave per 32 weight rows x 32 tokens, operands from global memory.
__global__ __launch_bounds__(64) void k_i8_gemm(gemm_args a)
{
    const int lane = threadIdx.x, l = lane & 31, h = lane >> 5;
    const int r0 = blockIdx.x * 32, t0 = blockIdx.y * 32;
    const int8_t *w = a.w + (r0 >> 5) * a.kb * 2048 + lane * 16;
    const int8_t *x = a.x + (long)min(t0 + l, a.T - 1) * a.x_ld;
    const int last = (a.K - 1) / 16 * 16;
    i32x16 acc = {};
    for (int k = 0; k < a.kb * 64; k += 32) {
        const i32x4 wf = *(const i32x4 *)(w + (long)k * 32);
        const i32x4 xf = *(const i32x4 *)(x + min(k + 16 * h, last));
        acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf, xf, acc, 0, 0, 0);
    }
    const int t = t0 + l;
    if (t >= a.T) return;
    const float xs = a.xs[t];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int r = r0 + 8 * (i >> 2) + 4 * h + (i & 3);
        if (r >= a.R) continue;
        const float y = value(acc[i], xs, a.ws[r]);
        put1(a.out, t * a.out_ld + r, a.type, a.bias ? y + a.bias[r] : y);
    }
}

} // namespace

extern "C" {

MLLM_API long mllm_i8_gemm_workspace_size(int T, int n_rows, int n_cols)
{
    if (T < 0 || mllm_i8_packed_size(n_rows, n_cols) < 0) return -1;
    return 0;
}

MLLM_API int mllm_i8_gemm(const void *packed, const float *w_scale, const int8_t *x, long x_ld, const float *x_scale,
                          int T, int n_rows, int n_cols, const float *bias, int type, void *out, long out_ld,
                          void *workspace, long ws_bytes, void *stream)
{
    const char *who = "mllm_i8_gemm";
    if (T < 0 || mllm_i8_packed_size(n_rows, n_cols) < 0)
        return pk_fail(who, "T is not negative, n_rows positive, n_cols from 1 to 131071");
    if (!i8_real(type)) return pk_fail(who, "the type of out is F32, F16 or BF16");
    if (x_ld < n_cols || out_ld < n_rows) return pk_fail(who, "rows of x lie at least n_cols apart, of out n_rows");
    if (((uintptr_t)x | (uintptr_t)x_ld | (uintptr_t)packed | (uintptr_t)workspace) & 15)
        return pk_fail(who, "x, its rows, packed and the workspace lie at multiples of 16 bytes");
    if (T && (!packed || !w_scale || !x || !x_scale || !out))
        return pk_fail(who, "packed, w_scale, x, x_scale and out are given");
    const long need = mllm_i8_gemm_workspace_size(T, n_rows, n_cols);
    if (need > 0 && (!workspace || ws_bytes < need)) return pk_fail(who, "the workspace is too small");
    if (!T) return 0;
    gemm_args a{(const int8_t *)packed, x, w_scale, x_scale, bias, out, x_ld, out_ld, i8_kblocks(n_cols), T, n_rows, n_cols,
                type};
    hipLaunchKernelGGL(k_i8_gemm, dim3((unsigned)i8_rblocks(n_rows), (unsigned)((T + 31l) / 32)), dim3(64), 0,
                       (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? 0 : pk_fail(who, "the launch failed");
}

} // extern "C"
