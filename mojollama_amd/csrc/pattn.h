// pattn.h — attention over a paged cache: what its kernels and their launcher share.
#pragma once
#include "paged.h"

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
    // set by the launcher
    int rep, groups;               // query heads per kv head; of 16 (decode), or 32 rows of a tile (prompt)
    unsigned div_mul;              // s / page_size = s * div_mul >> div_sh for 0 <= s < 2^31
    int div_sh;
    int chunk, splits;             // rows per split, splits of a query's range of rows
    int tiles;                     // prompt: tiles at most
    float *part, *stat;            // with splits > 1: sums [T * NH][splits][HD], (maximum, sum) [T * NH][splits]
};

// A row of a sequence, 0 <= s: its block.
__device__ __forceinline__ int pa_block(const pa_args &a, int s)
{
    return (int)(((uint64_t)(unsigned)s * a.div_mul) >> a.div_sh);
}

// The table through the scalar cache: a vector load here would wait for every load issued before it.
__device__ __forceinline__ int pa_table(const pa_args &a, int seq, int blk)
{
    typedef const __attribute__((address_space(4))) int *sptr;
    return ((sptr)(uintptr_t)a.kv.tables)[(long)seq * a.kv.table_ld + blk];
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int CT> __device__ __forceinline__ f32x4 pa_mfma16(uint4 x, uint4 y, f32x4 c)
{
    if constexpr (CT == MLLM_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3e38f;   // below every score: exp2(-inf - kLowest) is 0, not NaN
// A running maximum is moved, and the sums scaled, only when a score passes it by 2^kSlack: weights
// then reach 2^kSlack, which no type here minds.  fp16 weights are formed 2^7 larger, so that those
// down to 2^-21 of the maximum stay normal.
constexpr float kSlack = 8.0f;
template <int CT> constexpr float kBias = CT == MLLM_F16 ? 7.0f : 0.0f;

// x and y as planes of 16-bit values, one word each: bf16 takes three (8 + 8 + 8 bits), fp16 two
// (11 + 11); NP == 1 rounds.  W: weights, x and y >= 0.  No plane of theirs is then negative, and none 0 beside
// one that is not (they sum to kPlanesSum x; in fp16 as far as its subnormals reach): an infinity of V times
// them is infinite, where a plane of 0 or below would make it NaN.  The sum of the weights is multiplied by
// kPlanesSum as well, once, and the factor cancels.
constexpr float kPlanesSum = 1.00000011920928955078125f;     // 1 + 2^-23
template <int CT, int NP, bool W = false> __device__ __forceinline__ void pa_planes(float x, float y, uint32_t (&w)[NP])
{
    constexpr float E = W ? kPlanesSum : 1.0f;
    if constexpr (NP == 1) {
        w[0] = pack16(x, y, CT == MLLM_F16 ? MLLM_F16 : MLLM_BF16);
    } else if constexpr (CT == MLLM_F16) {
        f16x2 h = {(_Float16)x, (_Float16)y};
        if constexpr (W) h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x, y));
        w[0] = __builtin_bit_cast(uint32_t, h);
        w[1] = __builtin_bit_cast(uint32_t, (f16x2){(_Float16)fmaf(x, E, -(float)h.x), (_Float16)fmaf(y, E, -(float)h.y)});
    } else {
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
            w[p] = __builtin_amdgcn_perm(b, a, 0x07060302);
            x = fmaf(x, E, -__uint_as_float(a & 0xFFFF0000u));
            y = fmaf(y, E, -__uint_as_float(b & 0xFFFF0000u));
        }
    }
}
template <int CT> constexpr int kPlanes = CT == MLLM_F16 ? 2 : 3;

// Two e4m3 codes of a word as bf16, times a power of two (both exact).
template <bool HI> __device__ __forceinline__ uint32_t pa_cvt8(uint32_t w, float scale)
{
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
__device__ __forceinline__ float pa_exp8(uint32_t byte) { return __uint_as_float((byte & 255u) << 23); }

// Four elements, from d on, of the query t's head h: the weighted sum y over the sum l under the
// maximum m (in units of log 2), with the head's sink.
__device__ __forceinline__ void pa_finish(const pa_args &a, int h, int t, int d, float m, float l, float4 y)
{
    float f = 1.0f / l;
    if (a.sinks && l != 0.0f) {
        const float s = a.sinks[h] * kLog2e, top = fmaxf(m, s), u = __builtin_amdgcn_exp2f(m - top);
        f = u / (l * u + __builtin_amdgcn_exp2f(s - top + (a.kv.type == MLLM_F16 ? kBias<MLLM_F16> : 0.0f)));
    }
    if (l == 0.0f) { f = 0.0f; y = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    const long at = t * a.out_ld + (long)h * a.kv.head_dim + d;
    if (a.out_type == MLLM_F32)
        *(float4 *)((float *)a.out + at) = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
    else
        *(uint2 *)((uint16_t *)a.out + at) = make_uint2(pack16(y.x * f, y.y * f, a.out_type), pack16(y.z * f, y.w * f, a.out_type));
}

// The prompt kernel's tile: groups of 32 rows, and whether two waves share each, one half of every step's
// rows of K and V for each (two waves a SIMD in small launches: prompts of 1 to 1100 tokens, window 512, 36.4 ->
// 33.4 us; drafts in fp32 on 64 rows instead of 128, whose waves were half idle, 29.6 -> 26.7).
constexpr int pa_row_groups(int type, bool wide, int hdb) { return wide ? 2 : 4; }
// ... or, at head sizes above 128, the columns of the output: the registers of a wave hold half of them (fp32,
// fp16 cache, head size 256, 2789 tokens: 403 -> 180 us; the whole of them spilled).
constexpr int pa_parts(int hdb) { return hdb > 128 ? 2 : 1; }
constexpr int pa_halves(int type, bool wide, int hdb) { return hdb > 128 || (!wide && type == MLLM_E4M3 && hdb == 64) ? 1 : 2; }

void pa_decode_bf16(const pa_args &a, bool wide, bool uniform, hipStream_t st);
void pa_decode_f16(const pa_args &a, bool wide, bool uniform, hipStream_t st);
void pa_decode_e4m3(const pa_args &a, bool wide, bool uniform, hipStream_t st);
void pa_prompt_bf16(const pa_args &a, bool uniform, hipStream_t st);
void pa_prompt_f16(const pa_args &a, bool uniform, hipStream_t st);
void pa_prompt_e4m3(const pa_args &a, bool uniform, hipStream_t st);
void pa_prompt_wide_bf16(const pa_args &a, bool uniform, hipStream_t st);
void pa_prompt_wide_f16(const pa_args &a, bool uniform, hipStream_t st);
void pa_prompt_wide_e4m3(const pa_args &a, bool uniform, hipStream_t st);
