// paged.h — the paged 16- or 8-bit KV cache (mllm_paged_kv) inside the library:
// its checks, row addressing and element types.
#pragma once
#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdint.h>
#include "mllm.h"
#include "moe.h"

inline int pk_size(int type) { return type == MLLM_F32 ? 4 : type == MLLM_E4M3 ? 1 : 2; }

// Why a view is not served, or null.
inline const char *pk_refusal(const mllm_paged_kv *kv)
{
    if (!kv || !kv->k || !kv->v || !kv->tables) return "a cache needs k, v and tables";
    if (kv->type != MLLM_F16 && kv->type != MLLM_BF16 && kv->type != MLLM_E4M3) return "a cache holds F16, BF16 or E4M3";
    if (kv->type == MLLM_E4M3 && (!kv->k_exp || !kv->v_exp)) return "an E4M3 cache needs k_exp and v_exp";
    if (kv->n_kv_head <= 0 || kv->head_dim <= 0 || kv->head_dim > 256 || kv->head_dim % 16)
        return "head_dim is a multiple of 16 up to 256, n_kv_head positive";
    if (kv->n_pages <= 0 || kv->page_size <= 0 || kv->n_seqs <= 0 || kv->max_blocks <= 0 || kv->table_ld < kv->max_blocks)
        return "n_pages, page_size, n_seqs and max_blocks are positive, table_ld at least max_blocks";
    const long b = pk_size(kv->type);
    if (((uintptr_t)kv->k | (uintptr_t)kv->v | (uintptr_t)(kv->page_stride * b) | (uintptr_t)(kv->row_stride * b) |
         (uintptr_t)(kv->head_stride * b)) & 15)
        return "k, v and the strides are multiples of 16 bytes";
    if (kv->page_stride < 0 || kv->row_stride < 0 || kv->head_stride < 0) return "strides are not negative";
    return nullptr;
}

inline int pk_fail(const char *who, const char *why)
{
    char m[256];
    snprintf(m, sizeof m, "%s: %s", who, why);
    mllm_set_error(m);
    return -1;
}

// The page of row s of sequence seq (0 <= seq < n_seqs, s >= 0), -1 unmapped; s becomes the row in the page.
__device__ __forceinline__ int pk_page(const mllm_paged_kv &kv, int seq, int &s)
{
    const int blk = s / kv.page_size;
    if (blk >= kv.max_blocks) return -1;
    s -= blk * kv.page_size;
    const int p = kv.tables[(long)seq * kv.table_ld + blk];
    return p >= 0 && p < kv.n_pages ? p : -1;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Eight elements of a row of the given type at element `at`, as floats (the address a multiple
// of 16 bytes if `wide`, else of the element's size).
__device__ __forceinline__ void load8(const void *p, long at, int type, bool wide, float (&x)[8])
{
    if (type == MLLM_F32) {
        const float *f = (const float *)p + at;
        if (wide) {
            const float4 a = ((const float4 *)f)[0], b = ((const float4 *)f)[1];
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = f[i];
        }
        return;
    }
    uint32_t w[4];
    const uint16_t *h = (const uint16_t *)p + at;
    if (wide) {
        const uint4 u = *(const uint4 *)h;
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (type == MLLM_BF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const f16x2 v = __builtin_bit_cast(f16x2, w[i]);
            x[2 * i] = (float)v.x;
            x[2 * i + 1] = (float)v.y;
        }
    }
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int type)
{
    if (type == MLLM_BF16) return __builtin_bit_cast(uint32_t, (bf16x2){(__bf16)a, (__bf16)b});
    return __builtin_bit_cast(uint32_t, (f16x2){(_Float16)a, (_Float16)b});
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <bool PAST> __device__ __forceinline__ void put16(void *p, u32x4 v)
{
    if constexpr (PAST) __builtin_nontemporal_store(v, (u32x4 *)p);
    else *(u32x4 *)p = v;
}

// PAST: past the caches (rows that are multiples of 16 bytes).
template <bool PAST = false>
__device__ __forceinline__ void store8(void *p, long at, int type, bool wide, const float (&x)[8])
{
    if (type == MLLM_F32) {
        float *f = (float *)p + at;
        if (wide) {
            put16<PAST>(f, __builtin_bit_cast(u32x4, (f32x4){x[0], x[1], x[2], x[3]}));
            put16<PAST>(f + 4, __builtin_bit_cast(u32x4, (f32x4){x[4], x[5], x[6], x[7]}));
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = x[i];
        }
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = pack16(x[2 * i], x[2 * i + 1], type);
    uint16_t *h = (uint16_t *)p + at;
    if (wide) {
        put16<PAST>(h, (u32x4){w[0], w[1], w[2], w[3]});
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) { h[2 * i] = (uint16_t)w[i]; h[2 * i + 1] = (uint16_t)(w[i] >> 16); }
    }
}
