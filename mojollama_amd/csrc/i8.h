// i8.h — layers in 8-bit integers (mllm_i8_*): the packed weight layout, element access at any
// alignment and the rounding of a row.
//
// Packed weights: blocks of 32 rows x 64 columns, 2 KB each, the blocks of 32 rows one after the other
// along K.  A block holds [column chunk of 16][row][16 bytes], so that the 64 lanes of one load take 1 KB
// in lane order and hold a v_mfma_i32_32x32x32_i8 operand (row lane % 32, chunk lane / 32), and the lanes
// of v_mfma_i32_16x16x64_i8 (row lane % 16, chunk lane / 16) runs of 256 bytes.  Rows and columns are
// padded with zeros (columns to 512): what a kernel reads of x behind its last column has no part in a sum.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdio.h>
#include <string.h>
#include "mllm.h"
#include "moe.h"
#include "paged.h"

constexpr int kI8MaxCols = 131071;         // 128 * 128 * 131071 < 2^31

__host__ __device__ inline long i8_kblocks(int n_cols) { return ((long)n_cols + 511) / 512 * 8; }
__host__ __device__ inline long i8_rblocks(int n_rows) { return ((long)n_rows + 31) / 32; }
// Byte of element (r, k).
__host__ __device__ inline long i8_at(long kb, int r, int k)
{
    return ((r >> 5) * kb + (k >> 6)) * 2048 + ((k >> 4) & 3) * 512 + (r & 31) * 16 + (k & 15);
}

// A launch of `blocks` workgroups, more than fit the 2^32 lanes of one dimension too: block() of the kernel is below
// blocks or behind them.
constexpr long kI8Blocks = 1l << 21;
inline dim3 i8_grid(long blocks, unsigned y = 1)
{
    return dim3((unsigned)(blocks < kI8Blocks ? blocks : kI8Blocks), y, (unsigned)((blocks + kI8Blocks - 1) / kI8Blocks));
}
__device__ __forceinline__ long i8_block() { return (long)blockIdx.z * gridDim.x + blockIdx.x; }

inline bool i8_real(int type) { return type == MLLM_F32 || type == MLLM_F16 || type == MLLM_BF16; }

// One or two floats as elements of the type.  A sum or product is a number of 32 bits before it is one of 16: the
// compiler would round some of them to F16 once.
__device__ __forceinline__ void put1(void *p, long at, int type, float x)
{
    if (type == MLLM_F32) { ((float *)p)[at] = x; return; }
    asm("" : "+v"(x));
    if (type == MLLM_BF16) ((__bf16 *)p)[at] = (__bf16)x;
    else ((_Float16 *)p)[at] = (_Float16)x;
}
template <int TYPE> __device__ __forceinline__ uint32_t pack2(float a, float b)
{
    if constexpr (TYPE == MLLM_F16) asm("" : "+v"(a), "+v"(b));
    return pack16(a, b, TYPE);
}
