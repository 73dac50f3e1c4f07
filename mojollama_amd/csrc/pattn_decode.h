// pattn_decode.h — the split decode kernel over a paged cache, instantiated per cache type.
#pragma once
#include <math.h>
#include "pattn.h"

// One query token of up to 16 heads that share a kv head, over a range of its rows.
//
// The work is one read of the range's K and V rows; everything is laid out so that the bytes go from
// memory to the matrix cores through registers alone.  A wave takes 32 rows at a time as two tiles of
// 16 (i = lane % 16, g = lane / 16):
//   S^T = K Q^T   (16x16x32): lane (i, g) feeds K's row i, so it loads its operand from the row itself;
//                 it gets the scores of rows 4g .. 4g+3 for head i
//   O^T += V^T P  the k index of this product may run over the rows in any order that V and P share:
//                 slot 8g + r is row 4g + r of the first tile (r < 4) or 4g + r - 4 of the second, so
//                 the weights are in place where the scores came out.  Lane (i, g) loads those eight
//                 rows' columns i * HDB/16 .. (16 lanes cover a row, whole lines), and one v_perm per
//                 pair of rows gives the operands of HDB/16 products, column m of every lane in the m-th.
// The next 32 rows' K and V are requested as soon as their registers are free.  The softmax keeps a
// maximum per head and moves it rarely (kSlack), and each lane its own part of the sum, so the loop has
// no exchange between lanes.  The four waves of a workgroup take every fourth tile pair and join in LDS.
//
// One sequence of 131072 rows, 32/4 heads of 128, bf16: 57 us with the join, 4.7 TB/s (a 1 GiB copy reaches
// 5.1); eight of 2048 to 4096, 64/8 heads of 64, 16.7 us, of which the join and the launches are 6.  e4m3, 32/8 heads
// of 128: 48 sequences of 9000 rows each 172 us, 5.2 TB/s, whatever the pool's order; 48 of up to 9000, 108 MB in
// all, 43 us, 2.5 TB/s: the join (7 us) and the start of the workgroups weigh more, equal lengths of that sum take 38
// us, on a [page][head][row] pool 32 (unequal 41).  L2 misses are the same in all four.  Tried: the
// splits of all sequences in one list that 1024 workgroups walk (10 % slower: a scan of the lengths before each),
// heads fastest in the launch order (12 % slower there, 6 % faster with eight equal sequences), three waves a SIMD
// (no change), two tiles in flight a wave where the registers allow it (e4m3 43 -> 48 us, two waves a SIMD then).
//
// HP: q and the weights in planes that hold fp32's precision (each product once per plane); else q is
// 16 bits as it is, and the weights take two planes all the same: the loop stays bound by memory, and
// one plane's rounding is as large as the output's own.  PU: pages of a multiple of 16 rows: a tile lies in one page, whose
// number comes through the scalar cache two steps ahead; else every lane looks its row up.
template <int CT, bool HP, int HDB, bool PU>
__global__ __launch_bounds__(256, HDB == 256 || (HP && HDB == 128) ? 1 : 2) void k_pa_decode(pa_args a)
{
    constexpr bool E8 = CT == MLLM_E4M3;
    constexpr int ES = E8 ? 1 : 2, NP = HP ? kPlanes<CT> : 1, NW = HP ? kPlanes<CT> : 2;   // planes of q, of the weights
    constexpr int KS = HDB / 32;                     // 16x16x32 products per tile of scores
    constexpr int KW = E8 ? KS / 2 : KS;             // 16-byte loads per K row and lane
    constexpr int NM = HDB / 16;                     // columns per lane of V
    constexpr int VW = NM * ES / 4;                  // words per lane of a V row
    constexpr int LD = HDB + 4;                      // floats per head in LDS
    extern __shared__ __attribute__((aligned(16))) float lds[];
    __shared__ float sm[4][16], sl[4][16];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.z, sp = blockIdx.x, j = blockIdx.y / a.groups, hg = blockIdx.y - j * a.groups;
    const int G = min(16, a.rep - 16 * hg), h0 = j * a.rep + 16 * hg, HD = a.kv.head_dim;
    const int seq = a.seqs ? a.seqs[b] : b;
    int len = min(a.lens[b], a.max_len);
    if (seq < 0 || seq >= a.kv.n_seqs) len = 0;
    len = min(len, (int)min((long)a.kv.max_blocks * a.kv.page_size, 0x7FFFFFFFl));
    // a length past the tables: the rows behind them are unmapped, so the window is still the query's
    const int lo = a.window > 0 ? max(0, min(a.lens[b], a.max_len) - a.window) : 0;
    const int begin = lo / 32 * 32 + sp * a.chunk, end = min(len, begin + a.chunk);
    if (begin >= end && a.splits > 1) {              // nothing here: the join reads only the sum
        if ((int)threadIdx.x < G)
            *(float2 *)(a.stat + (((long)b * a.NH + h0 + threadIdx.x) * a.splits + sp) * 2) = make_float2(kLowest, 0.0f);
        return;
    }

    // the query, in the order of K's operands
    uint4 qf[NP][KS];
    float zs = a.scale * kLog2e;
    {
        const long at = b * a.q_ld + (long)(h0 + min(i, G - 1)) * HD;
        float q[KS][8], big = 0.0f;
#pragma unroll
        for (int c = 0; c < KS; c++) {
            const int col = E8 ? 64 * (c >> 1) + 16 * g + 8 * (c & 1) : 32 * c + 8 * g;
            load8(a.q, at + min(col, HD - 8), a.q_type, true, q[c]);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (col >= HD) q[c][e] = 0.0f;
                big = fmaxf(big, fabsf(q[c][e]));
            }
        }
        if constexpr (HP && CT == MLLM_F16) {
            // fp16 planes: the head's largest element to [2^14, 2^15)
            big = fmaxf(big, __shfl_xor(big, 16, 64));
            big = fmaxf(big, __shfl_xor(big, 32, 64));
            const int e = big > 0.0f && big < INFINITY ? 15 - (int)((__float_as_uint(big) >> 23) & 255) + 126 : 0;
            zs = ldexpf(zs, -e);
#pragma unroll
            for (int c = 0; c < KS; c++)
#pragma unroll
                for (int x = 0; x < 8; x++) q[c][x] = ldexpf(q[c][x], e);
        }
#pragma unroll
        for (int c = 0; c < KS; c++) {
            uint32_t p[4][NP];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                pa_planes<CT, NP>(q[c][2 * x], q[c][2 * x + 1], p[x]);
#pragma unroll
                for (int n = 1; n < NP; n++) {       // an infinity's rest is 0
                    if (!(fabsf(q[c][2 * x]) < INFINITY)) p[x][n] &= 0xFFFF0000u;
                    if (!(fabsf(q[c][2 * x + 1]) < INFINITY)) p[x][n] &= 0xFFFFu;
                }
            }
#pragma unroll
            for (int n = 0; n < NP; n++) qf[n][c] = make_uint4(p[0][n], p[1][n], p[2][n], p[3][n]);
        }
    }

    // offsets in a row (bytes); columns past head_dim read its start (q is 0 there, and V's are not stored)
    unsigned kcol[KW], vcol[HDB == 256 ? 2 : 1];
#pragma unroll
    for (int c = 0; c < KW; c++) {
        const int col = E8 ? 64 * c + 16 * g : 32 * c + 8 * g;
        kcol[c] = (col < HD ? col : 0) * ES;
    }
#pragma unroll
    for (int c = 0; c < (HDB == 256 ? 2 : 1); c++) {
        const int col = HDB == 64 ? 4 * i : 128 * c + 8 * i;
        vcol[c] = (col < HD ? col : 0) * ES;
    }
    const long rs = a.kv.row_stride * ES, ps = a.kv.page_stride * ES, hs = a.kv.head_stride * ES * j;
    const uint8_t *kb = (const uint8_t *)a.kv.k + hs, *vb = (const uint8_t *)a.kv.v + hs;

    // rows s0 .. s0 + 31: where they are, and which the query sees
    struct place {
        long t0, t1;                                 // PU: tile's first row; else this lane's row (lane % 32)
        long e0, e1;                                 // the same among the exponents
        uint32_t ok;
    };
    auto find = [&](int s0) __attribute__((always_inline)) {
        place p;
        if constexpr (PU) {
            p.ok = 0;
            long t[2], e[2];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int s = s0 + 16 * n, blk = pa_block(a, s);
                const int pg = pa_table(a, seq, min(blk, a.kv.max_blocks - 1));
                const bool on = s < len && pg >= 0 && pg < a.kv.n_pages;
                const int row = on ? s - blk * a.kv.page_size : 0;
                t[n] = (on ? pg : 0) * ps + row * rs;
                e[n] = ((on ? pg : 0) * (long)a.kv.n_kv_head + j) * a.kv.page_size + row;
                if (on) p.ok |= 0xFFFFu << (16 * n);
            }
            p.t0 = t[0]; p.t1 = t[1]; p.e0 = e[0]; p.e1 = e[1];
        } else {
            const int s = s0 + (lane & 31), blk = pa_block(a, s);
            int pg = -1;
            if (s < len && blk < a.kv.max_blocks) pg = a.kv.tables[(long)seq * a.kv.table_ld + blk];
            const bool on = pg >= 0 && pg < a.kv.n_pages;
            const int row = on ? s - blk * a.kv.page_size : 0;
            p.t0 = p.t1 = (on ? pg : 0) * ps + row * rs;
            p.e0 = p.e1 = ((on ? pg : 0) * (long)a.kv.n_kv_head + j) * a.kv.page_size + row;
            p.ok = (uint32_t)__ballot(on);
        }
        const int n = end - s0, f = lo - s0;         // rows before f and from n on are not the query's
        if (n < 32) p.ok &= (1u << (n > 0 ? n : 0)) - 1;
        if (f > 0) p.ok &= f < 32 ? ~0u << f : 0;
        return p;
    };
    uint4 kr[2][KW];
    uint32_t vr[8][VW], ke[2], ve[8];
    auto load_k = [&](const place &p) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const uint8_t *r;
            if constexpr (PU) r = kb + (n ? p.t1 : p.t0) + (unsigned)(i * (unsigned)rs);
            else r = kb + __shfl(p.t0, 16 * n + i, 64);
#pragma unroll
            for (int c = 0; c < KW; c++) kr[n][c] = *(const uint4 *)(r + kcol[c]);
            if constexpr (E8) {
                if constexpr (PU) ke[n] = a.kv.k_exp[(n ? p.e1 : p.e0) + i];
                else ke[n] = a.kv.k_exp[__shfl(p.e0, 16 * n + i, 64)];
            }
        }
    };
    auto load_v = [&](const place &p) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 8; r++) {
            const uint8_t *row;
            if constexpr (PU) row = vb + (r < 4 ? p.t0 : p.t1) + (unsigned)((4 * g + (r & 3)) * (unsigned)rs);
            else row = vb + __shfl(p.t0, (r < 4 ? 0 : 16) + 4 * g + (r & 3), 64);
            if constexpr (VW == 1) vr[r][0] = *(const uint32_t *)(row + vcol[0]);
            if constexpr (VW == 2) { const uint2 x = *(const uint2 *)(row + vcol[0]); vr[r][0] = x.x; vr[r][1] = x.y; }
            if constexpr (VW == 4 && HDB != 256) {
                const uint4 x = *(const uint4 *)(row + vcol[0]);
                vr[r][0] = x.x; vr[r][1] = x.y; vr[r][2] = x.z; vr[r][3] = x.w;
            }
            if constexpr (HDB == 256) {
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    if constexpr (E8) {
                        const uint2 x = *(const uint2 *)(row + vcol[c]);
                        vr[r][2 * c] = x.x; vr[r][2 * c + 1] = x.y;
                    } else {
                        const uint4 x = *(const uint4 *)(row + vcol[c]);
                        vr[r][4 * c] = x.x; vr[r][4 * c + 1] = x.y; vr[r][4 * c + 2] = x.z; vr[r][4 * c + 3] = x.w;
                    }
                }
            }
            if constexpr (E8 && !PU) ve[r] = a.kv.v_exp[__shfl(p.e0, (r < 4 ? 0 : 16) + 4 * g + (r & 3), 64)];
        }
        if constexpr (E8 && PU) {
            // four rows' exponents in a word (pages and the array are multiples of 4 there)
            const uint32_t x = *(const uint32_t *)(a.kv.v_exp + p.e0 + 4 * g), y = *(const uint32_t *)(a.kv.v_exp + p.e1 + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; r++) { ve[r] = x >> (8 * r); ve[4 + r] = y >> (8 * r); }
        }
    };

    float m = kLowest, l = 0.0f;
    f32x4 o[NM] = {};
    int s0 = begin + 32 * w;
    if (s0 < end) {
        place cur = find(s0), nxt = find(min(s0 + 128, end - 1) / 32 * 32);
        load_k(cur);
        load_v(cur);
        for (;;) {
            const bool more = s0 + 128 < end;
            f32x4 s[2];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                s[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                const float sc = E8 ? pa_exp8(ke[n]) : 1.0f;
#pragma unroll
                for (int c = 0; c < KS; c++) {
                    uint4 k;
                    if constexpr (E8) {
                        const uint4 x = kr[n][c >> 1];
                        const uint32_t u = c & 1 ? x.z : x.x, v = c & 1 ? x.w : x.y;
                        k = make_uint4(pa_cvt8<false>(u, sc), pa_cvt8<true>(u, sc), pa_cvt8<false>(v, sc), pa_cvt8<true>(v, sc));
                    } else {
                        k = kr[n][c];
                    }
#pragma unroll
                    for (int x = NP - 1; x >= 0; x--) s[n] = pa_mfma16<CT>(k, qf[x][c], s[n]);
                }
            }
            const place now = cur;
            if (more) load_k(nxt);
            cur = nxt;
            if (more) nxt = find(min(s0 + 256, end - 1) / 32 * 32);
            float z[8], top = kLowest;
#pragma unroll
            for (int r = 0; r < 8; r++) z[r] = s[r >> 2][r & 3] * zs;
            const bool all = now.ok == 0xFFFFFFFFu;
            if (!all) {
#pragma unroll
                for (int r = 0; r < 8; r++)
                    if (!(now.ok >> ((r < 4 ? 0 : 16) + 4 * g + (r & 3)) & 1)) z[r] = -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 8; r++) top = fmaxf(top, z[r]);
            if (__any(top > m + kSlack)) {
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(fmaxf(top, __shfl_xor(top, 32, 64)), m);
                const float f = __builtin_amdgcn_exp2f(m - top);
                m = top;
                l *= f;
#pragma unroll
                for (int x = 0; x < NM; x++) o[x] *= f;
            }
            uint32_t pw[4][NW];
#pragma unroll
            for (int r = 0; r < 8; r++) {
                z[r] = __builtin_amdgcn_exp2f(z[r] - (m - kBias<CT>));
                l += z[r];
            }
#pragma unroll
            for (int x = 0; x < 4; x++) pa_planes<CT, NW, true>(z[2 * x], z[2 * x + 1], pw[x]);
            if (!all) {                              // what lies in rows that are not the query's may be NaN
#pragma unroll
                for (int r = 0; r < 8; r++)
                    if (!(now.ok >> ((r < 4 ? 0 : 16) + 4 * g + (r & 3)) & 1)) {
#pragma unroll
                        for (int x = 0; x < VW; x++) vr[r][x] = 0;
                        ve[r] = 127;
                    }
            }
#pragma unroll
            for (int x = 0; x < NM / 2; x++) {       // columns 2x, 2x + 1 of every lane
                uint32_t v[8];
#pragma unroll
                for (int r = 0; r < 8; r++) {
                    if constexpr (E8) v[r] = x & 1 ? pa_cvt8<true>(vr[r][x >> 1], pa_exp8(ve[r])) : pa_cvt8<false>(vr[r][x >> 1], pa_exp8(ve[r]));
                    else v[r] = vr[r][x];
                }
#pragma unroll
                for (int hi = 0; hi < 2; hi++) {
                    uint32_t f[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) f[r] = __builtin_amdgcn_perm(v[2 * r + 1], v[2 * r], hi ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int n = NW - 1; n >= 0; n--)
                        o[2 * x + hi] = pa_mfma16<CT>(make_uint4(f[0], f[1], f[2], f[3]),
                                                      make_uint4(pw[0][n], pw[1][n], pw[2][n], pw[3][n]), o[2 * x + hi]);
                }
            }
            if (!more) break;
            load_v(cur);
            s0 += 128;
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    l *= kPlanesSum;

    // the four waves' parts
    if (g == 0) { sm[w][i] = m; sl[w][i] = l; }
    __syncthreads();
    const float top = fmaxf(fmaxf(sm[0][i], sm[1][i]), fmaxf(sm[2][i], sm[3][i]));
    const float f = __builtin_amdgcn_exp2f(m - top);
    if (i < G) {
        float *row = lds + (w * G + i) * LD;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int x = 0; x < NM; x += 4) {
                const int d = HDB == 64 ? 4 * (4 * g + r) : (x >> 3) * 128 + 8 * (4 * g + r) + (x & 7);
                *(float4 *)(row + d) = make_float4(o[x][r] * f, o[x + 1][r] * f, o[x + 2][r] * f, o[x + 3][r] * f);
            }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < G * (HD / 4); x += 256) {
        const int h = x / (HD / 4), d = 4 * (x - h * (HD / 4));
        const float mh = fmaxf(fmaxf(sm[0][h], sm[1][h]), fmaxf(sm[2][h], sm[3][h]));
        float lh = 0.0f;
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int n = 0; n < 4; n++) {
            lh += sl[n][h] * __builtin_amdgcn_exp2f(sm[n][h] - mh);
            const float4 u = *(const float4 *)(lds + (n * G + h) * LD + d);
            y.x += u.x; y.y += u.y; y.z += u.z; y.w += u.w;
        }
        const long row = (long)b * a.NH + h0 + h;
        if (a.splits > 1) {
            *(float4 *)(a.part + (row * a.splits + sp) * HD + d) = y;
            if (d == 0) *(float2 *)(a.stat + (row * a.splits + sp) * 2) = make_float2(mh, lh);
        } else {
            pa_finish(a, h0 + h, b, d, mh, lh, y);
        }
    }
}

template <int CT, bool HP, int HDB, bool PU> static void pa_decode_go(const pa_args &a, hipStream_t st)
{
    const int G = a.rep < 16 ? a.rep : 16;
    hipLaunchKernelGGL((k_pa_decode<CT, HP, HDB, PU>), dim3(a.splits, a.kv.n_kv_head * a.groups, a.B), dim3(256),
                       (size_t)4 * G * (HDB + 4) * 4, st, a);
}
template <int CT, bool HP, int HDB> static void pa_decode_pu(const pa_args &a, bool uniform, hipStream_t st)
{
    uniform ? pa_decode_go<CT, HP, HDB, true>(a, st) : pa_decode_go<CT, HP, HDB, false>(a, st);
}
template <int CT, bool HP> static void pa_decode_hd(const pa_args &a, bool uniform, hipStream_t st)
{
    const int HD = a.kv.head_dim;
    HD <= 64 ? pa_decode_pu<CT, HP, 64>(a, uniform, st) : HD <= 128 ? pa_decode_pu<CT, HP, 128>(a, uniform, st)
                                                                    : pa_decode_pu<CT, HP, 256>(a, uniform, st);
}
template <int CT> static void pa_decode(const pa_args &a, bool wide, bool uniform, hipStream_t st)
{
    wide ? pa_decode_hd<CT, true>(a, uniform, st) : pa_decode_hd<CT, false>(a, uniform, st);
}
