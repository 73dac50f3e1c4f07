// pattn_prompt.h — the tiled prompt kernel over a paged cache, instantiated per cache type.
#pragma once
#include <math.h>
#include <type_traits>
#include "pattn.h"

template <int CT> __device__ __forceinline__ f32x16 pa_mfma32(uint4 x, uint4 y, f32x16 c)
{
    if constexpr (CT == MLLM_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}

// A tile of 64, 128 or 256 rows of queries against the rows of one kv head, 64 of these at a time (32 at
// head sizes above 128).  A row is a (token, head) pair of the heads that share the kv head, tokens outer,
// so a tile of K and V serves all of them and a few drafted tokens fill a wave.  RG groups of 32 rows; a
// group is one wave's, or two waves share it: KH, each takes half of every step's rows of K and V, and
// they join at the end; above head size 128, each takes half of the output's columns.
//   S^T = K Q^T   (32x32x16): q stays in registers as the second operand; a lane holds half of the
//                 scores of one row (lane % 32), so maximum and sum are the lane's own
//   O^T += V^T P  the scores' registers are this product's second operand as they stand: slot
//                 8 (lane / 32) + e of its k index is row 8 (e / 4) + 4 (lane / 32) + e % 4, and V's
//                 operand is read transposed from LDS (ds_read_b64_tr_b16) in the same order
// K and V go straight to LDS, one step ahead, in two buffers (separate objects: a wait for one is no
// wait for the other); 16-byte pieces are permuted within their row so that the operand reads of 16
// lanes (K: 16 rows; V: 4 rows of 64 bytes) fall on distinct banks.  8-bit caches pass through
// registers, where they become bf16.
//
// HP (fp32 q or out): q and the weights in planes that hold fp32's precision, three products for one (two
// in fp16).  Else q is 16 bits as it is, and the weights take two planes, as in decode: rounded to one they
// raise the error against 64 bits to 1.3 times that of the output rounded alone (6011 tokens, bf16, 2.16e-3
// for 1.64e-3, 326 us for 418; prompts of 1 to 1100 tokens, fp16, 2.9e-4 for 2.1e-4, 30 us for 33).
//
// A weight of 0 times an infinity or a NaN that a masked row of V holds is NaN, so in the steps where
// some row of the tile is masked V is looked through for such rows; they are cleared in LDS and added
// element by element to the queries that do see them.
//
// One prompt of 6011 tokens, 32/8 heads of 128, bf16: 418 to 431 us on three cards, 697 TFLOP/s of the operator's
// operations, 1046 with the weights' second plane (a bf16 product of 8192^3 reaches 1288).  Per step of 32 x 64 scores a wave
// issues 48 matrix instructions (1536 cycles) and about 275 vector ones (32 exponentials among them, at a quarter of
// the rate), and the two hardly overlap on a SIMD: some 6000 cycles for its two waves (matrix cores busy 47 % of the
// kernel's cycles).  The operand reads are issued ahead, but the waits, five a step, are for all of them at once: a part of
// that lead is lost.  Tried, with one plane of weights (a step 4300 cycles of 4900 measured): three or four buffers
// instead of two 1 to 2 % slower (the loads are hidden by then), 32-row steps 6 %, the sum of the weights by v_dot2
// 16 % (it issues slowly), scores two waves a SIMD without the order of LDS reads fixed below 10 %, the page looked up
// by a vector load 5 %, matrix instructions at a higher wave priority 1 % faster or slower.
template <int CT, bool HP, int HDB, int RG, int KH, int EV>
__global__ __launch_bounds__(64 * RG * KH * pa_parts(HDB), HP && HDB > 64 || RG * KH * pa_parts(HDB) == 8 ? 1 : 2) void k_pa_prompt(pa_args a)
{
    constexpr bool E8 = CT == MLLM_E4M3;
    constexpr int ES = E8 ? 1 : 2, NP = HP ? kPlanes<CT> : 1, PW = HP ? kPlanes<CT> : 2;   // planes of q, of the weights
    constexpr int DH = pa_parts(HDB), NW = RG * KH * DH, ROWS = 32 * RG;
    static_assert(KH == 1 || DH == 1, "a row group has at most two waves");
    constexpr int TK = HDB > 128 ? 32 : 64, TW = TK / KH, NB = TW / 32;   // rows per step, and of them a wave's, in blocks of 32
    constexpr int KS = HDB / 16, OB = HDB / 32 / DH;         // K's operands per row, V's (of a wave's columns)
    constexpr int RB = HDB * 2;                              // bytes of a row in LDS
    constexpr int LPR = HDB * ES / 16, RI = 64 / LPR, WR = TK / NW, NI = WR / RI;   // lanes per row, rows per load, rows and loads per wave
    __shared__ __attribute__((aligned(1024))) uint8_t k0[TK * RB], v0[TK * RB], k1[TK * RB], v1[TK * RB];
    __shared__ uint32_t odd[2][NW];                          // of a wave's rows of V: those that hold an infinity or a NaN
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hh = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), rg = w % RG, kh = KH > 1 ? w / RG : 0, dh = DH > 1 ? w / RG : 0;
    const int NKH = a.kv.n_kv_head, j = blockIdx.x % NKH, HD = a.kv.head_dim, sp = blockIdx.y, rep = a.rep;

    auto start = [&](int x) { return max(0, min(a.starts[x], a.T)); };
    // which sequence and tile: 64 sequences at a time
    int t = blockIdx.x / NKH, b = -1, tiles = 0;
    for (int b0 = 0; b0 < a.B && b < 0; b0 += 64) {
        const int bb = b0 + lane;
        const int n = bb < a.B ? (max(0, start(bb + 1) - start(bb)) * rep + ROWS - 1) / ROWS : 0;
        int sum = n;
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(sum, d, 64);
            if (lane >= d) sum += y;
        }
        const unsigned long long in = __ballot(t < sum);
        if (in) {
            const int f = __builtin_ctzll(in);
            b = b0 + f;
            tiles = __shfl(n, f, 64);
            t -= __shfl(sum, f, 64) - tiles;
        } else {
            t -= __shfl(sum, 63, 64);
        }
    }
    if (b < 0) return;
    b = __builtin_amdgcn_readfirstlane(b);
    const int tile = __builtin_amdgcn_readfirstlane(tiles - 1 - t);     // the last rows, which see most, first
    const int q0 = start(b), nq = start(b + 1) - q0;
    const int seq = a.seqs ? a.seqs[b] : b;
    const int len0 = min(a.lens[b], a.max_len);
    int len = seq >= 0 && seq < a.kv.n_seqs ? len0 : 0;
    len = min(len, (int)min((long)a.kv.max_blocks * a.kv.page_size, 0x7FFFFFFFl));
    const int nrows = min(ROWS, nq * rep - tile * ROWS);     // of the tile (queries times heads are below 2^30)
    const int first = (unsigned)(tile * ROWS) / (unsigned)rep, last = (unsigned)(tile * ROWS + nrows - 1) / (unsigned)rep;   // tokens
    // positions of a token's query: len0 - nq + token; it sees (p - window, p]
    const int off = len0 - nq;
    const int lo = a.window > 0 ? max(0, off + first - a.window + 1) : 0, hi = min(len, off + last + 1);
    const int begin = lo / TK * TK + sp * a.chunk, end = min(hi, begin + a.chunk);
    // this lane's row
    const int rr = 32 * rg + c, r = min(rr, nrows - 1), tok = (int)((unsigned)(tile * ROWS + r) / (unsigned)rep), h = j * rep + (int)((tile * ROWS + r) - tok * rep);
    const int pr = off + tok, lr = a.window > 0 ? max(0, pr - a.window + 1) : 0;
    // The rows that all of the workgroup's queries see, [full_begin, full_end); of the wave's: those that some
    // sees, [lmin, pmax], and that all see, [lmax, wave_end)
    const int full_begin = a.window > 0 ? off + last - a.window + 1 : 0, full_end = min(off + first + 1, len);
    const int wtok0 = (int)((unsigned)(tile * ROWS + min(32 * rg, nrows - 1)) / (unsigned)rep), wtok1 = (int)((unsigned)(tile * ROWS + min(32 * rg + 31, nrows - 1)) / (unsigned)rep);
    const int pmax = 32 * rg < nrows ? off + wtok1 : -1, lmax = a.window > 0 ? max(0, off + wtok1 - a.window + 1) : 0;
    const int lmin = a.window > 0 ? max(0, off + wtok0 - a.window + 1) : 0, wave_end = min(off + wtok0 + 1, len);
    const long orow = (long)(q0 + tok) * a.NH + h;

    if (begin >= end && a.splits > 1) {
        if (hh == 0 && kh == 0 && dh == 0 && rr < nrows) *(float2 *)(a.stat + (orow * a.splits + sp) * 2) = make_float2(kLowest, 0.0f);
        return;
    }

    uint4 qf[NP][KS];
    float zs = fabsf(a.scale) * kLog2e;                      // its sign goes into q: the largest product is the largest score
    {
        const long at = (long)(q0 + tok) * a.q_ld + (long)h * HD;
        int e = 0;
        if constexpr (HP && CT == MLLM_F16) {
            // fp16 planes: the row's largest element to [2^14, 2^15)
            float big = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                float x[8];
                load8(a.q, at + min(16 * s + 8 * hh, HD - 8), a.q_type, true, x);
#pragma unroll
                for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(x[i]));
            }
            big = fmaxf(big, __shfl_xor(big, 32, 64));
            e = big > 0.0f && big < INFINITY ? 15 - (int)((__float_as_uint(big) >> 23) & 255) + 126 : 0;
            zs = ldexpf(zs, -e);
        }
        zs = fmaxf(zs, 1e-37f);                              // masked scores, -inf, times it stay -inf
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int col = 16 * s + 8 * hh;
            float x[8];
            load8(a.q, at + min(col, HD - 8), a.q_type, true, x);
            uint32_t p[4][NP];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float u = col < HD ? x[2 * i] : 0.0f, v = col < HD ? x[2 * i + 1] : 0.0f;
                if constexpr (HP && CT == MLLM_F16) { u = ldexpf(u, e); v = ldexpf(v, e); }
                if (a.scale < 0.0f) { u = -u; v = -v; }
                pa_planes<CT, NP>(u, v, p[i]);
#pragma unroll
                for (int n = 1; n < NP; n++) {               // an infinity's rest is 0
                    if (!(fabsf(u) < INFINITY)) p[i][n] &= 0xFFFF0000u;
                    if (!(fabsf(v) < INFINITY)) p[i][n] &= 0xFFFFu;
                }
            }
#pragma unroll
            for (int n = 0; n < NP; n++) qf[n][s] = make_uint4(p[0][n], p[1][n], p[2][n], p[3][n]);
        }
    }

    // ---- staging.  Row x's 16-byte piece y of K lies at piece y ^ kx(x), of V at y ^ vx(x).
    auto kx = [](int x) { return HDB == 64 ? (x >> 1) & 7 : x & 15; };
    auto vx = [](int x) { return HDB == 64 ? (x >> 1 & 1) << 2 : (x & 3) << 2; };
    const long rs = a.kv.row_stride * ES, ps = a.kv.page_stride * ES, hs = a.kv.head_stride * ES * j;
    const uint8_t *kb = (const uint8_t *)a.kv.k + hs, *vb = (const uint8_t *)a.kv.v + hs;
    const int lrow = lane / LPR, lpc = lane & (LPR - 1);     // row of a load and piece
    // The pages of a step's rows, looked up a step before they are used.
    //   EV 2: a step lies in one page (p0; block and row are counted on from step to step)
    //   EV 1: every 16 rows do, and so do a wave's; 0: p0 is the page of row s0 + lane.
    struct pages { int p0, p1, p2, p3; };
    // all ones for the 16 rows that the wave brings
    const int own0 = WR * w / 16 == 0 ? -1 : 0, own1 = WR * w / 16 == 1 ? -1 : 0, own2 = WR * w / 16 == 2 ? -1 : 0,
              own3 = WR * w / 16 == 3 ? -1 : 0;
    const int blk0 = EV == 2 && begin < end ? pa_block(a, begin) : 0;
    int nblk = blk0, nrow = begin - blk0 * a.kv.page_size, row0 = nrow;   // EV 2: of the looked-up step; row0: in p0
    auto look = [&](int s0) __attribute__((always_inline)) {
        pages g{};
        if constexpr (EV == 2) {
            g.p0 = pa_table(a, seq, nblk);
        } else if constexpr (EV == 1) {
            auto page = [&](int s) { return pa_table(a, seq, min(pa_block(a, s), a.kv.max_blocks - 1)); };
            g.p0 = page(s0);
            g.p1 = page(s0 + 16);
            if constexpr (TK == 64) { g.p2 = page(s0 + 32); g.p3 = page(s0 + 48); }
        } else {
            const int s = s0 + (lane & (TK - 1)), blk = pa_block(a, s);
            g.p0 = s < len && blk < a.kv.max_blocks ? a.kv.tables[(long)seq * a.kv.table_ld + blk] : -1;
        }
        return g;
    };
    // Bits: rows of the step on mapped pages (those past the length count as mapped).
    constexpr uint64_t ALL = TK == 64 ? ~0ull : 0xFFFFFFFFull;
    auto mapped = [&](int s0, const pages &g) __attribute__((always_inline)) {
        uint64_t on = 0;
        auto is = [&](int s, int p) { return s >= len || (unsigned)p < (unsigned)a.kv.n_pages; };
        if constexpr (EV == 2) {
            if (is(s0, g.p0)) on = ALL;
        } else if constexpr (EV == 1) {
            if (is(s0, g.p0)) on |= 0xFFFFull;
            if (is(s0 + 16, g.p1)) on |= 0xFFFFull << 16;
            if (is(s0 + 32, g.p2)) on |= 0xFFFFull << 32;
            if (is(s0 + 48, g.p3)) on |= 0xFFFFull << 48;
        } else {
            on = __ballot(is(s0 + (lane & (TK - 1)), g.p0));
        }
        return on & ALL;
    };
    // this lane's pieces of its rows: bytes from the wave's first row (EV) or in the row; columns past head_dim
    // read the row's start
    unsigned pk_[NI], pv_[NI];
#pragma unroll
    for (int n = 0; n < NI; n++) {
        const int x = WR * w + RI * n + lrow;
        const int ck = 16 * (E8 ? lpc : lpc ^ kx(x)), cv = 16 * (E8 ? lpc : lpc ^ vx(x));
        const unsigned o = EV ? (RI * n + lrow) * (unsigned)rs : 0;
        pk_[n] = o + (ck < HD * ES ? ck : 0);
        pv_[n] = o + (cv < HD * ES ? cv : 0);
    }
    uint4 sk[E8 ? NI : 1], sv[E8 ? NI : 1];
    uint32_t se[2][E8 ? NI : 1];
    // The wave's part of the step at s0, always 2 NI loads.  Rows past the length read what their page holds (with
    // EV 0 the pool's first row), rows on no page the pool's first: it is masked, and looked through like every edge.
    auto fetch = [&](int s0, const pages &g, uint8_t *kl, uint8_t *vl) __attribute__((always_inline)) {
        const int mine = s0 + WR * w;
        long at = 0, ex = 0;
        if constexpr (EV) {
            const int pg = EV == 2 ? g.p0 : (g.p0 & own0) | (g.p1 & own1) | (g.p2 & own2) | (g.p3 & own3);
            const int row = EV == 2 ? row0 + WR * w : mine - pa_block(a, mine) * a.kv.page_size;
            if (mine < len && (unsigned)pg < (unsigned)a.kv.n_pages) {
                at = pg * ps + row * rs;
                ex = (pg * (long)NKH + j) * a.kv.page_size + row;
            }
        } else {
            const int s = s0 + (lane & (TK - 1)), row = s - pa_block(a, s) * a.kv.page_size;
            if (s < len && (unsigned)g.p0 < (unsigned)a.kv.n_pages) {
                at = g.p0 * ps + row * rs;
                ex = (g.p0 * (long)NKH + j) * a.kv.page_size + row;
            }
        }
        const uint8_t *bk = kb + at, *bv = vb + at;
#pragma unroll
        for (int n = 0; n < NI; n++) {
            const int x = RI * n + lrow;
            const uint8_t *gk, *gv;
            long e = ex + x;
            if constexpr (EV) {
                gk = bk + pk_[n];
                gv = bv + pv_[n];
            } else {
                const long r = __shfl(at, WR * w + x, 64);
                gk = kb + r + pk_[n];
                gv = vb + r + pv_[n];
                e = __shfl(ex, WR * w + x, 64);
            }
            if constexpr (E8) {
                sk[n] = *(const uint4 *)gk;
                sv[n] = *(const uint4 *)gv;
                se[0][n] = a.kv.k_exp[e];
                se[1][n] = a.kv.v_exp[e];
            } else {
                const int to = (WR * w + RI * n) * RB;       // the load's 1 KB
                __builtin_amdgcn_global_load_lds(gk, (__attribute__((address_space(3))) void *)(kl + to), 16, 0, 0);
                __builtin_amdgcn_global_load_lds(gv, (__attribute__((address_space(3))) void *)(vl + to), 16, 0, 0);
            }
        }
    };
    auto store = [&](uint8_t *kl, uint8_t *vl) __attribute__((always_inline)) {
        if constexpr (E8) {
#pragma unroll
            for (int n = 0; n < NI; n++) {
                const int x = WR * w + RI * n + lrow;
#pragma unroll
                for (int z = 0; z < 2; z++) {
                    const uint4 u = z ? sv[n] : sk[n];
                    const float f = pa_exp8(se[z][n]);
                    uint8_t *row = (z ? vl : kl) + x * RB;
                    const int y = z ? vx(x) : kx(x);
                    *(uint4 *)(row + 16 * ((2 * lpc) ^ y)) = make_uint4(pa_cvt8<false>(u.x, f), pa_cvt8<true>(u.x, f), pa_cvt8<false>(u.y, f), pa_cvt8<true>(u.y, f));
                    *(uint4 *)(row + 16 * ((2 * lpc + 1) ^ y)) = make_uint4(pa_cvt8<false>(u.z, f), pa_cvt8<true>(u.z, f), pa_cvt8<false>(u.w, f), pa_cvt8<true>(u.w, f));
                }
            }
        }
    };

    float m = kLowest, l0 = 0.0f, l1 = 0.0f;               // the sum in two parts: shorter chains
    f32x16 o[OB] = {};
    const int tr = (lane & 15) >> 2;                         // V operand: row of four, 8-byte piece of 32 bytes
    // K operand: row c (+ 32 n), piece 2 s + hh; V operand: row 4 hh + tr (+ 16 t, + 8), columns 32 x + 16 (lane / 16 % 2) + 4 (lane % 4)
    const int kbase = (TW * kh + c) * RB, kxor = kx(c);
    const int vbase = (TW * kh + 4 * hh + tr) * RB + 8 * (lane & 1), vpc = 2 * (lane >> 4 & 1) + (lane >> 1 & 1), vxor = vx(4 * hh + tr);

    auto work = [&](int s0, bool holes, uint8_t *kl, uint8_t *vl, int par) __attribute__((always_inline)) {
        // some row of the workgroup's is masked somewhere in this step
        if (EV == 2 && holes) return;                        // none of the step's rows is there
        const bool edge = s0 + TK > full_end || s0 < full_begin || (EV < 2 && holes);
        uint64_t bad = 0;
        if (edge) {                                          // the wave looks through its part of V
            uint32_t mine = 0;
            constexpr int PCS = RB / 16;                     // pieces per row
#pragma unroll
            for (int n = 0; n < WR * PCS / 64; n++) {
                const int x = WR * w + (64 * n + lane) / PCS, y = (64 * n + lane) % PCS;
                const uint4 u = *(const uint4 *)(vl + x * RB + 16 * y);
                constexpr uint32_t E = CT == MLLM_F16 ? 0x7C00u : 0x7F80u;
                auto f = [&](uint32_t q) { return (q & E) == E || (q >> 16 & E) == E; };
                const uint64_t any = __ballot(f(u.x) || f(u.y) || f(u.z) || f(u.w));
#pragma unroll
                for (int z = 0; z < 64 / PCS; z++)
                    if (any >> (z * PCS) & (PCS == 64 ? ~0ull : (1ull << PCS) - 1)) mine |= 1u << (64 / PCS * n + z);
            }
            if (lane == 0) odd[par][w] = mine;
            __syncthreads();
#pragma unroll
            for (int z = 0; z < NW; z++) bad |= (uint64_t)odd[par][z] << (WR * z);
            bad = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)bad) | (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(bad >> 32)) << 32;
            if (bad) {
                __syncthreads();
                for (int x = 0; x < WR; x++)
                    if (bad >> (WR * w + x) & 1)
                        for (int y = lane; y < RB / 4; y += 64) *(uint32_t *)(vl + (WR * w + x) * RB + 4 * y) = 0;
                __syncthreads();
            }
        }
        const int sw = s0 + TW * kh;                         // the wave's rows of K and V
        if (sw > pmax || sw + TW <= lmin) return;            // nothing that the wave's queries see
        // Operands are read from LDS ahead of the products that take them: K's two products' worth (KD), V's
        // a group of VG; the scheduler is held to that order, or it issues each read right before its use.
        constexpr int KD = KS < 2 ? 1 : 2;
        f32x16 s[NB] = {};
        uint4 kf[KD + 1][NB];
        auto read_k = [&](int y) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < NB; n++)
                kf[y % (KD + 1)][n] = *(const uint4 *)(kl + kbase + 32 * n * RB + 16 * ((2 * y + hh) ^ kxor));
        };
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 *lptr;
        constexpr int VG = OB < 4 ? OB : 4, VS = OB / VG;    // V's operands per group, groups per 16 rows
        uint2 vf[2][VG][2];
        auto read_v = [&](int z) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < VG; x++) {
                const uint8_t *va = vl + vbase + 16 * (z / VS) * RB + 16 * ((4 * (OB * dh + VG * (z % VS) + x) + vpc) ^ vxor);
                vf[z & 1][x][0] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)va));
                vf[z & 1][x][1] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(va + 8 * RB)));
            }
        };
#pragma unroll
        for (int y = 0; y < KD; y++) read_k(y);
#pragma unroll
        for (int y = 0; y < KS; y++) {
            if (y + KD < KS) read_k(y + KD);
            else if (y + KD == KS) read_v(0);
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int x = NP - 1; x >= 0; x--) s[n] = pa_mfma32<CT>(kf[y % (KD + 1)][n], qf[x][y], s[n]);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, KD * NB, 0);
#pragma unroll
        for (int y = 0; y < KS; y++) {
            if (y + KD < KS) __builtin_amdgcn_sched_group_barrier(0x100, NB, 0);
            if (y + KD == KS) __builtin_amdgcn_sched_group_barrier(0x100, 2 * VG, 0);
            __builtin_amdgcn_sched_group_barrier(0x8, NB * NP, 0);
        }
        float top = -INFINITY;
        if (sw + TW > wave_end || sw < lmax || (EV < 2 && holes)) {
            asm volatile("");                                // a branch: the selects are for the few edges
            const int u = min(pr, len - 1) - sw - 4 * hh, v = lr - sw - 4 * hh;
            uint64_t bits = ~0ull;
            if (EV < 2 && holes) bits = mapped(s0, look(s0));
            bits >>= TW * kh + 4 * hh;
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int x = 32 * n + 8 * (e >> 2) + (e & 3);
                    if (!(x <= u && x >= v && (bits >> x & 1))) s[n][e] = -INFINITY;
                }
        }
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int e = 0; e < 16; e += 2) top = fmaxf(fmaxf(top, s[n][e]), s[n][e + 1]);
        top = fmaxf(top * zs, kLowest);
        if (__any(top > m + kSlack)) {
            asm volatile("");
            top = fmaxf(fmaxf(top, __shfl_xor(top, 32, 64)), m);
            const float f = __builtin_amdgcn_exp2f(m - top);
            m = top;
            l0 *= f;
            l1 *= f;
#pragma unroll
            for (int x = 0; x < OB; x++) o[x] *= f;
        }
        const float mb = kBias<CT> - m;
#pragma unroll
        for (int y = 0; y < TW / 16; y++) {
            uint32_t p[4][PW];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int at = 8 * (y & 1) + 2 * e;
                const float u = __builtin_amdgcn_exp2f(fmaf(s[y >> 1][at], zs, mb));
                const float v = __builtin_amdgcn_exp2f(fmaf(s[y >> 1][at + 1], zs, mb));
                s[y >> 1][at] = u;
                s[y >> 1][at + 1] = v;
                pa_planes<CT, PW, true>(u, v, p[e]);
                float &l = e & 1 ? l1 : l0;
                l += u + v;
            }
#pragma unroll
            for (int g = 0; g < VS; g++) {
                const int z = VS * y + g;
                if (z + 1 < VS * TW / 16) read_v(z + 1);
#pragma unroll
                for (int x = 0; x < VG; x++) {
                    const uint2 f0 = vf[z & 1][x][0], f1 = vf[z & 1][x][1];
#pragma unroll
                    for (int n = PW - 1; n >= 0; n--)
                        o[VG * g + x] = pa_mfma32<CT>(make_uint4(f0.x, f0.y, f1.x, f1.y), make_uint4(p[0][n], p[1][n], p[2][n], p[3][n]), o[VG * g + x]);
                }
            }
        }
#pragma unroll
        for (int z = 0; z < VS * TW / 16; z++) {
            if (z + 1 < VS * TW / 16) __builtin_amdgcn_sched_group_barrier(0x100, 2 * VG, 0);
            __builtin_amdgcn_sched_group_barrier(0x8, VG * PW, 0);
        }
        if constexpr (KH > 1) bad = bad >> (TW * kh) & 0xFFFFFFFFull;
        while (bad) {                                        // rare: V rows that were cleared
            const int x = __builtin_ctzll(bad);
            bad &= bad - 1;
            const int pos = sw + x, blk = pa_block(a, pos);
            const int pg = blk < a.kv.max_blocks ? pa_table(a, seq, blk) : -1;
            if (pos >= len || pg < 0 || pg >= a.kv.n_pages) continue;
            float p = 0.0f;
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if ((x & ~4) == 32 * n + 8 * (e >> 2) + (e & 3)) p = s[n][e];
            const float q = __shfl_xor(p, 32, 64);
            if (hh != (x >> 2 & 1)) p = q;
            const int row = pos - blk * a.kv.page_size;
            const uint8_t *vr = vb + pg * ps + row * rs;
            const float f = E8 ? pa_exp8(a.kv.v_exp[(pg * (long)NKH + j) * a.kv.page_size + row]) : 1.0f;
            if (pos <= pr && pos >= lr)
#pragma unroll
                for (int y = 0; y < OB; y++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int d = 32 * (OB * dh + y) + 8 * (e >> 2) + 4 * hh + (e & 3);
                        float z;
                        if (d >= HD) z = 0.0f;
                        else if constexpr (E8) z = __builtin_amdgcn_cvt_f32_fp8(vr[d], 0) * f;
                        else if constexpr (CT == MLLM_BF16) z = (float)((const __bf16 *)vr)[d];
                        else z = (float)((const _Float16 *)vr)[d];
                        o[y][e] = fmaf(p, z, o[y][e]);
                    }
        }
    };

    if (begin < end) {
        // Before its barrier a wave waits until its loads of the step have landed and its reads of the buffer that
        // is filled next have returned.
        uint32_t holes = 0;                                  // per buffer: some row is on no page
        pages g = look(begin);
        auto bring = [&](int s0, uint8_t *kl, uint8_t *vl, int buf) __attribute__((always_inline)) {
            fetch(s0, g, kl, vl);
            const bool hole = EV == 2 ? s0 < len && (unsigned)g.p0 >= (unsigned)a.kv.n_pages : mapped(s0, g) != ALL;
            holes = (holes & ~(1u << buf)) | (uint32_t)hole << buf;
            if (s0 + TK < end) {
                if constexpr (EV == 2) {
                    nrow += TK;
                    if (nrow == a.kv.page_size) { nrow = 0; nblk++; }
                    row0 = nrow;
                }
                g = look(s0 + TK);
            }
        };
        auto step = [&](int s0, uint8_t *kl, uint8_t *vl, int buf, uint8_t *kn, uint8_t *vn, int next) __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(0x0070);              // vmcnt(0), lgkmcnt(0)
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            bring(s0 + TK, kn, vn, next);
            work(s0, holes >> buf & 1, kl, vl, buf & 1);
            store(kn, vn);
            return s0 + TK < end;
        };
        bring(begin, k0, v0, 0);
        store(k0, v0);
        for (int s0 = begin;; s0 += 2 * TK) {
            if (!step(s0, k0, v0, 0, k1, v1, 1)) break;
            if (!step(s0 + TK, k1, v1, 1, k0, v0, 0)) break;
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);                  // no load may still be on its way into LDS at the end
    }
    float l = (l0 + l1) * kPlanesSum;
    if constexpr (KH == 2) {
        // the two halves of the rows of K and V: the second waves' sums through the buffers of the steps
        __shared__ float hm[RG][64], hl[RG][64];
        __syncthreads();
        f32x4 *to = (f32x4 *)(rg == 0 ? k0 : rg == 1 ? v0 : rg == 2 ? k1 : v1);
        if (kh) {
            hm[rg][lane] = m;
            hl[rg][lane] = l;
#pragma unroll
            for (int x = 0; x < OB; x++)
#pragma unroll
                for (int e = 0; e < 4; e++) to[(4 * x + e) * 64 + lane] = f32x4{o[x][4 * e], o[x][4 * e + 1], o[x][4 * e + 2], o[x][4 * e + 3]};
        }
        __syncthreads();
        if (kh) return;
        const float n = hm[rg][lane], top = fmaxf(m, n), f = __builtin_amdgcn_exp2f(m - top), g = __builtin_amdgcn_exp2f(n - top);
        m = top;
        l = l * f + hl[rg][lane] * g;
#pragma unroll
        for (int x = 0; x < OB; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const f32x4 y = to[(4 * x + e) * 64 + lane];
#pragma unroll
                for (int z = 0; z < 4; z++) o[x][4 * e + z] = o[x][4 * e + z] * f + y[z] * g;
            }
    }
    if (rr >= nrows) return;
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int x = 0; x < OB; x++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int d = 32 * (OB * dh + x) + 8 * e + 4 * hh;
            if (d >= HD) continue;
            const float4 y = make_float4(o[x][4 * e], o[x][4 * e + 1], o[x][4 * e + 2], o[x][4 * e + 3]);
            if (a.splits > 1) *(float4 *)(a.part + (orow * a.splits + sp) * HD + d) = y;
            else pa_finish(a, h, q0 + tok, d, m, l, y);
        }
    if (a.splits > 1 && hh == 0 && dh == 0) *(float2 *)(a.stat + (orow * a.splits + sp) * 2) = make_float2(m, l);
}

template <int CT, bool HP, int HDB, int RG, int KH, int EV> static void pa_prompt_ev(const pa_args &a, hipStream_t st)
{
    hipLaunchKernelGGL((k_pa_prompt<CT, HP, HDB, RG, KH, EV>), dim3(a.tiles * a.kv.n_kv_head, a.splits), dim3(64 * RG * KH * pa_parts(HDB)), 0, st, a);
}
template <int CT, bool HP, int HDB> static void pa_prompt_go(const pa_args &a, bool uniform, hipStream_t st)
{
    constexpr int RG = pa_row_groups(CT, HP, HDB), KH = pa_halves(CT, HP, HDB);
    if constexpr (KH == 2 && RG == 4)
        if (a.groups == 8) return pa_prompt_ev<CT, HP, HDB, 8, 1, 2>(a, st);
    if (!uniform) pa_prompt_ev<CT, HP, HDB, RG, KH, 0>(a, st);
    else if (a.kv.page_size % 64) pa_prompt_ev<CT, HP, HDB, RG, KH, 1>(a, st);
    else pa_prompt_ev<CT, HP, HDB, RG, KH, 2>(a, st);
}
template <int CT, bool HP> static void pa_prompt(const pa_args &a, bool uniform, hipStream_t st)
{
    const int HD = a.kv.head_dim;
    HD <= 64 ? pa_prompt_go<CT, HP, 64>(a, uniform, st) : HD <= 128 ? pa_prompt_go<CT, HP, 128>(a, uniform, st)
                                                                    : pa_prompt_go<CT, HP, 256>(a, uniform, st);
}
