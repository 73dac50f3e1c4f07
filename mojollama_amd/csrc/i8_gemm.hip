// i8_gemm.hip — the product of 8-bit integer rows with packed 8-bit integer weights (i8.h), scales per
// token and per weight row.
//
// out[t][r] = (sum_k x[t][k] w[r][k]) * xs[t] * ws[r] + bias[r]; the sums are whole numbers below 2^31 and
// exact in any order, so K may be split freely and the result does not depend on how.
//
// Every kernel multiplies weights (MFMA rows) by tokens (MFMA columns): a lane then holds four neighbouring
// output channels of one token.
//
// Measured (MI355X, bf16 out, codes of normal values): 8192 tokens x 8192 x 8192 in 418 to 423 us, 2600 to 2630 TOPS,
// where a loop of these matrix instructions on registers alone reaches 3400 (4500 with codes of zero, as this product
// comes to 3900 with them: what bounds it is power); with weights from memory (in the last cache) 1024 tokens x
// 4096 x 4096 in 22.7 us (22.8), 256 in 13.7 (11.0), 64 in 11.1 (8.7), 32 in 8.7 (6.5), 16 in 6.9 (5.9), one in 6.4 (4.6),
// of which the launch is 2.2.  From 20 tokens to 1000 against 4096 x 4096 (3000 against 2880 x 2880) it takes 1.7 to 5
// times what its bytes or products need: K is split only where a second launch to join the sums (4.4 us and their traffic)
// pays, so tiles are small, or fewer than CUs.  Tiles walk K to its next 512: 8192 x 8192 x 64 takes 65 us, x 256 67.5.
#include <algorithm>
#include <type_traits>
#include "i8.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

struct gemm_args {
    const int8_t *w, *x;
    const float *ws, *xs, *bias;
    void *out;
    long x_ld, out_ld;
    int kb;                        // blocks of 64 columns, a multiple of eight
    int T, R, K, type;
    int nt, nr;                    // tiles along tokens and rows
    int splits, per;               // K in `splits` runs of `per` blocks
    int panel;                     // tiles of tokens that go together (tile_at)
    int *part;                     // [split][tile][wave's sums in register order], where splits > 1
};

template <int N> using I = std::integral_constant<int, N>;
// f(I<0>{}) .. f(I<N - 1>{}): indexes of register arrays stay constants whatever the loop's size.
template <int N, int K = 0, class F> __device__ __forceinline__ void each(F &&f)
{
    if constexpr (K < N) {
        f(I<K>{});
        each<N, K + 1>(f);
    }
}

// The result of a sum, the same bits from every kernel here.  bias: -0 where there is none (y + -0 is y, -0 too).
__device__ __forceinline__ float value(int acc, float xs, float ws, float bias) { return fmaf((float)acc * xs, ws, bias); }
__device__ __forceinline__ float bias_of(const gemm_args &a, int r) { return a.bias ? a.bias[r] : -0.0f; }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void *p, int bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, bytes, 0x00020000);
}

// 16 bytes a lane from r + at + base straight to LDS: 1 KB from `to` on in lane order.
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t r, uint8_t *to, int at, int base)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)to, 16, at, base, 0, 0);
}

// Vector memory operations younger than n may be under way, no LDS access.
template <int n> __device__ __forceinline__ void wait_mem()
{
    static_assert(n < 64, "vmcnt is six bits");
    __builtin_amdgcn_s_waitcnt((n & 15) | ((n >> 4) << 14) | 0x0070);
}

// The order of half a step: LOADS loads spread over MUL matrix instructions, READS operand reads over the first half
// of them, so that the operands are there when the next half begins; and nothing across.
template <int READS, int MUL, int LOADS> __device__ __forceinline__ void order()
{
    each<MUL>([](auto i) __attribute__((always_inline)) {
        constexpr int H = (MUL + 1) / 2, a = i < H ? i : H, b = i + 1 < H ? i + 1 : H;
        constexpr int r = b * READS / H - a * READS / H, v = (i + 1) * LOADS / MUL - i * LOADS / MUL;
        if constexpr (v > 0) __builtin_amdgcn_sched_group_barrier(0x10, v, 0);
        if constexpr (r > 0) __builtin_amdgcn_sched_group_barrier(0x100, r, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    });
    __builtin_amdgcn_sched_barrier(0);
}

// ------------------------------------------------------------------------------------ the tail
// What the tail needs of a tile of TT tokens and TR rows, in LDS from the start.
template <int TT, int TR> struct scales {
    float ws[TR], bias[TR], xs[TT];
};
// Asked for before the loop's loads, stored behind them: nothing waits for them alone.  IDS lanes share the work.
template <int TT, int TR, int IDS> struct scales_of {
    float ws[(TR + IDS - 1) / IDS], bias[(TR + IDS - 1) / IDS], xs[(TT + IDS - 1) / IDS];
};
template <int TT, int TR, int IDS> __device__ __forceinline__ void get_scales(const gemm_args &a, int t0, int r0,
                                                                              scales_of<TT, TR, IDS> &s, int id)
{
#pragma unroll
    for (int i = 0; i < (TR + IDS - 1) / IDS; i++) {
        const int r = min(r0 + i * IDS + id, a.R - 1);
        s.ws[i] = a.ws[r];
        s.bias[i] = bias_of(a, r);
    }
#pragma unroll
    for (int i = 0; i < (TT + IDS - 1) / IDS; i++) s.xs[i] = a.xs[min(t0 + i * IDS + id, a.T - 1)];
}
template <int TT, int TR, int IDS> __device__ __forceinline__ void put_scales(const scales_of<TT, TR, IDS> &s, scales<TT, TR> &to,
                                                                              int id)
{
#pragma unroll
    for (int i = 0; i < (TR + IDS - 1) / IDS; i++)
        if (i * IDS + id < TR) {
            to.ws[i * IDS + id] = s.ws[i];
            to.bias[i * IDS + id] = s.bias[i];
        }
#pragma unroll
    for (int i = 0; i < (TT + IDS - 1) / IDS; i++)
        if (i * IDS + id < TT) to.xs[i * IDS + id] = s.xs[i];
}

// A wave's sums of 32 tokens x 32 NF output channels to out, by way of `room`, its own LDS: there the channels of a
// token lie side by side, and a lane scales and stores eight of them, in whole lines.  The code is short (the sums
// pass through LDS as integers, the rest is a loop): a tail of straight code took as long as 40 steps of K, most of it
// for its instructions.
template <int NF> constexpr int room_bytes() { return 32 * 128 * NF; }
// Byte of four channels (chunk c) of token t there: eight tokens' chunks of one number meet distinct banks.
template <int NF> __device__ __forceinline__ int room_at(int t, int c) { return t * 128 * NF + ((c ^ (t & 7)) << 4); }

template <int NF, class T> __device__ __forceinline__ void tail_as(const gemm_args &a, int t0, int r0, const uint8_t *room,
                                                                   const float *xs, const float (&ws)[8], const float (&bias)[8],
                                                                   int lane)
{
    constexpr int LPR = 4 * NF, TPW = 64 / LPR;              // lanes of a token, tokens of a pass
    constexpr int type = sizeof(T) == 4 ? MLLM_F32 : std::is_same<T, __bf16>::value ? MLLM_BF16 : MLLM_F16;
    const int c = lane % LPR * 8, t = lane / LPR;
    T *to = (T *)a.out + (long)(t0 + t) * a.out_ld + r0 + c;
    auto form = [&](int t, float (&y)[8]) __attribute__((always_inline)) {
        const i32x4 u = *(const i32x4 *)(room + room_at<NF>(t, c >> 2)), v = *(const i32x4 *)(room + room_at<NF>(t, (c >> 2) + 1));
        const float x = xs[t];
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = value(i < 4 ? u[i] : v[i - 4], x, ws[i], bias[i]);
    };
    if (t0 + 32 <= a.T && r0 + 32 * NF <= a.R) {
#pragma unroll 4
        for (int j = 0; j < 32 / TPW; j++, to += TPW * a.out_ld) {
            float y[8];
            form(t + j * TPW, y);
            if constexpr (sizeof(T) == 4) {
                __builtin_memcpy(to, y, 32);
            } else {
                const u32x4 w = {pack2<type>(y[0], y[1]), pack2<type>(y[2], y[3]), pack2<type>(y[4], y[5]), pack2<type>(y[6], y[7])};
                __builtin_memcpy(to, &w, 16);
            }
        }
        return;
    }
#pragma unroll 1
    for (int j = t; j < min(32, a.T - t0); j += TPW, to += TPW * a.out_ld) {
        float y[8];
        form(j, y);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (r0 + c + i < a.R) put1(to, i, type, y[i]);
    }
}

// All MF x 32 tokens of a wave, 32 at a time, in a loop that stays one (the sums of a turn, by constant index, in a
// case of their own).
template <int MF, int NF> __device__ __forceinline__ void tail(const gemm_args &a, const i32x16 (&acc)[MF][NF], int t0, int r0,
                                                               uint8_t *room, const float *xs, const float (&ws)[8],
                                                               const float (&bias)[8], int lane)
{
    const int l = lane & 31, h = lane >> 5;
#pragma unroll 1
    for (int m = 0; m < MF; m++, t0 += 32, xs += 32) {
        __builtin_amdgcn_wave_barrier();                     // the reads before are done
        each<MF>([&](auto k) __attribute__((always_inline)) {
            if (k != m) return;
#pragma unroll
            for (int n = 0; n < NF; n++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *(i32x4 *)(room + room_at<NF>(l, 8 * n + 2 * g + h)) =
                        (i32x4){acc[k][n][4 * g], acc[k][n][4 * g + 1], acc[k][n][4 * g + 2], acc[k][n][4 * g + 3]};
        });
        __builtin_amdgcn_wave_barrier();
        if (a.type == MLLM_F32) tail_as<NF, float>(a, t0, r0, room, xs, ws, bias, lane);
        else if (a.type == MLLM_BF16) tail_as<NF, __bf16>(a, t0, r0, room, xs, ws, bias, lane);
        else tail_as<NF, _Float16>(a, t0, r0, room, xs, ws, bias, lane);
    }
}

// ------------------------------------------------------------------------------------ many tokens
// Workgroup b of n runs on XCD b % 8: each XCD takes one run of the tiles, in panels of a.panel tiles of tokens with
// the rows in turn inside, so that the tiles it works on at a time are a block of the output and share both operands
// in its L2 (4096 x 4096 x 4096: 60.5 us, 67.7 with the tiles dealt round the XCDs; panels of 2 to 8 are alike).
struct work_tile { int z, t, r; };
__device__ __forceinline__ work_tile tile_at(const gemm_args &a, int b, int n)
{
    const int xcd = b & 7;
    int i = xcd * (n >> 3) + min(xcd, n & 7) + (b >> 3);
    const int z = __builtin_amdgcn_readfirstlane(i / (a.nt * a.nr));
    i -= z * a.nt * a.nr;
    const int p = __builtin_amdgcn_readfirstlane(i / (a.panel * a.nr)), wide = min(a.panel, a.nt - p * a.panel);
    i -= p * a.panel * a.nr;
    const int r = __builtin_amdgcn_readfirstlane(i / wide);
    return {z, p * a.panel + i - r * wide, r};
}

// WM x WN waves make a tile of 32 MF WM tokens x 32 NF WN rows, a wave 32 MF x 32 NF of it.  K goes by
// 64 columns a step.  Both operands come to LDS past the registers: the weights of a step into one of four buffers, up
// to four steps ahead; x for two steps at once, so that a row is read in whole lines of 128 bytes (64 bytes at a time
// cost twice the L2 traffic), into one of two.  Where tiles are fewer than CUs a step is as long as its latency: KG = 2
// groups of waves, with buffers of their own, take half of K each, and the second hands its sums to the first by way of
// LDS (256 x 4096 x 4096 with weights from memory: 15.9 -> 13.7 us, 512: 17.6 -> 16.5; for tiles of 128 x 128 and more,
// whose steps are bound by their products, no gain).
template <int MF, int NF, int WM, int WN> struct tile_of {
    static constexpr int waves = WM * WN, TT = 32 * MF * WM, TR = 32 * NF * WN;
    // 1 KB pieces of two steps of x, of a step of weights, and a wave's
    static constexpr int xp = TT / 8, wp = TR / 16, px = xp / waves, pw = wp / waves;
    static_assert(xp % waves == 0 && wp % waves == 0, "pieces go evenly to waves");
};

// Slot of a row's chunk of 16 bytes is chunk ^ swz(row): the reads of 16 rows, one chunk each, meet distinct banks.
__device__ __forceinline__ int swz(int row) { return (row ^ (row >> 3 & 3)) & 7; }

template <int MF, int NF, int WM, int WN, int KG, int OCC>
__global__ __launch_bounds__(64 * WM * WN * KG, OCC) void k_i8_tiles(gemm_args a)
{
    using C = tile_of<MF, NF, WM, WN>;
    // buffers of their own each: the compiler then knows which loads a read may meet
    constexpr int XB = C::xp * 1024, WB = C::wp * 1024;
    __shared__ __attribute__((aligned(1024))) uint8_t x0[KG * XB], x1[KG * XB], w0[KG * WB], w1[KG * WB], w2[KG * WB], w3[KG * WB];
    const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = all / C::waves, wave = all - group * C::waves;
    const int wm = wave % WM, wn = wave / WM, l = lane & 31, h = lane >> 5;
    const work_tile wt = tile_at(a, blockIdx.x, gridDim.x);
    const int z = wt.z, tile = wt.r * a.nt + wt.t, t0 = wt.t * C::TT, r0 = wt.r * C::TR;
    const int most = min(a.kb - z * a.per, a.per), steps = most / KG;   // multiples of four
    const int s_beg = z * a.per + group * steps, s_end = s_beg + steps;
    __shared__ scales<C::TT, C::TR> sc;
    scales_of<C::TT, C::TR, 64 * C::waves * KG> have;
    if (a.splits == 1) get_scales(a, t0, r0, have, threadIdx.x);

    // ---- loads: a piece of x is 8 tokens x 128 columns (lane: token lane / 8, slot lane % 8), of the weights 1 KB as
    // they lie.  What lies behind the last row of x is not read, what lies behind a row meets weights of zero.
    const int8_t *xb = a.x + (long)t0 * a.x_ld;
    const long left = (long)(min(a.T - t0, C::TT) - 1) * a.x_ld + (a.K + 15) / 16 * 16;
    const __amdgpu_buffer_rsrc_t xr = rsrc(xb, (int)left), wr = rsrc(a.w + (long)(r0 >> 5) * a.kb * 2048, -1);
    int xo[C::px], wo[C::pw];
#pragma unroll
    for (int p = 0; p < C::px; p++) {
        const int row = 8 * (p * C::waves + wave) + (lane >> 3);
        xo[p] = row * (int)a.x_ld + 16 * ((lane & 7) ^ swz(row)) + 64 * s_beg;
    }
#pragma unroll
    for (int p = 0; p < C::pw; p++) {
        const int q = p * C::waves + wave, rb = min(q >> 1, ((a.R - 1) >> 5) - (r0 >> 5));
        wo[p] = rb * a.kb * 2048 + (q & 1) * 1024 + lane * 16;
    }
    int xs = s_beg, ws = s_beg;                              // the next steps to load; the last ones over and over
    auto load_x = [&](uint8_t *to) __attribute__((always_inline)) {
        const int more = xs + 2 < s_end;
#pragma unroll
        for (int p = 0; p < C::px; p++) {
            to_lds(xr, to + group * XB + 1024 * (p * C::waves + wave), xo[p], 0);
            xo[p] += 128 * more;
        }
        xs += 2 * more;
    };
    auto load_w = [&](uint8_t *to) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < C::pw; p++) to_lds(wr, to + group * WB + 1024 * (p * C::waves + wave), wo[p], ws * 2048);
        ws += ws + 1 < s_end;
    };
    i32x16 acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int n = 0; n < NF; n++) acc[m][n] = i32x16{};
    // ---- operands of half a step (32 columns), j: which of the four of a pair of steps
    struct frags { i32x4 x[MF], w[NF]; };
    int xa[4];
#pragma unroll
    for (int j = 0; j < 4; j++) xa[j] = l * 128 + 16 * ((2 * j + h) ^ swz(l));
    auto get = [&](const uint8_t *fx, const uint8_t *fw, auto j, frags &f) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NF; n++) f.w[n] = *(const i32x4 *)(fw + group * WB + (wn * NF + n) * 2048 + (j & 1) * 1024 + lane * 16);
#pragma unroll
        for (int m = 0; m < MF; m++) f.x[m] = *(const i32x4 *)(fx + group * XB + (wm * MF + m) * 4096 + xa[j]);
    };
    auto multiply = [&](const frags &f) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < MF; m++)
#pragma unroll
            for (int n = 0; n < NF; n++) acc[m][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[n], f.x[m], acc[m][n], 0, 0, 0);
    };
    frags f0, f1;
    auto then = []() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };
    load_x(x0);
    load_w(w0);
    then();
    load_w(w1);
    then();
    load_w(w2);
    then();
    load_x(x1);
    then();
    if (a.splits == 1) put_scales(have, sc, threadIdx.x);
    wait_mem<2 * C::pw + C::px>();
    __builtin_amdgcn_s_barrier();
    get(x0, w0, I<0>{}, f0);
    // A step: its second half's operands are read while the first half multiplies, the next step's first while the
    // second does.  Between, the loads that the next step needs have landed for every wave, and nobody reads this step's
    // buffers any more.  Loads are spread evenly: the first half of an even step asks for weights (into the buffer of
    // the step before), the second for weights again (its own), the second half of an odd step for x of the second
    // pair from here.  So under way may be, in the middle of an even step, whose next needs the weights of the first
    // half two steps ago: weights, x, weights; in the middle of an odd step, whose next needs x of two steps ago:
    // weights twice.  The order of loads within a half has no part in this.
    auto step = [&](auto odd, uint8_t *x_here, const uint8_t *x_next, uint8_t *w_before, uint8_t *w_here, const uint8_t *w_next)
                    __attribute__((always_inline)) {
        if constexpr (!odd) load_w(w_before);
        get(x_here, w_here, I<2 * odd + 1>{}, f1);
        multiply(f0);
        order<MF + NF, MF * NF, odd ? 0 : C::pw>();
        wait_mem<odd ? 2 * C::pw : 2 * C::pw + C::px>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (odd) load_x(x_here);
        else load_w(w_here);
        get(x_next, w_next, I<odd ? 0 : 2>{}, f0);
        multiply(f1);
        order<MF + NF, MF * NF, odd ? C::px : C::pw>();
    };
    int s = s_beg;
    do {
        step(I<0>{}, x0, x0, w3, w0, w1);
        step(I<1>{}, x0, x1, w0, w1, w2);
        step(I<0>{}, x1, x1, w1, w2, w3);
        step(I<1>{}, x1, x0, w2, w3, w0);
        s += 4;
    } while (s < s_end);
    wait_mem<0>();
    __builtin_amdgcn_s_barrier();
    if constexpr (KG > 1) {
        // the second group's sums to the first, by way of LDS: a wave's 4 KB pieces in its weights' buffers
        static_assert(KG == 2 && MF * NF * 4 * C::waves <= KG * 4 * C::wp, "the sums fit the weights' buffers");
        constexpr int each_buffer = KG * WB / (4096 * C::waves);         // pieces of a wave that a buffer takes
        static_assert(each_buffer >= 1 && MF * NF <= 4 * each_buffer, "");
        auto piece = [&](int i) __attribute__((always_inline)) {
            uint8_t *b = i / each_buffer == 0 ? w0 : i / each_buffer == 1 ? w1 : i / each_buffer == 2 ? w2 : w3;
            return b + (wave * each_buffer + i % each_buffer) * 4096 + lane * 16;
        };
        each<MF * NF>([&](auto i) __attribute__((always_inline)) {
            if (group == 1) {
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *(i32x4 *)(piece(i) + g * 1024) = (i32x4){acc[i / NF][i % NF][4 * g], acc[i / NF][i % NF][4 * g + 1],
                                                              acc[i / NF][i % NF][4 * g + 2], acc[i / NF][i % NF][4 * g + 3]};
            }
        });
        __syncthreads();
        if (group == 1) return;
        each<MF * NF>([&](auto i) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const i32x4 v = *(const i32x4 *)(piece(i) + g * 1024);
#pragma unroll
                for (int k = 0; k < 4; k++) acc[i / NF][i % NF][4 * g + k] += v[k];
            }
        });
        wait_mem<0>();
    }

    if (a.splits > 1) {
        int *p = a.part + (((long)z * a.nt * a.nr + tile) * C::waves + wave) * (MF * NF * 1024) + lane * 4;
#pragma unroll
        for (int m = 0; m < MF; m++)
#pragma unroll
            for (int n = 0; n < NF; n++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *(i32x4 *)(p + ((m * NF + n) * 4 + g) * 256) =
                        (i32x4){acc[m][n][4 * g], acc[m][n][4 * g + 1], acc[m][n][4 * g + 2], acc[m][n][4 * g + 3]};
        return;
    }
    static_assert(C::waves == 4 && room_bytes<NF>() <= C::wp * 1024, "the tail of a wave fits a buffer of weights");
    uint8_t *room = KG > 1 ? (wave < 2 ? x0 : x1) + (wave & 1) * room_bytes<NF>()
                           : wave == 0 ? w0 : wave == 1 ? w1 : wave == 2 ? w2 : w3;
    static_assert(KG == 1 || 2 * room_bytes<NF>() <= KG * XB, "x's buffers hold the tails of four waves");
    const int c = wn * NF * 32 + lane % (4 * NF) * 8;
    float rs[8], bias[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        rs[i] = sc.ws[c + i];
        bias[i] = sc.bias[c + i];
    }
    const int t = wm * MF * 32;
    tail<MF, NF>(a, acc, t0 + t, r0 + wn * NF * 32, room, sc.xs + t, rs, bias, lane);
}

// The sums of all splits, and the tail.
template <int MF, int NF, int WM, int WN> __global__ __launch_bounds__(64) void k_i8_join(gemm_args a)
{
    using C = tile_of<MF, NF, WM, WN>;
    __shared__ __attribute__((aligned(16))) uint8_t room[room_bytes<NF>()];
    const int lane = threadIdx.x;
    const int m = blockIdx.x % MF, wave = blockIdx.x / MF % C::waves, tile = blockIdx.x / (MF * C::waves);
    const int wm = wave % WM, wn = wave / WM;
    const int t = tile % a.nt * C::TT + (wm * MF + m) * 32, r = tile / a.nt * C::TR + wn * NF * 32;
    if (t >= a.T || r >= a.R) return;
    __shared__ scales<32, 32 * NF> sc;
    scales_of<32, 32 * NF, 64> have;
    get_scales(a, t, r, have, lane);
    put_scales(have, sc, lane);
    __syncthreads();
    i32x16 acc[1][NF];
#pragma unroll
    for (int n = 0; n < NF; n++) acc[0][n] = i32x16{};
    const int *p = a.part + ((long)tile * C::waves + wave) * (MF * NF * 1024) + m * NF * 1024 + lane * 4;
    for (int z = 0; z < a.splits; z++, p += (long)a.nt * a.nr * C::waves * MF * NF * 1024)
#pragma unroll
        for (int n = 0; n < NF; n++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const i32x4 v = *(const i32x4 *)(p + (n * 4 + g) * 256);
#pragma unroll
                for (int i = 0; i < 4; i++) acc[0][n][4 * g + i] += v[i];
            }
    const int c = lane % (4 * NF) * 8;
    float rs[8], bias[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        rs[i] = sc.ws[c + i];
        bias[i] = sc.bias[c + i];
    }
    tail<1, NF>(a, acc, t, r, room, sc.xs, rs, bias, lane);
}

// ------------------------------------------------------------------------------------ few tokens
// 16 weight rows x up to 16 tokens a workgroup of W waves, which take blocks of 64 columns in turn and join their sums in
// LDS.  Weights stream from memory straight into the matrix cores, each byte once; x comes from the caches.  Bound by the
// launch and one memory round trip where they are few (2048 x 2048: 4.2 us), by memory else (28672 x 4096: 23 us,
// 5.1 TB/s).
template <int W> __global__ __launch_bounds__(64 * W) void k_i8_few(gemm_args a)
{
    constexpr int D = 2;                                     // blocks under way a wave
    __shared__ __attribute__((aligned(16))) int sums[W][64][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, c = lane >> 4;
    const int r0 = blockIdx.x * 16, nb = (a.K + 63) / 64;
    const int8_t *w = a.w + (long)(r0 >> 5) * a.kb * 2048 + (r0 & 16) * 16 + c * 512 + l * 16;
    const __amdgpu_buffer_rsrc_t xr = rsrc(a.x, (int)((a.T - 1) * a.x_ld + (a.K + 15) / 16 * 16));
    const bool live = l < a.T;                               // the other lanes ask for what is not there: zeros
    const int xo = live ? l * (int)a.x_ld + 16 * c : 0x7FFFFF00;
    i32x4 acc = {};
    for (int b = wave; b < nb; b += W * D) {
        i32x4 wf[D], xf[D];
#pragma unroll
        for (int d = 0; d < D; d++) {
            const int k = min(b + d * W, nb - 1);
            wf[d] = *(const i32x4 *)(w + (long)k * 2048);
            xf[d] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(xr, live ? xo + 64 * k : xo, 0, 0));
        }
#pragma unroll
        for (int d = 0; d < D; d++)
            if (b + d * W < nb) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[d], xf[d], acc, 0, 0, 0);
    }
    *(i32x4 *)sums[wave][lane] = acc;
    __syncthreads();
    if (wave > 0 || l >= a.T) return;                        // lane: token l, rows 4 c + i
    i32x4 s = {};
#pragma unroll
    for (int i = 0; i < W; i++) s += *(const i32x4 *)sums[i][lane];
    const float xs = a.xs[l];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = r0 + 4 * c + i;
        if (r < a.R) put1(a.out, l * a.out_ld + r, a.type, value(s[i], xs, a.ws[r], bias_of(a, r)));
    }
}

// 32 weight rows x 32 TF tokens a workgroup of W waves, which take blocks of 128 columns in turn and join their sums in
// LDS.  A wave's block of x comes to its own part of LDS in whole lines and its weights to registers, asked for two blocks
// ahead; waves meet at the end alone.  The loads stand behind a condition, so that the compiler takes a block's weights for
// the youngest loads and waits for all: in every other block the next one's loads are waited for too, and a pair of blocks
// takes a round trip to memory.  (32 tokens x 4096 x 4096 with weights in the last cache: 6.5 us, 8.0 with x from the
// caches; 16 x 8192 x 8192 from memory: 14.5 us, 4.6 TB/s, 19.4 with 16 rows a workgroup.  96 and 128 tokens would be
// bound by LDS: 12.6 and 14 us, tiles 11.  64 rows a workgroup: 48 tokens x 14336 x 4096 18.0 us for 21.6, but tiles take
// 17.6, and 10 to 60 % slower where rows are fewer.)
template <int TF, int W> __global__ __launch_bounds__(64 * W) void k_i8_stream(gemm_args a)
{
    constexpr int XB = TF * 4096, LOADS = 4 * TF + 4;            // bytes and loads of a block
    __shared__ __attribute__((aligned(1024))) uint8_t x0[W * XB], x1[W * XB];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 31, h = lane >> 5;
    const int r0 = blockIdx.x * 32, nb = (a.K + 127) / 128;
    const int8_t *w = a.w + (long)blockIdx.x * a.kb * 2048 + lane * 16;
    const __amdgpu_buffer_rsrc_t xr = rsrc(a.x, (int)((a.T - 1) * a.x_ld + (a.K + 15) / 16 * 16));
    int xo[4 * TF], xa[4];
#pragma unroll
    for (int p = 0; p < 4 * TF; p++) {
        const int row = 8 * p + (lane >> 3);
        xo[p] = row * (int)a.x_ld + 16 * ((lane & 7) ^ swz(row));
    }
#pragma unroll
    for (int j = 0; j < 4; j++) xa[j] = wave * XB + l * 128 + 16 * ((2 * j + h) ^ swz(l));
    auto load = [&](uint8_t *to, i32x4 (&wf)[4], int b) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int p = 0; p < 4 * TF; p++) to_lds(xr, to + wave * XB + 1024 * p, xo[p] + 128 * b, 0);
#pragma unroll
        for (int j = 0; j < 4; j++) wf[j] = *(const i32x4 *)(w + (long)b * 4096 + j * 1024);
        __builtin_amdgcn_sched_barrier(0);
    };
    i32x16 acc[TF];
#pragma unroll
    for (int f = 0; f < TF; f++) acc[f] = i32x16{};
    i32x4 w0[4], w1[4];
    if (wave < nb) load(x0, w0, wave);
    if (wave + W < nb) load(x1, w1, wave + W);
    // block b: its x has landed (the loads of block b + W, if there is one, may be under way as far as x goes; the weights
    // have the compiler's waits); when its operands are read, its buffer takes block b + 2 W
    auto block = [&](uint8_t *x, i32x4 (&wf)[4], int b) __attribute__((always_inline)) {
        if (b + W < nb) wait_mem<LOADS>();
        else wait_mem<0>();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int f = 0; f < TF; f++)
                acc[f] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[j], *(const i32x4 *)(x + f * 4096 + xa[j]), acc[f], 0, 0, 0);
        if (b + 2 * W < nb) load(x, wf, b + 2 * W);
    };
    for (int b = wave; b < nb; b += 2 * W) {
        block(x0, w0, b);
        if (b + W < nb) block(x1, w1, b + W);
    }
    __syncthreads();
#pragma unroll
    for (int f = 0; f < TF; f++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *(i32x4 *)(x0 + ((wave * TF + f) * 4 + g) * 1024 + lane * 16) =
                (i32x4){acc[f][4 * g], acc[f][4 * g + 1], acc[f][4 * g + 2], acc[f][4 * g + 3]};
    __syncthreads();
    for (int u = wave; u < 4 * TF; u += W) {                     // frag u / 4, rows 8 (u % 4) + 4 h and on
        const int t = u / 4 * 32 + l, r = r0 + u % 4 * 8 + 4 * h;
        i32x4 s = {};
#pragma unroll
        for (int i = 0; i < W; i++) s += *(const i32x4 *)(x0 + (i * 4 * TF + u) * 1024 + lane * 16);
        if (t >= a.T) continue;
        const float xs = a.xs[t];
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (r + i < a.R) put1(a.out, t * a.out_ld + r + i, a.type, value(s[i], xs, a.ws[r + i], bias_of(a, r + i)));
    }
}

// ------------------------------------------------------------------------------------ rows far apart
// Rows of x so far apart that a tile's offsets leave 32 bits: a wave per 32 weight rows x 32 tokens, operands from
// global memory.
__global__ __launch_bounds__(64) void k_i8_far(gemm_args a)
{
    const int lane = threadIdx.x, l = lane & 31, h = lane >> 5;
    const long tile = i8_block();
    if (tile >= (long)a.nt * a.nr) return;
    const int r0 = (int)(tile / a.nt) * 32, t0 = (int)(tile % a.nt) * 32;
    const int8_t *w = a.w + (long)(r0 >> 5) * a.kb * 2048 + lane * 16;
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
        if (r < a.R) put1(a.out, t * a.out_ld + r, a.type, value(acc[i], xs, a.ws[r], bias_of(a, r)));
    }
}

// ------------------------------------------------------------------------------------ the choice
struct tile_kind {
    int TT, TR, groups, per_cu;    // groups of waves, workgroups of it that a CU holds
    float step, each, tail;        // for a step of K, each workgroup in it, a workgroup beside (see plan_of)
    void (*go)(const gemm_args &, int grid, hipStream_t);
    // A tile is not mostly empty.  Up to 32 tokens the time is that of the weights' stream, which two groups do not
    // shorten: 16 tokens of 11264 x 2048 take them 9.3 us, k_i8_stream 7.4.
    bool fits(int T) const { return groups > 1 ? T > 32 && TT < 2 * T : TT < 64 || TT < 2 * T; }
    long at_once() const { return 256l * per_cu; }                       // workgroups that the GPU holds: splits go no further
};
constexpr int kMostSplits = 12;
constexpr long kMostBlocks = (1l << 24) - 1;                         // of 256 lanes: the lanes of a launch stay below 2^32
template <int MF, int NF, int WM, int WN, int KG, int OCC> void go_tiles(const gemm_args &a, int grid, hipStream_t st)
{
    hipLaunchKernelGGL((k_i8_tiles<MF, NF, WM, WN, KG, OCC>), dim3(grid), dim3(64 * WM * WN * KG), 0, st, a);
    if (a.splits > 1)
        hipLaunchKernelGGL((k_i8_join<MF, NF, WM, WN>), dim3(a.nt * a.nr * MF * WM * WN), dim3(64), 0, st, a);
}
template <int MF, int NF, int WM, int WN, int KG, int OCC> constexpr tile_kind kind_of(float step, float each, float tail)
{
    using C = tile_of<MF, NF, WM, WN>;
    return {C::TT, C::TR, KG, OCC, step, each, tail, go_tiles<MF, NF, WM, WN, KG, OCC>};
}
const tile_kind kinds[] = {
    kind_of<4, 4, 2, 2, 1, 1>(0.37f, 0.202f, 10.7f),
    kind_of<2, 4, 2, 2, 1, 1>(0.134f, 0.26f, 5.23f),
    kind_of<2, 2, 2, 2, 1, 2>(0.000872f, 0.265f, 2.08f),
    kind_of<1, 2, 2, 2, 1, 3>(0.000546f, 0.274f, 0.0339f),
    kind_of<1, 1, 1, 4, 1, 3>(0.0854f, 0.121f, 0.0782f),
    kind_of<1, 2, 2, 2, 2, 1>(0.00158f, 0.175f, 2.41f),
    kind_of<1, 1, 1, 4, 2, 1>(0.0051f, 0.156f, 0.805f)};

struct plan {
    const tile_kind *kind;         // or null:
    int few;                       // 0: no kernel, 1: k_i8_few, 2, 3: k_i8_stream<few - 1>
    int nt, nr, splits, per;
};

// The kernel that an estimate of their times in microseconds, from sizes alone, puts first; its constants are fitted to
// the kernels' times with weights from memory, at 1 to 4096 tokens and seventeen matrices from 512 x 2048 to
// 32000 x 2048 and 1024 x 14336, every tile with K split up to twelve times (3540 times).  On these same times its choice
// is 0.6 % slower than the best on average, 18 % at most; sizes outside them were not measured with every kernel.  The
// constants were fitted together: a kind's step, each and tail make up its time as a sum and measure nothing alone.
plan plan_of(int T, int R, int kb, int cols)
{
    plan best{};
    float least = INFINITY;
    const float mb = (float)cols * R * 1e-6f;
    if (T <= 16 && R < 1 << 26) {
        const int n = (R + 15) / 16, turns = (cols + 1023) / 1024;
        least = 2.11f + std::max((n + 511) / 512 * (0.711f + turns * 0.38f) + turns * (n / 512.0f) * (0.669f + T * 0.0419f),
                                 mb / (4.46f - 0.0333f * T));
        best.few = 1;
    }
    if (T <= 64 && R < 1 << 26) {
        const int n = (R + 31) / 32, turns = (cols + 1023) / 1024;
        const float us = T <= 32 ? 2.19f + std::max(turns * 1.14f, mb / 5.66f) + n / 256.0f * (0.376f + turns * T * 0.00271f)
                                 : 1.79f + std::max(turns * 2.02f, mb / 4.28f) + n / 256.0f * 2.1f;
        if (us < least) {
            least = us;
            best.few = T <= 32 ? 2 : 3;
        }
    }
    const int units = kb / 8;
    for (const tile_kind &k : kinds) {
        if (!k.fits(T)) continue;
        for (int want : {1, 2, 3, 4, 6, 8, kMostSplits}) {
            plan p{&k, 0, (T + k.TT - 1) / k.TT, (R + k.TR - 1) / k.TR, 0, 0};
            if (want > units) continue;
            p.per = (units + want - 1) / want * 8;
            p.splits = (kb + p.per - 1) / p.per;
            const long n = (long)p.nt * p.nr * want;
            if (p.splits != want || n > (want > 1 ? k.at_once() : kMostBlocks)) continue;
            const int most = (int)((n + 255) / 256), full = most / k.per_cu, rest = most % k.per_cu;
            float us = full * (p.per * (k.step + k.per_cu * k.each) + k.tail) + (rest ? p.per * (k.step + rest * k.each) + k.tail : 0.0f);
            us = 2.54f + std::max(us, (float)cols * ((float)R + T) / 5.38e6f);
            if (want > 1) us += 4.44f + (float)n * k.TT * k.TR * 8 / 7.49e6f;
            if (us < least) {
                least = us;
                best = p;
            }
        }
    }
    return best;
}

// Bytes of the sums of any plan with splits for T tokens or fewer.
long sums_of(int T, int R, int kb)
{
    long most = 0;
    for (const tile_kind &k : kinds) {
        const long nr = (R + k.TR - 1) / k.TR, n = std::min((long)std::min(kb / 8, kMostSplits) * ((T + k.TT - 1) / k.TT) * nr, k.at_once());
        if (k.fits(T) && kb > 8 && 2 * nr <= k.at_once()) most = std::max(most, n * k.TT * k.TR * 4);
    }
    return most;
}

} // namespace

extern "C" {

MLLM_API long mllm_i8_gemm_workspace_size(int T, int n_rows, int n_cols)
{
    if (T < 0 || T > 1 << 30 || mllm_i8_packed_size(n_rows, n_cols) < 0) return -1;
    return T ? sums_of(T, n_rows, (int)i8_kblocks(n_cols)) : 0;
}

MLLM_API int mllm_i8_gemm(const void *packed, const float *w_scale, const int8_t *x, long x_ld, const float *x_scale,
                          int T, int n_rows, int n_cols, const float *bias, int type, void *out, long out_ld,
                          void *workspace, long ws_bytes, void *stream)
{
    const char *who = "mllm_i8_gemm";
    if (T < 0 || T > 1 << 30 || mllm_i8_packed_size(n_rows, n_cols) < 0)
        return pk_fail(who, "T is not negative, n_rows positive (both at most 2^30), n_cols from 1 to 131071");
    if (!i8_real(type)) return pk_fail(who, "the type of out is F32, F16 or BF16");
    if (x_ld < n_cols || out_ld < n_rows) return pk_fail(who, "rows of x lie at least n_cols apart, of out n_rows");
    if (((uintptr_t)x | (uintptr_t)x_ld | (uintptr_t)packed | (uintptr_t)workspace) & 15)
        return pk_fail(who, "x, its rows, packed and the workspace lie at multiples of 16 bytes");
    if (T && (!packed || !w_scale || !x || !x_scale || !out))
        return pk_fail(who, "packed, w_scale, x, x_scale and out are given");
    const long need = mllm_i8_gemm_workspace_size(T, n_rows, n_cols);
    if (need > 0 && (!workspace || ws_bytes < need)) return pk_fail(who, "the workspace is too small");
    if (!T) return 0;
    const int kb = (int)i8_kblocks(n_cols);
    const bool far = x_ld >= 1l << 22;                       // 256 rows and a step more stay below 2^31
    const plan p = plan_of(T, n_rows, kb, n_cols);
    gemm_args a{(const int8_t *)packed, x, w_scale, x_scale, bias, out, x_ld, out_ld, kb, T, n_rows, n_cols, type,
                p.nt, p.nr, p.splits, p.per, p.nt < 4 ? p.nt : 4, (int *)workspace};
    hipStream_t st = (hipStream_t)stream;
    if (far) {
        a.nt = (T + 31) / 32;
        a.nr = (n_rows + 31) / 32;
        const long blocks = (long)a.nt * a.nr;
        if (blocks > kI8Blocks * 65535) return pk_fail(who, "T * n_rows is too large for one call");
        hipLaunchKernelGGL(k_i8_far, i8_grid(blocks), dim3(64), 0, st, a);
    } else if (p.kind) {
        p.kind->go(a, p.nt * p.nr * p.splits, st);
    } else if (p.few > 1) {
        const int grid = (n_rows + 31) / 32;
        if (p.few == 2) hipLaunchKernelGGL((k_i8_stream<1, 8>), dim3(grid), dim3(512), 0, st, a);
        else hipLaunchKernelGGL((k_i8_stream<2, 8>), dim3(grid), dim3(512), 0, st, a);
    } else if (p.few) {
        const int grid = (n_rows + 15) / 16;
        // many workgroups hide each other's ends: eight waves each then (32000 x 2048, one token: 17.3 -> 14.9 us), few
        // are done sooner with sixteen (2048 x 5632: 7.0 -> 5.4 us)
        if (grid > 1024) hipLaunchKernelGGL(k_i8_few<8>, dim3(grid), dim3(512), 0, st, a);
        else hipLaunchKernelGGL(k_i8_few<16>, dim3(grid), dim3(1024), 0, st, a);
    } else {
        return pk_fail(who, "T * n_rows is too large for one call");
    }
    return hipGetLastError() == hipSuccess ? 0 : pk_fail(who, "the launch failed");
}

} // extern "C"
