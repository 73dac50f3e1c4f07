// pages.hip — which sequence holds which page of a paged cache, kept on the
// device: reserving, giving back, forking (shared pages, counted), compacting
// and copying pages.
//
// All of it is integer bookkeeping on tables and reference counts, next to
// copies of whole pages that are bound by memory.  Pages are given lowest free
// first in the order of the requests: ranks come from prefix sums in one
// workgroup, never from the order of atomics, and the counts' atomic additions
// give the same sum in any order.
//
// That workgroup passes over all pages and requests, which is short where they
// are some thousands and is not in larger pools: compacting (nothing moves) 7.8,
// 20 and 147 us at 1000, 10^4 and 10^5 pages; a step's reserve, nothing to add,
// 7 us for 64 sequences of 128 blocks, 17 of 8192 blocks, 124 us for 1024
// sequences and 944 for 4096 (each request is compared with those before it);
// giving 90 % of 10^5 pages to 64 sequences 120 us.
#include "paged.h"

namespace {

constexpr int kWG = 1024;

struct copy_args {
    mllm_page_plane plane[MLLM_PAGE_PLANES];
    int n_planes;
    int units[MLLM_PAGE_PLANES + 1];   // units of a page before plane i (all its layers)
    int chunks[MLLM_PAGE_PLANES];      // units of one layer's slice, or
    int group[MLLM_PAGE_PLANES];       // layers whose slices a unit takes together (0: none)
    int n_pages;
};
constexpr int kCopy = 16384;           // bytes per unit: 256 threads x 4 x 16 bytes

__device__ __forceinline__ bool page_ok(const mllm_page_map &m, int p) { return p >= 0 && p < m.n_pages; }

// The exclusive prefix sum of v over the workgroup's threads, and the whole sum.
__device__ __forceinline__ int block_scan(int v, int &total, int *sh)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int x = v;
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    if (lane == 63) sh[w] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < kWG / 64; i++) {
        if (i < w) before += sh[i];
        total += sh[i];
    }
    __syncthreads();
    return before + x - v;
}

// The first `want` free pages in ascending order; returns how many there are (at most want).
__device__ int free_pages(const mllm_page_map &m, int want, int *list, int *sh)
{
    int found = 0;
    for (int p0 = 0; p0 < m.n_pages && found < want; p0 += 4 * kWG) {
        const int p = p0 + 4 * threadIdx.x;
        bool f[4];
        int n = 0, total;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[i] = p + i < m.n_pages && m.refs[p + i] == 0;
            n += f[i];
        }
        int at = found + block_scan(n, total, sh);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (f[i]) {
                if (at < want) list[at] = p + i;
                at++;
            }
        found += total;
    }
    __syncthreads();
    return found < want ? found : want;
}

// Whether request i of a wave's lanes is the first that names seqs[i].
__device__ __forceinline__ bool first_of(const int *seqs, int i, int lane)
{
    bool seen = false;
    for (int j = lane; j < i; j += 64) seen |= seqs[j] == seqs[i];
    return !__any(seen);
}

// One workgroup: counts of unmapped blocks per request (a wave each), their prefix sum, the free
// pages, then the blocks in order.  off: [n], list: [n_pages].
__global__ __launch_bounds__(kWG) void k_pages_reserve(mllm_page_map m, int n, const int *seqs, const int *lens,
                                                       int *status, int *off, int *list)
{
    __shared__ int sh[kWG / 64], left;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (threadIdx.x == 0) left = 0;
    __syncthreads();
    for (int i = w; i < n; i += kWG / 64) {
        const int seq = seqs[i], len = lens[i];
        const bool ok = seq >= 0 && seq < m.n_seqs && len >= 0 && len <= (long)m.max_blocks * m.page_size &&
                        first_of(seqs, i, lane);
        int cnt = 0;
        if (ok) {
            const int nb = (int)(((long)len + m.page_size - 1) / m.page_size);
            for (int b = lane; b < nb; b += 64) cnt += !page_ok(m, m.tables[seq * m.table_ld + b]);
            for (int d = 32; d; d >>= 1) cnt += __shfl_xor(cnt, d, 64);
        }
        if (lane == 0) {
            off[i] = ok ? cnt : -1;
            if (!ok) atomicAdd(&left, 1);
        }
    }
    __syncthreads();
    int want = 0;
    for (int i0 = 0; i0 < n; i0 += kWG) {
        const int i = i0 + threadIdx.x, c = i < n ? off[i] : 0;
        int total;
        const int at = block_scan(c > 0 ? c : 0, total, sh);
        if (i < n) off[i] = c > 0 ? want + at : -1;   // nothing to do: -1
        want += total;
    }
    __syncthreads();
    const int got = free_pages(m, want, list, sh);
    for (int i = w; i < n; i += kWG / 64) {
        int at = off[i];
        if (at < 0) continue;
        int *row = m.tables + seqs[i] * m.table_ld;
        const int nb = (int)(((long)lens[i] + m.page_size - 1) / m.page_size);
        for (int b0 = 0; b0 < nb; b0 += 64) {
            const int b = b0 + lane;
            const bool need = b < nb && !page_ok(m, row[b]);
            const unsigned long long mask = __ballot(need);
            const int r = at + __popcll(mask & ((1ull << lane) - 1));
            if (need) {
                row[b] = r < got ? list[r] : -1;
                if (r < got) m.refs[list[r]] = 1;
            }
            at += __popcll(mask);
        }
    }
    if (threadIdx.x == 0) *status = left + want - got;
}

// grid (blocks / 256, n): the exchange makes a sequence that is listed twice harmless.
__global__ __launch_bounds__(256) void k_pages_free(mllm_page_map m, const int *seqs, const int *lens)
{
    const int i = blockIdx.y, b = blockIdx.x * 256 + threadIdx.x, seq = seqs[i];
    const int len = lens ? lens[i] : 0;
    if (seq < 0 || seq >= m.n_seqs || len < 0 || b >= m.max_blocks) return;
    if (b < ((long)len + m.page_size - 1) / m.page_size) return;
    const int p = atomicExch(m.tables + seq * m.table_ld + b, -1);
    if (page_ok(m, p)) atomicSub(m.refs + p, 1);
}

// Fork, first step: the children's new rows (without the copied page) from the parents' rows as they
// are, and the shared pages' counts.  grid (blocks / 256, n).  src[i]: the page to copy, -1 none,
// -2 nothing to do, -3 left out.
__global__ __launch_bounds__(256) void k_fork_rows(mllm_page_map m, int n, const int *parents, const int *children,
                                                   const int *lens, int *rows, int *src)
{
    const int i = blockIdx.y, b = blockIdx.x * 256 + threadIdx.x, par = parents[i], ch = children[i], len = lens[i];
    bool ok = par >= 0 && par < m.n_seqs && ch >= 0 && ch < m.n_seqs && len >= 0 &&
              len <= (long)m.max_blocks * m.page_size;
    bool seen = false;
    for (int j = threadIdx.x; j < i; j += 256) seen |= children[j] == ch;
    if (__syncthreads_or(seen)) ok = false;
    const int full = ok ? len / m.page_size : 0;
    const int *row = m.tables + (ok ? par : 0) * m.table_ld;
    if (b == 0) {
        int s = !ok ? -3 : par == ch ? -2 : -1;
        if (s == -1 && len % m.page_size) {
            const int p = row[full];
            if (page_ok(m, p)) s = p;
        }
        src[i] = s;
    }
    if (!ok || par == ch || b >= m.max_blocks) return;
    const int p = b < full ? row[b] : -1;
    const bool shared = page_ok(m, p);
    rows[(long)i * m.max_blocks + b] = shared ? p : -1;
    if (shared) atomicAdd(m.refs + p, 1);
}

// Second step, one workgroup: a free page for each copied one.  The pages that the children give
// back are still counted, so none of them is overwritten before it has been copied.
__device__ __forceinline__ void fork_pages(const mllm_page_map &m, int n, const int *src, int *dst, int *list, int *status,
                                           int *sh, int &left)
{
    if (threadIdx.x == 0) left = 0;
    __syncthreads();
    int want = 0;
    for (int i0 = 0; i0 < n; i0 += kWG) {
        const int i = i0 + threadIdx.x, s = i < n ? src[i] : -1;
        if (s == -3) atomicAdd(&left, 1);
        int total;
        const int at = block_scan(s >= 0, total, sh);
        if (i < n) dst[i] = s >= 0 ? want + at : -1;
        want += total;
    }
    __syncthreads();
    const int got = free_pages(m, want, list, sh);
    for (int i = threadIdx.x; i < n; i += kWG) {
        const int r = dst[i], p = r >= 0 && r < got ? list[r] : -1;
        dst[i] = p;
        if (p >= 0) m.refs[p] = 1;
    }
    if (threadIdx.x == 0) *status = left + want - got;
}

__global__ __launch_bounds__(kWG) void k_fork_pages(mllm_page_map m, int n, const int *src, int *dst, int *list,
                                                    int *status)
{
    __shared__ int sh[kWG / 64], left;
    fork_pages(m, n, src, dst, list, status, sh, left);
}

// Both steps in one workgroup, a wave per request.
__global__ __launch_bounds__(kWG) void k_fork_plan(mllm_page_map m, int n, const int *parents, const int *children,
                                                   const int *lens, int *rows, int *src, int *dst, int *list, int *status)
{
    __shared__ int sh[kWG / 64], left;
    const int lane = threadIdx.x & 63;
    for (int i = threadIdx.x >> 6; i < n; i += kWG / 64) {
        const int par = parents[i], ch = children[i], len = lens[i];
        const bool ok = par >= 0 && par < m.n_seqs && ch >= 0 && ch < m.n_seqs && len >= 0 &&
                        len <= (long)m.max_blocks * m.page_size && first_of(children, i, lane);
        const int full = ok ? len / m.page_size : 0;
        const int *row = m.tables + (ok ? par : 0) * m.table_ld;
        if (lane == 0) {
            const int p = ok && par != ch && len % m.page_size ? row[full] : -1;
            src[i] = !ok ? -3 : par == ch ? -2 : page_ok(m, p) ? p : -1;
        }
        if (!ok || par == ch) continue;
        for (int b = lane; b < m.max_blocks; b += 64) {
            const int p = b < full ? row[b] : -1;
            const bool shared = page_ok(m, p);
            rows[(long)i * m.max_blocks + b] = shared ? p : -1;
            if (shared) atomicAdd(m.refs + p, 1);
        }
    }
    __syncthreads();
    fork_pages(m, n, src, dst, list, status, sh, left);
}

// One unit of a page's copy: 16 KB of one layer's slice of one plane, or the slices of several layers
// that are 16 KB together.  The pages are not read again soon and pass the caches by: 17 copies of 3.1 MB
// pages 28.9 -> 20.2 us, 134 of 0.5 MB 56.5 -> 37.5 us (stores that stay in L2 evict what is read; loads
// past the caches as well 44 us).
__device__ __forceinline__ void copy_unit(const copy_args &c, int unit, int src, int dst)
{
    int i = 0;
    while (i + 1 < c.n_planes && unit >= c.units[i + 1]) i++;
    const mllm_page_plane &pl = c.plane[i];
    const int k = unit - c.units[i];
    uint8_t *base = (uint8_t *)pl.base;
    const long from = src * pl.page_bytes, to = dst * pl.page_bytes;
    const bool wide = !(((uintptr_t)base | (uintptr_t)pl.page_bytes | (uintptr_t)pl.layer_bytes) & 15);
    if (c.group[i]) {
        const int l0 = k * c.group[i], nl = min(c.group[i], pl.n_layers - l0);
        if (wide) {
            const int per = (int)(pl.page_bytes / 16);
            for (int x = threadIdx.x; x < nl * per; x += 256) {
                const int layer = x / per;
                uint8_t *p = base + (l0 + layer) * pl.layer_bytes + 16 * (x - layer * per);
                __builtin_nontemporal_store(*(const u32x4 *)(p + from), (u32x4 *)(p + to));
            }
        } else {
            const int per = (int)pl.page_bytes;
            for (int x = threadIdx.x; x < nl * per; x += 256) {
                const int layer = x / per;
                uint8_t *p = base + (l0 + layer) * pl.layer_bytes + (x - layer * per);
                p[to] = p[from];
            }
        }
        return;
    }
    const int layer = k / c.chunks[i], chunk = k - layer * c.chunks[i];
    const long o = (long)chunk * kCopy;
    base += layer * pl.layer_bytes + o;
    const int n = (int)(pl.page_bytes - o < kCopy ? pl.page_bytes - o : kCopy);
    if (wide) {
        u32x4 v[4];
        const int e = n / 16;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (threadIdx.x + 256 * j < e) v[j] = ((const u32x4 *)(base + from))[threadIdx.x + 256 * j];
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (threadIdx.x + 256 * j < e) __builtin_nontemporal_store(v[j], (u32x4 *)(base + to) + threadIdx.x + 256 * j);
    } else {
        for (int j = threadIdx.x; j < n; j += 256) base[to + j] = base[from + j];
    }
}

// Units wg, + wgs, ... of `moves` page copies.
__device__ __forceinline__ void copy_pages(const copy_args &c, const int *src, const int *dst, int moves, int wg, int wgs)
{
    const int per = c.units[c.n_planes];
    for (long u = wg; u < (long)moves * per; u += wgs) {
        const int i = (int)(u / per), s = src[i], d = dst[i];
        if (s < 0 || s >= c.n_pages || d < 0 || d >= c.n_pages || s == d) continue;
        copy_unit(c, (int)(u - (long)i * per), s, d);
    }
}

// Third step of the fork: workgroups below `rowg` write the children's rows and give their former
// pages back, the others copy.
__global__ __launch_bounds__(256) void k_fork_apply(mllm_page_map m, copy_args c, int n, const int *children,
                                                    const int *lens, const int *rows, const int *src, const int *dst,
                                                    int rowg, int per_row)
{
    if ((int)blockIdx.x >= rowg) {
        copy_pages(c, src, dst, n, blockIdx.x - rowg, gridDim.x - rowg);
        return;
    }
    const int i = blockIdx.x / per_row, b = (blockIdx.x - i * per_row) * 256 + threadIdx.x;
    if (src[i] <= -2 || b >= m.max_blocks) return;
    int p = rows[(long)i * m.max_blocks + b];
    if (src[i] >= 0 && b == lens[i] / m.page_size) p = dst[i];
    int *e = m.tables + children[i] * m.table_ld + b;
    const int old = *e;
    *e = p;
    if (page_ok(m, old)) atomicSub(m.refs + old, 1);
}

// Compact, first step, one workgroup: the number L of live pages, which of them move where, and the
// counts of the moved ones.  to[p]: where page p >= L goes.
__global__ __launch_bounds__(kWG) void k_compact_plan(mllm_page_map m, int *src, int *dst, int *to, int *count,
                                                      int *status)
{
    __shared__ int sh[kWG / 64];
    int live = 0;
    for (int p = threadIdx.x; p < m.n_pages; p += kWG) live += m.refs[p] != 0;
    int L;
    block_scan(live, L, sh);
    int holes = 0, moved = 0;
    for (int p0 = 0; p0 < m.n_pages; p0 += kWG) {
        const int p = p0 + threadIdx.x;
        const bool used = p < m.n_pages && m.refs[p] != 0;
        const bool hole = p < L && p < m.n_pages && !used, move = p >= L && used;
        int nh, nm;
        const int ah = holes + block_scan(hole, nh, sh), am = moved + block_scan(move, nm, sh);
        if (hole) dst[ah] = p;
        if (move) src[am] = p;
        if (p >= L && p < m.n_pages) to[p] = p;
        holes += nh;
        moved += nm;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < moved; i += kWG) {
        to[src[i]] = dst[i];
        m.refs[dst[i]] = m.refs[src[i]];
        m.refs[src[i]] = 0;
    }
    if (threadIdx.x == 0) {
        *status = L;
        count[0] = moved;
        count[1] = L;
    }
}

__global__ __launch_bounds__(256) void k_compact_apply(mllm_page_map m, copy_args c, const int *src, const int *dst,
                                                       const int *to, const int *count, int rowg)
{
    if ((int)blockIdx.x >= rowg) {
        copy_pages(c, src, dst, count[0], blockIdx.x - rowg, gridDim.x - rowg);
        return;
    }
    const int L = count[1];
    for (long i = blockIdx.x * 256l + threadIdx.x; i < (long)m.n_seqs * m.max_blocks; i += rowg * 256l) {
        const long s = i / m.max_blocks;
        int *e = m.tables + s * m.table_ld + (i - s * m.max_blocks);
        const int p = *e;
        if (p >= L && p < m.n_pages) *e = to[p];
    }
}

__global__ __launch_bounds__(256) void k_pages_copy(copy_args c, const int *src, const int *dst, int n)
{
    copy_pages(c, src, dst, n, blockIdx.x, gridDim.x);
}

const char *map_refusal(const mllm_page_map *m)
{
    if (!m || !m->tables || !m->refs) return "a map needs tables and refs";
    if (m->n_seqs <= 0 || m->max_blocks <= 0 || m->n_pages <= 0 || m->page_size <= 0 || m->table_ld < m->max_blocks)
        return "n_seqs, max_blocks, n_pages and page_size are positive, table_ld at least max_blocks";
    return nullptr;
}

const char *planes_refusal(const mllm_page_plane *planes, int n_planes, int n_pages, copy_args &c)
{
    if (n_planes < 0 || n_planes > MLLM_PAGE_PLANES || (n_planes && !planes)) return "0 to MLLM_PAGE_PLANES planes";
    c = copy_args{};
    c.n_planes = n_planes;
    c.n_pages = n_pages;
    long units = 0;
    for (int i = 0; i < n_planes; i++) {
        const mllm_page_plane &p = planes[i];
        if (!p.base || p.page_bytes <= 0 || p.n_layers <= 0 ||
            (p.n_layers > 1 && p.layer_bytes < p.page_bytes * n_pages))
            return "a plane needs a base, page_bytes, n_layers and layers that do not overlap";
        c.plane[i] = p;
        const long chunks = (p.page_bytes + kCopy - 1) / kCopy;
        c.units[i] = (int)units;
        c.chunks[i] = (int)chunks;
        c.group[i] = 2 * p.page_bytes <= kCopy ? (int)(kCopy / p.page_bytes) : 0;
        units += c.group[i] ? (p.n_layers + c.group[i] - 1) / c.group[i] : chunks * p.n_layers;
        if (units > 1 << 30) return "pages of at most 2^44 bytes";
    }
    c.units[n_planes] = (int)units;
    return nullptr;
}

long a64(long ints) { return (ints + 63) / 64 * 64; }

// Workgroups of a copy: enough to fill the GPU several times over, no more than units.
int copy_grid(const copy_args &c, long moves)
{
    const long u = moves * c.units[c.n_planes];
    return (int)(u < 1 ? 1 : u < 4096 ? u : 4096);
}

int launched(const char *who) { return hipGetLastError() == hipSuccess ? 0 : pk_fail(who, "the launch failed"); }

} // namespace

extern "C" {

// ints: offsets or sources [n], destinations [n], new rows [n * max_blocks], a list of pages, and
// for compact two more and two counts
MLLM_API long mllm_pages_workspace_size(const mllm_page_map *m, int n)
{
    if (map_refusal(m) || n < 0) return -1;
    return 4 * (2 * a64(n) + a64((long)n * m->max_blocks) + 3 * a64(m->n_pages) + 64);
}

MLLM_API int mllm_pages_reserve(const mllm_page_map *m, int n, const int *seqs, const int *lens, int *status,
                                void *workspace, long ws_bytes, void *stream)
{
    const char *who = "mllm_pages_reserve";
    if (const char *why = map_refusal(m)) return pk_fail(who, why);
    if (n < 0 || (n && (!seqs || !lens)) || !status) return pk_fail(who, "seqs, lens and status are needed");
    if (!workspace || ws_bytes < mllm_pages_workspace_size(m, n)) return pk_fail(who, "workspace below mllm_pages_workspace_size");
    int *w = (int *)workspace;
    hipLaunchKernelGGL(k_pages_reserve, dim3(1), dim3(kWG), 0, (hipStream_t)stream, *m, n, seqs, lens, status, w, w + a64(n));
    return launched(who);
}

MLLM_API int mllm_pages_free(const mllm_page_map *m, int n, const int *seqs, const int *lens, void *stream)
{
    const char *who = "mllm_pages_free";
    if (const char *why = map_refusal(m)) return pk_fail(who, why);
    if (n < 0 || n > 65535 || (n && !seqs)) return pk_fail(who, "seqs is needed, at most 65535 of them");
    if (!n) return 0;
    hipLaunchKernelGGL(k_pages_free, dim3((m->max_blocks + 255) / 256, n), dim3(256), 0, (hipStream_t)stream, *m, seqs, lens);
    return launched(who);
}

MLLM_API int mllm_pages_fork(const mllm_page_map *m, const mllm_page_plane *planes, int n_planes, int n,
                             const int *parents, const int *children, const int *lens, int *status, void *workspace,
                             long ws_bytes, void *stream)
{
    const char *who = "mllm_pages_fork";
    copy_args c;
    if (const char *why = map_refusal(m)) return pk_fail(who, why);
    if (const char *why = planes_refusal(planes, n_planes, m->n_pages, c)) return pk_fail(who, why);
    const long per_row = ((long)m->max_blocks + 255) / 256;
    if (n < 0 || n > 65535 || (n && (!parents || !children || !lens)) || !status || n * per_row > 1 << 30)
        return pk_fail(who, "parents, children, lens and status are needed, at most 65535 requests");
    if (!workspace || ws_bytes < mllm_pages_workspace_size(m, n)) return pk_fail(who, "workspace below mllm_pages_workspace_size");
    hipStream_t st = (hipStream_t)stream;
    int *src = (int *)workspace, *dst = src + a64(n), *rows = dst + a64(n), *list = rows + a64((long)n * m->max_blocks);
    // a workgroup has 16 waves: up to four rounds of them take no longer than another launch (4 us)
    if ((long)n * ((m->max_blocks + 63) / 64) <= 64) {
        hipLaunchKernelGGL(k_fork_plan, dim3(1), dim3(kWG), 0, st, *m, n, parents, children, lens, rows, src, dst, list, status);
    } else {
        hipLaunchKernelGGL(k_fork_rows, dim3(per_row, n), dim3(256), 0, st, *m, n, parents, children, lens, rows, src);
        hipLaunchKernelGGL(k_fork_pages, dim3(1), dim3(kWG), 0, st, *m, n, src, dst, list, status);
    }
    if (n) {
        const int rowg = (int)(n * per_row);
        hipLaunchKernelGGL(k_fork_apply, dim3(rowg + copy_grid(c, n)), dim3(256), 0, st, *m, c, n, children, lens, rows,
                           src, dst, rowg, (int)per_row);
    }
    return launched(who);
}

MLLM_API int mllm_pages_compact(const mllm_page_map *m, const mllm_page_plane *planes, int n_planes, int *status,
                                void *workspace, long ws_bytes, void *stream)
{
    const char *who = "mllm_pages_compact";
    copy_args c;
    if (const char *why = map_refusal(m)) return pk_fail(who, why);
    if (const char *why = planes_refusal(planes, n_planes, m->n_pages, c)) return pk_fail(who, why);
    if (!status) return pk_fail(who, "status is needed");
    if (!workspace || ws_bytes < mllm_pages_workspace_size(m, 0)) return pk_fail(who, "workspace below mllm_pages_workspace_size");
    hipStream_t st = (hipStream_t)stream;
    int *count = (int *)workspace, *src = count + 64, *dst = src + a64(m->n_pages), *to = dst + a64(m->n_pages);
    hipLaunchKernelGGL(k_compact_plan, dim3(1), dim3(kWG), 0, st, *m, src, dst, to, count, status);
    const long e = (long)m->n_seqs * m->max_blocks;
    const int rowg = (int)(e < 256l * 512 ? (e + 255) / 256 : 512);
    hipLaunchKernelGGL(k_compact_apply, dim3(rowg + copy_grid(c, m->n_pages / 2)), dim3(256), 0, st, *m, c, src, dst, to,
                       count, rowg);
    return launched(who);
}

MLLM_API int mllm_pages_copy(const mllm_page_plane *planes, int n_planes, int n_pages, int n, const int *src,
                             const int *dst, void *stream)
{
    const char *who = "mllm_pages_copy";
    copy_args c;
    if (n_pages <= 0) return pk_fail(who, "n_pages is positive");
    if (const char *why = planes_refusal(planes, n_planes, n_pages, c)) return pk_fail(who, why);
    if (n < 0 || (n && (!src || !dst))) return pk_fail(who, "src and dst are needed");
    if (!n || !n_planes) return 0;
    hipLaunchKernelGGL(k_pages_copy, dim3(copy_grid(c, n)), dim3(256), 0, (hipStream_t)stream, c, src, dst, n);
    return launched(who);
}

} // extern "C"
