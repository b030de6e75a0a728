// kv_evict.cuh — eviction of a paged cache's rows by score, in place.
//
// Per (stream, KV head), of n rows the m = min(n, keep) best stay.
// kv_evict_select_kernel finds them (one CTA per (stream, head)), writes the new
// score / position / source arrays and the list of moves; kv_evict_move_kernel
// copies the K and V rows of the moves and writes the new lengths.  With few
// moves the first kernel does that too (UNIT > 0).  A move takes a kept row at or behind m to a gap below m, so no row
// is both read and written and the moves run in any order.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>
#include "vtx_ptx.cuh"
#include "paged_kv.cuh"

namespace vtx {

struct PagedEvictArgs {
    PagedView kv;
    const float *score; const int *row_pos; const int *next_pos;
    float *score_out; int *pos_out, *src_out, *kv_len_out;
    int keep, n_sink, n_recent, row_cap, out_cap;
    int2 *moves;              // [n_seq * Hkv][max_moves] (source row, destination row)
    int2 *counts;             // [n_seq * Hkv] (moves, rows left)
    int max_moves;
    int row_bytes;            // bytes of one head's row
    int slices;               // CTAs per (stream, head) of the move kernel
};

constexpr int kEvictThreads = 512, kEvictWarps = kEvictThreads / 32;
constexpr int kEvictBins = 2048;                  // 11-bit digits: 11 + 11 + 10 bits of a key
constexpr int kEvictKeysInSmem = 48 * 1024;       // rows whose keys fit in shared memory
constexpr int kEvictBatch = 8;                    // moves a warp has in flight

// Order-preserving key: protected rows above everything, NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t evict_key(float x, bool safe) {
    if (safe) return 0xffffffffu;
    if (x != x) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Copies moves i0, i0 + step, ... (batches of eight) of a (stream, head): lanes
// 0-7 read the moves and their pages, then half of the warp takes the K row and
// half the V row of each move, all loads before the first store.  UNIT: bytes a
// lane copies at once (16, 8 or 4).
template <int UNIT> struct EvictUnit;
template <> struct EvictUnit<16> { using V = uint4; };
template <> struct EvictUnit<8> { using V = uint2; };
template <> struct EvictUnit<4> { using V = uint32_t; };
template <int UNIT>
__device__ __forceinline__ void evict_move(const PagedEvictArgs &a, const int2 *mv, int count, int i0, int step, int b,
                                           int g, int lane)
{
    using V = typename EvictUnit<UNIT>::V;
    constexpr int N = UNIT == 16 ? 1 : 2;          // rows of 128 / 256, 136 and 68 bytes over 16 lanes
    char *pool = lane < 16 ? a.kv.k : a.kv.v;
    const int units = a.row_bytes / UNIT, u0 = lane & 15;
    const long long head = (long long)g * a.kv.nb2;
    const int mask = (1 << a.kv.shift) - 1;
    for (; i0 < count; i0 += step) {
        long long src = -1, dst = -1;
        if (lane < kEvictBatch && i0 + lane < count) {
            const int2 x = mv[i0 + lane];
            const int ps = paged_page(a.kv, b, x.x), pd = paged_page(a.kv, b, x.y);
            if (ps >= 0 && pd >= 0) {
                src = head + (long long)ps * a.kv.nb3 + (long long)(x.x & mask) * a.kv.nb1;
                dst = head + (long long)pd * a.kv.nb3 + (long long)(x.y & mask) * a.kv.nb1;
            }
        }
        V v[kEvictBatch][N];
#pragma unroll
        for (int i = 0; i < kEvictBatch; ++i) {
            const long long at = __shfl_sync(0xffffffffu, src, i);
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (at >= 0 && u0 + 16 * k < units) v[i][k] = reinterpret_cast<const V *>(pool + at)[u0 + 16 * k];
        }
#pragma unroll
        for (int i = 0; i < kEvictBatch; ++i) {
            const long long at = __shfl_sync(0xffffffffu, dst, i);
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (at >= 0 && u0 + 16 * k < units) reinterpret_cast<V *>(pool + at)[u0 + 16 * k] = v[i][k];
        }
    }
}

// The m-th largest key by a radix select from the top digit down: a histogram of
// the keys that match the prefix so far, then the bin that holds the m-th.  Rows
// with a larger key are kept, of those with an equal one the first ones.  A warp
// owns a run of rows and walks it 32 at a time, so ballots number the equal keys,
// the gaps and the moved rows in row order.  Bound by latency: about a dozen
// barriers and four dependent trips to memory per (stream, head).
template <bool SMEM, int UNIT>
__global__ void __launch_bounds__(kEvictThreads)
kv_evict_select_kernel(const PagedEvictArgs a)
{
    grid_dep_wait();
    grid_dep_launch();
    extern __shared__ uint32_t keys[];
    __shared__ int hist[kEvictBins];
    __shared__ int2 warp_sum[kEvictWarps];
    __shared__ int pick[2];
    const int b = blockIdx.x / a.kv.Hkv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned below = (1u << lane) - 1;
    const long long item = blockIdx.x;
    const int n = a.kv.kv_len[b];
    const int most = (int)min((long long)min(a.kv.max_kv, a.row_cap), (long long)a.kv.max_pages << a.kv.shift);
    if (n < 0 || n > most) {                       // nothing of this stream is touched
        if (tid == 0) {
            paged_report(a.kv, VTX_KERR_BOUND);
            if (UNIT == 0) a.counts[item] = make_int2(0, n);
            else if (item % a.kv.Hkv == 0) a.kv_len_out[b] = n;
        }
        return;
    }
    const int m = min(n, a.keep);
    const float *score = a.score + item * a.row_cap;
    const int *row_pos = a.row_pos ? a.row_pos + item * a.row_cap : nullptr;
    const int recent = (a.next_pos ? a.next_pos[b] : n) - a.n_recent;
    auto key_of = [&](int j) {
        const int p = row_pos ? row_pos[j] : j;
        return evict_key(score[j], p < a.n_sink || p >= recent);
    };
    const bool some = m > 0 && m < n;              // there is a choice to make
    if (SMEM && some)
        for (int j = tid; j < n; j += kEvictThreads) keys[j] = key_of(j);
    uint32_t prefix = 0;
    int need = m;                                  // rank of the threshold among the keys that match the prefix
    if (some) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            for (int i = tid; i < kEvictBins; i += kEvictThreads) hist[i] = 0;
            __syncthreads();
            for (int j = tid; j < n; j += kEvictThreads) {
                const uint32_t k = SMEM ? keys[j] : key_of(j);
                if (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits)))
                    atomicAdd(&hist[(k >> shift) & ((1 << bits) - 1)], 1);
            }
            __syncthreads();
            // thread i: the four bins from 2047 - 4i down; the sum of all above it by a scan
            int c[4], t = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) { c[i] = hist[kEvictBins - 1 - 4 * tid - i]; t += c[i]; }
            int inc = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += x;
            }
            if (lane == 31) warp_sum[warp].x = inc;
            __syncthreads();
            int above = inc - t;
#pragma unroll
            for (int w = 0; w < kEvictWarps; ++w) above += w < warp ? warp_sum[w].x : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (above < need && above + c[i] >= need) {
                    pick[0] = kEvictBins - 1 - 4 * tid - i;
                    pick[1] = need - above;
                }
                above += c[i];
            }
            __syncthreads();
            prefix |= (uint32_t)pick[0] << shift;
            need = pick[1];
        }
    }
    // keys > prefix stay, and the first `need` of those equal to it
    const int run = (n + kEvictThreads - 1) / kEvictThreads * 32;
    const int r0 = min(warp * run, n), r1 = min(r0 + run, n);
    // exclusive sums over the warps of two counts, and their totals
    auto sums = [&](int x, int y, int2 &total) {
        __syncthreads();
        if (lane == 0) warp_sum[warp] = make_int2(x, y);
        __syncthreads();
        int2 before = make_int2(0, 0);
        total = before;
#pragma unroll
        for (int w = 0; w < kEvictWarps; ++w) {
            if (w == warp) before = total;
            total.x += warp_sum[w].x;
            total.y += warp_sum[w].y;
        }
        return before;
    };
    int2 tot;
    int eq0 = 0;
    if (some) {
        for (int j = r0 + lane; j - lane < r1; j += 32)
            eq0 += __popc(__ballot_sync(0xffffffffu, j < r1 && (SMEM ? keys[j] : key_of(j)) == prefix));
        eq0 = sums(eq0, 0, tot).x;
    }
    auto each = [&](auto f) {                      // f(row, live, kept), a warp's rows in order
        int e = eq0;
        for (int j = r0 + lane; j - lane < r1; j += 32) {
            const bool live = j < r1;
            bool kept = live && m == n;
            if (some) {
                const uint32_t k = live ? (SMEM ? keys[j] : key_of(j)) : 0u;
                const unsigned same = __ballot_sync(0xffffffffu, live && k == prefix);
                kept = live && (k > prefix || (k == prefix && e + __popc(same & below) < need));
                e += __popc(same);
            }
            f(j, live, kept);
        }
    };
    int gaps = 0, late = 0;                        // gaps below m, kept rows behind it
    if (some)
        each([&](int j, bool live, bool kept) {
            gaps += __popc(__ballot_sync(0xffffffffu, live && j < m && !kept));
            late += __popc(__ballot_sync(0xffffffffu, j >= m && kept));
        });
    int2 at = sums(gaps, late, tot);
    int2 *mv = a.moves + item * a.max_moves;
    float *so = a.score_out ? a.score_out + item * a.out_cap : nullptr;
    int *po = a.pos_out ? a.pos_out + item * a.out_cap : nullptr;
    int *ro = a.src_out ? a.src_out + item * a.out_cap : nullptr;
    each([&](int j, bool live, bool kept) {
        const unsigned gap = __ballot_sync(0xffffffffu, live && j < m && !kept);
        const unsigned far = __ballot_sync(0xffffffffu, j >= m && kept);
        if ((gap >> lane) & 1u) mv[at.x + __popc(gap & below)].y = j;
        if ((far >> lane) & 1u) mv[at.y + __popc(far & below)].x = j;
        at.x += __popc(gap);
        at.y += __popc(far);
        if (j < m && kept) {                       // in place these stand already
            if (so && so != score) so[j] = score[j];
            if (po && po != row_pos) po[j] = row_pos ? row_pos[j] : j;
            if (ro) ro[j] = j;
        }
    });
    __syncthreads();
    for (int i = tid; i < tot.x; i += kEvictThreads) {
        const int2 x = mv[i];
        if (so) so[x.y] = score[x.x];
        if (po) po[x.y] = row_pos ? row_pos[x.x] : x.x;
        if (ro) ro[x.y] = x.x;
    }
    if constexpr (UNIT == 0) {
        if (tid == 0) a.counts[item] = make_int2(tot.x, m);
    } else {
        evict_move<UNIT>(a, mv, tot.x, warp * kEvictBatch, kEvictWarps * kEvictBatch, b, (int)(item % a.kv.Hkv), lane);
        if (tid == 0 && item % a.kv.Hkv == 0) a.kv_len_out[b] = m;
    }
}

// Grid (n_seq * Hkv * slices).
template <int UNIT>
__global__ void __launch_bounds__(256)
kv_evict_move_kernel(const PagedEvictArgs a)
{
    grid_dep_wait();
    grid_dep_launch();
    const int slice = blockIdx.x % a.slices, item = blockIdx.x / a.slices;
    const int g = item % a.kv.Hkv, b = item / a.kv.Hkv;
    const int2 c = a.counts[item];
    if (slice == 0 && g == 0 && threadIdx.x == 0) a.kv_len_out[b] = c.y;
    evict_move<UNIT>(a, a.moves + (long long)item * a.max_moves, c.x, (slice * 8 + (threadIdx.x >> 5)) * kEvictBatch,
                     a.slices * 8 * kEvictBatch, b, g, threadIdx.x & 31);
}

}  // namespace vtx
