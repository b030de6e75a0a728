// kv_evict.cuh — eviction of a paged cache's rows by score, in place.
//
// Per (stream, KV head), of n rows the m = min(n, keep) best stay.
// kv_evict_select_kernel finds them (one CTA per (stream, head)), writes the new
// score / position / source arrays and the list of moves; kv_evict_move_kernel
// copies the K and V rows of the moves and writes the new lengths.  With few
// moves the first kernel does that too (UNIT > 0).  A move takes a kept row at or
// behind m to a gap below m, so no row is both read and written and the moves run
// in any order.
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
// owns a run of rows and walks it 128 at a time, four consecutive rows per lane, so
// a scan over the lanes numbers the gaps and the moved rows in row order.  Bound by
// latency: about a dozen barriers and four dependent trips to memory per (stream,
// head), so rows are read four at a time and four such loads together (64 items of
// 1500 to 8192 rows with their moves 38 -> 24.6 -> 22.6 us, 256 items 78 -> 71).
template <bool SMEM, int UNIT>
__global__ void __launch_bounds__(kEvictThreads)
kv_evict_select_kernel(const PagedEvictArgs a)
{
    grid_dep_wait();
    grid_dep_launch();
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ int hist[kEvictBins];
    __shared__ int2 warp_sum[kEvictWarps];
    __shared__ int pick[3];
    const int b = blockIdx.x / a.kv.Hkv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const long long item = blockIdx.x;
    const int n = a.kv.kv_len[b];
    const int most = min(min(a.kv.max_kv, a.row_cap), a.kv.cap);
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
    const int n4 = (n + 3) >> 2;
    const bool wide = a.row_cap % 4 == 0 &&        // rows of four start on 16 bytes
                      ((reinterpret_cast<uintptr_t>(a.score) | reinterpret_cast<uintptr_t>(a.row_pos)) & 15) == 0;
    auto load4 = [&](int q, float (&s)[4], int (&p)[4]) {       // rows 4q ... 4q + 3 (below n)
        if (wide) {
            const float4 x = reinterpret_cast<const float4 *>(score)[q];
            s[0] = x.x; s[1] = x.y; s[2] = x.z; s[3] = x.w;
            if (row_pos) {
                const int4 y = reinterpret_cast<const int4 *>(row_pos)[q];
                p[0] = y.x; p[1] = y.y; p[2] = y.z; p[3] = y.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = min(4 * q + i, n - 1);
                s[i] = score[j];
                if (row_pos) p[i] = row_pos[j];
            }
        }
        if (!row_pos) {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = 4 * q + i;
        }
    };
    // keys of rows 4q ... 4q + 3; 0, below every key, behind the last row
    auto key4 = [&](int q, const float (&s)[4], const int (&p)[4]) {
        uint32_t k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            k[i] = 4 * q + i < n ? evict_key(s[i], p[i] < a.n_sink || p[i] >= recent) : 0u;
        return make_uint4(k[0], k[1], k[2], k[3]);
    };
    auto make4 = [&](int q) {
        float s[4];
        int p[4];
        load4(q, s, p);
        return key4(q, s, p);
    };
    auto keys4 = [&](int q) { return SMEM ? reinterpret_cast<const uint4 *>(keys)[q] : make4(q); };
    const bool some = m > 0 && m < n;              // there is a choice to make
    constexpr int B = UNIT == 0 ? 4 : 1;           // trips to memory at once (UNIT > 0: one is all there is)
    if (SMEM && some) {
        for (int qb = tid; qb < n4; qb += B * kEvictThreads) {
            float s[B][4];
            int p[B][4];
#pragma unroll
            for (int i = 0; i < B; ++i)
                if (qb + i * kEvictThreads < n4) load4(qb + i * kEvictThreads, s[i], p[i]);
#pragma unroll
            for (int i = 0; i < B; ++i)
                if (const int q = qb + i * kEvictThreads; q < n4) reinterpret_cast<uint4 *>(keys)[q] = key4(q, s[i], p[i]);
        }
    }
    uint32_t prefix = 0;
    int need = m;                                  // rank of the threshold among the keys that match the prefix
    bool ties = false;                             // not all keys equal to the threshold stay
    if (some) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            for (int i = tid; i < kEvictBins; i += kEvictThreads) hist[i] = 0;
            __syncthreads();
            for (int q = tid; q < n4; q += kEvictThreads) {
                const uint4 k4 = keys4(q);
                const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (pass == 0 || (k[i] >> (shift + bits)) == (prefix >> (shift + bits)))
                        atomicAdd(&hist[(k[i] >> shift) & ((1 << bits) - 1)], 1);
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
                    pick[2] = c[i];
                }
                above += c[i];
            }
            __syncthreads();
            prefix |= (uint32_t)pick[0] << shift;
            need = pick[1];
            ties = pick[1] < pick[2];
        }
    }
    // keys > prefix stay, and the first `need` of those equal to it
    const int run = (n4 + kEvictThreads - 1) / kEvictThreads * 32;      // fours per warp
    const int q0 = min(warp * run, n4), q1 = min(q0 + run, n4);
    auto scan = [&](int x) {                       // exclusive sum over the lanes
        int inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        return inc - x;
    };
    auto all = [&](int x) {                        // sum over the lanes
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        return x;
    };
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
    int2 tot = make_int2(0, 0);
    int eq0 = 0;
    if (ties) {                                    // number the equal keys
        for (int q = q0 + lane; q < q1; q += 32) {
            const uint4 k = keys4(q);
            eq0 += (k.x == prefix) + (k.y == prefix) + (k.z == prefix) + (k.w == prefix);
        }
        eq0 = sums(all(eq0), 0, tot).x;
    }
    auto each = [&](auto f) {                      // f(four, bits of the rows that stay), a warp's fours in order
        int e = eq0;
        for (int q = q0 + lane; q - lane < q1; q += 32) {
            unsigned kept = 0;
            if (some) {
                const uint4 k4 = q < q1 ? keys4(q) : make_uint4(0u, 0u, 0u, 0u);
                const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
                if (ties) {
                    int same = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) same += k[i] == prefix;
                    int rank = e + scan(same);
                    e += all(same);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        kept |= (unsigned)(k[i] > prefix || (k[i] == prefix && rank < need)) << i;
                        rank += k[i] == prefix;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) kept |= (unsigned)(k[i] >= prefix) << i;
                }
            } else if (m == n) {
                kept = 15u;
            }
            // rows that exist, and those below m
            const int left = q < q1 ? min(max(n - 4 * q, 0), 4) : 0, low = min(max(m - 4 * q, 0), left);
            const unsigned live = (1u << left) - 1, front = (1u << low) - 1;
            f(q, kept & live, live, front);
        }
    };
    int gaps = 0, late = 0;                        // gaps below m, kept rows behind it
    if (some) {
        each([&](int, unsigned kept, unsigned live, unsigned front) {
            gaps += __popc(front & ~kept);
            late += __popc(kept & ~front);
        });
        gaps = all(gaps);
        late = all(late);
    }
    int2 at = sums(gaps, late, tot);
    int2 *mv = a.moves + item * a.max_moves;
    float *so = a.score_out ? a.score_out + item * a.out_cap : nullptr;
    int *po = a.pos_out ? a.pos_out + item * a.out_cap : nullptr;
    int *ro = a.src_out ? a.src_out + item * a.out_cap : nullptr;
    const bool put_s = so && so != score, put_p = po && po != row_pos;   // in place they stand already
    each([&](int q, unsigned kept, unsigned live, unsigned front) {
        const unsigned gap = front & ~kept, far = kept & ~front, stay = kept & front;
        const int x = scan(__popc(gap) | __popc(far) << 16), t = all(__popc(gap) | __popc(far) << 16);
        int g0 = at.x + (x & 0xffff), l0 = at.y + (x >> 16);
        at.x += t & 0xffff;
        at.y += t >> 16;
        float s[4];
        int p[4];
        if (stay && (put_s || put_p)) load4(q, s, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = 4 * q + i;
            if ((gap >> i) & 1u) mv[g0++].y = j;
            if ((far >> i) & 1u) mv[l0++].x = j;
            if ((stay >> i) & 1u) {
                if (put_s) so[j] = s[i];
                if (put_p) po[j] = p[i];
                if (ro) ro[j] = j;
            }
        }
    });
    __syncthreads();
    for (int ib = tid; ib < tot.x; ib += B * kEvictThreads) {
        int2 x[B];
        float s[B];
        int p[B];
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (ib + i * kEvictThreads < tot.x) x[i] = mv[ib + i * kEvictThreads];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (ib + i * kEvictThreads >= tot.x) break;
            if (so) s[i] = score[x[i].x];
            p[i] = po && row_pos ? row_pos[x[i].x] : x[i].x;
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (ib + i * kEvictThreads >= tot.x) break;
            if (so) so[x[i].y] = s[i];
            if (po) po[x[i].y] = p[i];
            if (ro) ro[x[i].y] = x[i].x;
        }
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
