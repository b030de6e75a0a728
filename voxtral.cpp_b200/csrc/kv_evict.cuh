// kv_evict.cuh — eviction of a paged cache's rows by score, in place.
//
// Per (stream, KV head), of n rows the m = min(n, keep) best stay.  Two
// kernels: kv_evict_select_kernel finds them (one CTA per (stream, head)),
// writes the new score / position / source arrays and the list of moves;
// kv_evict_move_kernel copies the K and V rows of the moves and writes the new
// lengths.  A move takes a kept row at or behind m to a gap below m, so no row
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
    int row_bytes, vec;       // bytes of one head's row; copy width
    int slices;               // CTAs per (stream, head) of the move kernel
};

constexpr int kEvictThreads = 1024;
constexpr int kEvictKeysInSmem = 48 * 1024;       // rows whose keys fit in shared memory

// Order-preserving key: protected rows above everything, NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t evict_key(float x, bool safe) {
    if (safe) return 0xffffffffu;
    if (x != x) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Exclusive sums over the CTA of two counts per thread; `total` gets both sums.
__device__ __forceinline__ int2 evict_scan(int2 x, int2 *warp_sum, int2 &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, inc.x, o), b = __shfl_up_sync(0xffffffffu, inc.y, o);
        if (lane >= o) { inc.x += a; inc.y += b; }
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    int2 base = make_int2(0, 0);
    total = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < kEvictThreads / 32; ++w) {
        if (w == warp) base = total;
        total.x += warp_sum[w].x;
        total.y += warp_sum[w].y;
    }
    return make_int2(base.x + inc.x - x.x, base.y + inc.y - x.y);
}

// The m-th largest key by a radix select, 8 bits at a time from the top: a
// histogram of the keys that match the prefix so far, then the bin that holds
// the m-th.  Rows with a larger key are kept, of those with an equal one the
// first ones.  Each thread owns a run of E consecutive rows, so two block
// scans number the gaps and the moved rows in row order.
template <bool SMEM>
__global__ void __launch_bounds__(kEvictThreads)
kv_evict_select_kernel(const PagedEvictArgs a)
{
    grid_dep_wait();
    grid_dep_launch();
    extern __shared__ uint32_t keys[];
    __shared__ int hist[256];
    __shared__ int2 warp_sum[kEvictThreads / 32];
    __shared__ int pick[2];
    const int b = blockIdx.x / a.kv.Hkv;
    const int tid = threadIdx.x;
    const long long item = blockIdx.x;
    int n = a.kv.kv_len[b];
    const int most = (int)min((long long)min(a.kv.max_kv, a.row_cap), (long long)a.kv.max_pages << a.kv.shift);
    if (n < 0 || n > most) {                       // nothing of this stream is touched
        if (tid == 0) {
            paged_report(a.kv, VTX_KERR_BOUND);
            a.counts[item] = make_int2(0, n);
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
    if (SMEM) {
        for (int j = tid; j < n; j += kEvictThreads) keys[j] = key_of(j);
    }
    uint32_t prefix = 0;
    int need = m;                                  // rank of the threshold among the keys that match the prefix
    if (m < n && m > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int j = tid; j < n; j += kEvictThreads) {
                const uint32_t k = SMEM ? keys[j] : key_of(j);
                if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid < 32) {                        // lane l: bins 255 - 8l ... 248 - 8l, from the top
                int c[8], t = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) { c[i] = hist[255 - 8 * tid - i]; t += c[i]; }
                int inc = t;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, inc, o);
                    if (tid >= o) inc += x;
                }
                int above = inc - t;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (above < need && above + c[i] >= need) { pick[0] = 255 - 8 * tid - i; pick[1] = need - above; }
                    above += c[i];
                }
            }
            __syncthreads();
            prefix |= (uint32_t)pick[0] << shift;
            need = pick[1];
        }
    }
    __syncthreads();
    // keys > prefix stay, and the first `need` of those equal to it
    const bool all = m == n;
    const int E = (n + kEvictThreads - 1) / kEvictThreads;
    const int j0 = min(tid * E, n), j1 = min(j0 + E, n);
    int2 tot;
    int eq = 0;
    if (!all && m > 0)
        for (int j = j0; j < j1; ++j) eq += (SMEM ? keys[j] : key_of(j)) == prefix;
    const int eq0 = evict_scan(make_int2(eq, 0), warp_sum, tot).x;
    auto each = [&](auto f) {                      // f(row, kept) over this thread's rows
        int e = eq0;
        for (int j = j0; j < j1; ++j) {
            bool kept = all;
            if (!all && m > 0) {
                const uint32_t k = SMEM ? keys[j] : key_of(j);
                kept = k > prefix || (k == prefix && e < need);
                e += k == prefix;
            }
            f(j, kept);
        }
    };
    int2 cnt = make_int2(0, 0);                    // gaps below m, kept rows behind it
    each([&](int j, bool kept) {
        cnt.x += j < m && !kept;
        cnt.y += j >= m && kept;
    });
    int2 at = evict_scan(cnt, warp_sum, tot);
    int2 *mv = a.moves + item * a.max_moves;
    float *so = a.score_out ? a.score_out + item * a.out_cap : nullptr;
    int *po = a.pos_out ? a.pos_out + item * a.out_cap : nullptr;
    int *ro = a.src_out ? a.src_out + item * a.out_cap : nullptr;
    each([&](int j, bool kept) {
        if (j < m && !kept) mv[at.x++].y = j;
        if (j >= m && kept) mv[at.y++].x = j;
        if (j < m && kept) {                       // in place these write what is there
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
    if (tid == 0) a.counts[item] = make_int2(tot.x, m);
}

template <typename V>
__device__ __forceinline__ void evict_copy_row(char *dst, const char *src, int n, int lane) {
    for (int i = lane; i < n; i += 32) reinterpret_cast<V *>(dst)[i] = reinterpret_cast<const V *>(src)[i];
}

// Grid (n_seq * Hkv * slices), a warp per move.
__global__ void __launch_bounds__(256)
kv_evict_move_kernel(const PagedEvictArgs a)
{
    grid_dep_wait();
    grid_dep_launch();
    const int slice = blockIdx.x % a.slices;
    const int item = blockIdx.x / a.slices;
    const int g = item % a.kv.Hkv, b = item / a.kv.Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int2 c = a.counts[item];
    if (slice == 0 && g == 0 && threadIdx.x == 0) a.kv_len_out[b] = c.y;
    const int2 *mv = a.moves + (long long)item * a.max_moves;
    for (int i = slice * 8 + warp; i < c.x; i += a.slices * 8) {
        const int2 x = mv[i];
        const int ps = paged_page(a.kv, b, x.x), pd = paged_page(a.kv, b, x.y);
        if (ps < 0 || pd < 0) continue;
        const int mask = (1 << a.kv.shift) - 1;
        const long long src = (long long)ps * a.kv.nb3 + (long long)(x.x & mask) * a.kv.nb1 + (long long)g * a.kv.nb2;
        const long long dst = (long long)pd * a.kv.nb3 + (long long)(x.y & mask) * a.kv.nb1 + (long long)g * a.kv.nb2;
        if (a.vec == 16) {
            evict_copy_row<uint4>(a.kv.k + dst, a.kv.k + src, a.row_bytes / 16, lane);
            evict_copy_row<uint4>(a.kv.v + dst, a.kv.v + src, a.row_bytes / 16, lane);
        } else {
            evict_copy_row<uint32_t>(a.kv.k + dst, a.kv.k + src, a.row_bytes / 4, lane);
            evict_copy_row<uint32_t>(a.kv.v + dst, a.kv.v + src, a.row_bytes / 4, lane);
        }
    }
}

}  // namespace vtx
