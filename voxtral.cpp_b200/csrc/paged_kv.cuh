// paged_kv.cuh — device view of a decoder cache kept in pages and of the
// ragged batch of new tokens over it (vtx_paged_kv), and the KV append into it.
//
// The reference keeps one cache buffer per context (src/voxtral.cpp:1126-1136);
// here row r of a stream is row r % page_size of the page its table names.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>
#include "vtx_ptx.cuh"
#include "kv_append.cuh"

namespace vtx {

// device error word values of the paged calls
enum { VTX_KERR_PAGE = 40, VTX_KERR_BOUND = 41 };

struct PagedView {
    char *k, *v;
    long long nb1, nb2, nb3;               // row, head and page strides (bytes), the same for k and v
    const int *table, *kv_len, *q_start;   // table NULL: stream s owns pages s * max_pages ...
    int n_seq, n_tokens, max_new, max_kv;
    int max_pages, n_pages, shift;         // page_size = 1 << shift
    int cap;                               // rows that a stream can have
    int Hkv;
    int *err;
};

// One stream: tokens q0 .. q0 + n_new of the packed arrays stand in rows off ..
// off + n_new - 1, and its table holds the rows below len.  off follows the kv_len
// as given, so a stream longer than its table keeps its tokens' rows: those at or
// behind len do not exist.
struct PagedSeq {
    int q0, n_new, len, off;
};

__device__ __forceinline__ void paged_report(const PagedView &kv, int code) {
    if (kv.err) atomicCAS(kv.err, 0, code);
}

__device__ __forceinline__ PagedSeq paged_seq(const PagedView &kv, int b) {
    PagedSeq s;
    const int a = kv.q_start[b], e = kv.q_start[b + 1], n = kv.kv_len[b];
    s.q0 = min(max(a, 0), kv.n_tokens);
    s.n_new = min(max(e, s.q0), kv.n_tokens) - s.q0;
    s.len = min(max(n, 0), kv.cap);
    s.off = max(n, 0) - s.n_new;
    if (s.len != n) paged_report(kv, VTX_KERR_BOUND);
    return s;
}

// The page of row `row` of stream b (row < its len); a table entry outside the
// pool is reported and answered with -1.
__device__ __forceinline__ int paged_page(const PagedView &kv, int b, int row) {
    const long long i = (long long)b * kv.max_pages + (row >> kv.shift);
    const int p = kv.table ? kv.table[i] : (int)i;
    if ((unsigned)p < (unsigned)kv.n_pages) return p;
    paged_report(kv, VTX_KERR_PAGE);
    return -1;
}

// Byte offset of a row of KV head g inside either pool, for reading: an entry
// outside the pool reads page 0.
__device__ __forceinline__ long long paged_row(const PagedView &kv, int b, int row, int g) {
    return (long long)max(paged_page(kv, b, row), 0) * kv.nb3 + (long long)(row & ((1 << kv.shift) - 1)) * kv.nb1 +
           (long long)g * kv.nb2;
}

// Stream of packed token t: the first whose tokens end behind t (n_seq: none).  A
// warp searches q_start 32 entries at a time; all lanes call it, `t` is uniform.
__device__ __forceinline__ int paged_find(const PagedView &kv, int t, int lane) {
    int lo = 0, hi = kv.n_seq;                              // the answer lies in [lo, hi]
    while (hi - lo > 32) {
        const int step = (hi - lo + 31) / 32, i = lo + lane * step;
        const int c = __popc(__ballot_sync(0xffffffffu, i < hi && kv.q_start[i + 1] <= t));
        hi = min(hi, lo + c * step);
        if (c > 0) lo += (c - 1) * step + 1;
    }
    const int i = lo + lane;
    return lo + __popc(__ballot_sync(0xffffffffu, i < hi && kv.q_start[i + 1] <= t));
}

// ---- append ---------------------------------------------------------------------

struct KvAppendPagedArgs {
    PagedView kv;
    int Hq, q8, qo_f16;
    const float *q; long long q_nb1;        // token strides in floats; heads contiguous
    const float *k; long long k_nb1;
    const float *v; long long v_nb1;
    void *q_out; long long qo_nb1;          // token stride in elements
    const int *positions;
    int *row_pos; float *score; int row_cap;
    int rows_per_cta;                       // of a token's Hq + 2 Hkv rows
    double turns[64];                       // base^(-2i/D) / (2 pi): turns per position of pair i
};

// A head row, 8 values per lane, as Q8_0 into 4-byte aligned `row`: the bytes of
// store_q8_lane in whole words.  A block is four lanes, two blocks are 17 words: the
// even block's values start 2 bytes in, so its words join two neighbours (the first
// takes the scale, the odd block's first lane closes it with its own scale); the odd
// block's values are aligned.  u: the lane's place in its row.
__device__ __forceinline__ void store_q8_words(const float (&x)[8], char *row, int u, bool put) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const float id = amax != 0.f ? 127.f / amax : 0.f;
    const uint32_t d = __half_as_ushort(__float2half_rn(amax / 127.f));
    uint32_t q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        q[i] = (uint32_t)(__float2int_rn(x[4 * i] * id) & 0xff) | (uint32_t)(__float2int_rn(x[4 * i + 1] * id) & 0xff) << 8 |
               (uint32_t)(__float2int_rn(x[4 * i + 2] * id) & 0xff) << 16 |
               (uint32_t)(__float2int_rn(x[4 * i + 3] * id) & 0xff) << 24;
    const uint32_t before = __shfl_up_sync(0xffffffffu, q[1], 1);
    if (!put) return;                                       // the shuffles want the whole warp
    const int j = u & 3;
    uint32_t *w = reinterpret_cast<uint32_t *>(row) + (u >> 3) * 17 + 2 * j;
    if (u & 4) {
        w[9] = q[0];
        w[10] = q[1];
        if (j == 0) w[8] = before >> 16 | d << 16;
    } else {
        w[0] = (j == 0 ? d : before >> 16) | q[0] << 16;
        w[1] = __funnelshift_r(q[0], q[1], 16);
    }
}

// 8 floats from 16-byte (W16) or 8-byte aligned memory.
template <bool W16>
__device__ __forceinline__ void load_f8(float (&x)[8], const float *p) {
    if constexpr (W16) {
        *reinterpret_cast<float4 *>(&x[0]) = *reinterpret_cast<const float4 *>(p);
        *reinterpret_cast<float4 *>(&x[4]) = *reinterpret_cast<const float4 *>(p + 4);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) *reinterpret_cast<float2 *>(&x[i]) = *reinterpret_cast<const float2 *>(p + i);
    }
}
template <bool W16>
__device__ __forceinline__ void store_8(void *dst, bool f16, const float (&x)[8]) {
    if (f16) {
        const uint4 h = make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]),
                                   pack_half2(x[6], x[7]));
        if constexpr (W16) {
            *static_cast<uint4 *>(dst) = h;
        } else {
            static_cast<uint2 *>(dst)[0] = make_uint2(h.x, h.y);
            static_cast<uint2 *>(dst)[1] = make_uint2(h.z, h.w);
        }
    } else if constexpr (W16) {
        static_cast<float4 *>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
        static_cast<float4 *>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) static_cast<float2 *>(dst)[i] = make_float2(x[2 * i], x[2 * i + 1]);
    }
}

// Grid (tokens, ceil((Hq + 2 Hkv) / rows_per_cta)), 8 warps; D / 8 lanes per row, 8
// values each, so a warp takes 2 (D = 128) or 4 rows at once.
// HBM-bound by its bytes: (Hq + 2 Hkv) * D * 4 read and Hq * D * (2 or 4) + 2 Hkv *
// row bytes written per token.  The way to a row's page (stream of the token, its
// lengths, the table) is three dependent trips to memory, so a warp loads its first
// rows before it takes them.  7639 tokens, 32 + 2 x 8 heads of 128: 50 us into F16
// pages (5.6 TB/s), 54 us into Q8_0 (4.9 TB/s); with a whole warp per row the
// instructions were the bound (5900 warp instructions per token, Q8_0 64 us).
// Angle of pair i: pos * turns[i] turns, reduced to (-1/2, 1/2] in double (three
// operations), then sincospi in float: an error of about 1e-7 at any position.
template <int D, bool W16>
__global__ void __launch_bounds__(256)
kv_append_paged_kernel(const __grid_constant__ KvAppendPagedArgs a)
{
    grid_dep_wait();
    grid_dep_launch();
    constexpr int LPR = D / 8, RPW = 32 / LPR, NR = 3;      // lanes per row, rows per warp, row sets in flight
    __shared__ float2 cs[D / 2];                            // (cos, sin) of pair i
    const int t = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, u = lane % LPR;
    const int r0 = blockIdx.y * a.rows_per_cta, r1 = min(r0 + a.rows_per_cta, a.Hq + 2 * a.kv.Hkv);
    const int first = r0 + warp * RPW + lane / LPR;         // this lane's rows: first, first + 8 RPW, ...
    float x[NR][8];
    // rows of a token: Q heads, then K heads, then V heads
    auto load = [&](int rb) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int r = rb + 8 * RPW * i;
            const float *src = r < a.Hq ? a.q + (long long)t * a.q_nb1 + (long long)r * D
                               : r < a.Hq + a.kv.Hkv ? a.k + (long long)t * a.k_nb1 + (long long)(r - a.Hq) * D
                               : a.v + (long long)t * a.v_nb1 + (long long)(r - a.Hq - a.kv.Hkv) * D;
            if (r < r1) load_f8<W16>(x[i], src + u * 8);
        }
    };
    load(first);
    const int pos = a.positions[t];
    if (r0 < a.Hq + a.kv.Hkv && threadIdx.x < D / 2) {      // some Q or K row here
        double y = (double)pos * a.turns[threadIdx.x];
        y -= rint(y);
        float s, c;
        sincospif(2.0f * (float)y, &s, &c);
        cs[threadIdx.x] = make_float2(c, s);
    }
    __syncthreads();
    const int b = paged_find(a.kv, t, lane);
    int row = -1;
    if (b < a.kv.n_seq) {
        const PagedSeq s = paged_seq(a.kv, b);
        if (t >= s.q0 && t < s.q0 + s.n_new) row = s.off + (t - s.q0);
        if (row >= s.len) row = -1;                         // behind the table: dropped (and reported)
        if (row >= 0 && row >= a.row_cap && (a.row_pos || a.score)) {
            paged_report(a.kv, VTX_KERR_BOUND);
            row = -1;
        }
    }
    const int page = row >= 0 ? paged_page(a.kv, b, row) : -1;
    const long long at = (long long)page * a.kv.nb3 + (long long)(row & ((1 << a.kv.shift) - 1)) * a.kv.nb1;
    for (int rb = first; rb - lane / LPR < r1; rb += 8 * RPW * NR) {     // uniform within the warp
        if (rb != first) load(rb);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int r = rb + 8 * RPW * i;
            if (r < a.Hq + a.kv.Hkv) {
#pragma unroll
                for (int j = 0; j < 4; ++j) rope_pair(x[i][2 * j], x[i][2 * j + 1], cs[u * 4 + j]);
            }
            const bool is_k = r < a.Hq + a.kv.Hkv;
            const int h = r - a.Hq - (is_k ? 0 : a.kv.Hkv);
            char *dst = (is_k ? a.kv.k : a.kv.v) + at + (long long)h * a.kv.nb2;
            const bool put = r >= a.Hq && r < r1 && page >= 0;
            if (r < a.Hq && r < r1)
                store_8<W16>(static_cast<char *>(a.q_out) + ((long long)t * a.qo_nb1 + (long long)r * D + u * 8) *
                                                                (a.qo_f16 ? 2 : 4), a.qo_f16, x[i]);
            if (put && is_k && u == 0) {                    // the row starts without weight
                const long long e = ((long long)b * a.kv.Hkv + h) * a.row_cap + row;
                if (a.row_pos) a.row_pos[e] = pos;
                if (a.score) a.score[e] = 0.0f;
            }
            if (a.q8) {
                if (__any_sync(0xffffffffu, put)) store_q8_words(x[i], dst, u, put);
            } else if (put) {
                store_8<true>(dst + u * 16, true, x[i]);    // pool rows are 16-byte aligned
            }
        }
    }
}

}  // namespace vtx
