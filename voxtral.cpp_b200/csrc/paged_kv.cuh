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
    int Hkv;
    int *err;
};

// One stream's lengths, cut to what the arrays hold: tokens q0 .. q0 + n_new
// of the packed arrays stand in rows len - n_new .. len - 1.
struct PagedSeq {
    int q0, n_new, len;
};

__device__ __forceinline__ void paged_report(const PagedView &kv, int code) {
    if (kv.err) atomicCAS(kv.err, 0, code);
}

__device__ __forceinline__ PagedSeq paged_seq(const PagedView &kv, int b) {
    PagedSeq s;
    const int a = kv.q_start[b], e = kv.q_start[b + 1], n = kv.kv_len[b];
    s.q0 = min(max(a, 0), kv.n_tokens);
    s.n_new = min(max(e, s.q0), kv.n_tokens) - s.q0;
    const long long cap = (long long)kv.max_pages << kv.shift;
    s.len = (int)min((long long)max(n, 0), cap);
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

// Stream of packed token t (the last one whose q_start is <= t and that has
// tokens): every thread of the CTA counts a share of the streams.  The CTA's
// threads all call it; `t` is uniform.
__device__ __forceinline__ int paged_find(const PagedView &kv, int t) {
    int n = 0;
    for (int i0 = 0; i0 < kv.n_seq; i0 += blockDim.x) {
        const int i = i0 + (int)threadIdx.x;
        n += __syncthreads_count(i < kv.n_seq && kv.q_start[i + 1] <= t);
    }
    return n;                               // n_seq when no stream holds t
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

// Grid (tokens, ceil((Hq + 2 Hkv) / rows_per_cta)), 8 warps, a warp per row,
// as kv_append_kernel.  HBM-bound: (Hq + 2 Hkv) * D * 4 bytes read and
// Hq * D * (2 or 4) + 2 Hkv * row bytes written per token.
// Angle of pair i: pos * turns[i] turns, reduced to (-1/2, 1/2] in double (three
// operations), then sincospi in float: an error of about 1e-7 at any position.
template <int D>
__global__ void __launch_bounds__(256)
kv_append_paged_kernel(const __grid_constant__ KvAppendPagedArgs a)
{
    grid_dep_wait();
    grid_dep_launch();
    constexpr int E = D / 32;                               // elements per lane
    __shared__ float2 cs[D / 2];                            // (cos, sin) of pair i
    const int t = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nwarps = blockDim.x >> 5, r0 = blockIdx.y * a.rows_per_cta;
    const int pos = a.positions[t];
    if (r0 < a.Hq + a.kv.Hkv && threadIdx.x < D / 2) {      // some Q or K row here
        double x = (double)pos * a.turns[threadIdx.x];
        x -= rint(x);
        float s, c;
        sincospif(2.0f * (float)x, &s, &c);
        cs[threadIdx.x] = make_float2(c, s);
    }
    const int b = paged_find(a.kv, t);                      // also orders the table
    __syncthreads();
    int row = -1;
    if (b < a.kv.n_seq) {
        const PagedSeq s = paged_seq(a.kv, b);
        if (t >= s.q0 && t < s.q0 + s.n_new) row = s.len - s.n_new + (t - s.q0);
        if (row >= 0 && row >= a.row_cap && (a.row_pos || a.score)) {
            paged_report(a.kv, VTX_KERR_BOUND);
            row = -1;
        }
    }
    const int page = row >= 0 ? paged_page(a.kv, b, row) : -1;
    const long long at = (long long)page * a.kv.nb3 + (long long)(row & ((1 << a.kv.shift) - 1)) * a.kv.nb1;
    const int per_tok = a.Hq + 2 * a.kv.Hkv;
    for (int r = r0 + warp; r < min(r0 + a.rows_per_cta, per_tok); r += nwarps) {
        const int kind = r < a.Hq ? 0 : (r < a.Hq + a.kv.Hkv ? 1 : 2);   // Q, K, V
        const int h = kind == 0 ? r : (kind == 1 ? r - a.Hq : r - a.Hq - a.kv.Hkv);
        const float *src = kind == 0 ? a.q + (long long)t * a.q_nb1
                                     : (kind == 1 ? a.k + (long long)t * a.k_nb1 : a.v + (long long)t * a.v_nb1);
        src += (long long)h * D + lane * E;
        float x[E];
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const float2 p = *reinterpret_cast<const float2 *>(src + i);
            x[i] = p.x;
            x[i + 1] = p.y;
        }
        if (kind != 2) {
#pragma unroll
            for (int j = 0; j < E / 2; ++j) rope_pair(x[2 * j], x[2 * j + 1], cs[lane * E / 2 + j]);
        }
        if (kind == 0) {
            const long long o = (long long)t * a.qo_nb1 + (long long)h * D + lane * E;
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                if (a.qo_f16)
                    *reinterpret_cast<__half2 *>(static_cast<__half *>(a.q_out) + o + i) =
                        __floats2half2_rn(x[i], x[i + 1]);
                else
                    *reinterpret_cast<float2 *>(static_cast<float *>(a.q_out) + o + i) = make_float2(x[i], x[i + 1]);
            }
            continue;
        }
        if (page < 0) continue;
        if (kind == 1 && lane == 0) {                       // the row starts without weight
            const long long e = ((long long)b * a.kv.Hkv + h) * a.row_cap + row;
            if (a.row_pos) a.row_pos[e] = pos;
            if (a.score) a.score[e] = 0.0f;
        }
        char *dst = (kind == 1 ? a.kv.k : a.kv.v) + at + (long long)h * a.kv.nb2;
        if (a.q8) {
            store_q8_lane<E>(x, dst, lane);
        } else {
#pragma unroll
            for (int i = 0; i < E; i += 2)
                *reinterpret_cast<__half2 *>(reinterpret_cast<__half *>(dst) + lane * E + i) =
                    __floats2half2_rn(x[i], x[i + 1]);
        }
    }
}

}  // namespace vtx
