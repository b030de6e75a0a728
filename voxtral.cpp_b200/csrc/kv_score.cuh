// kv_score.cuh — accumulated attention weight of a paged cache's rows.
//
//   out[g][j] = decay * in[g][j] + sum_{i, h in group g} 2^(x_hij - lse_hi)
//
// in log2 units, over the observed new tokens i that see row j.  The sum runs
// down a column of P, so nothing has to be carried between key tiles: a warp
// owns 32 keys, holds their K rows as the B fragments of mma.sync in registers
// for the whole call and walks the query rows 16 at a time, adding each tile's
// weights to one register per key; a shuffle over the row lanes at the end
// gives the sums in the same order on every run (no atomics).
// Few rows (a decode step): bound by reading K once.  Many rows: bound by the
// exponentials (one per query row and key) and mma.sync.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>
#include "vtx_ptx.cuh"
#include "paged_kv.cuh"
#include "fa_paged.cuh"

namespace vtx {

struct PagedScoreArgs {
    PagedView kv;
    const char *q; int q_f16; long long q_nbt, q_nbh;
    const float *lse;
    const float *score; float *score_out; int row_cap;
    float decay;
    int observe;
    int Hq, G;
    float scale, softcap;
    int causal, window;
};

// Grid (key tiles of 128, Hkv, n_seq), 4 warps of 32 keys.
template <int D, int KVT>
__global__ void __launch_bounds__(128)
kv_score_kernel(const PagedScoreArgs a)
{
    grid_dep_wait();
    grid_dep_launch();
    constexpr int NT = 4, KC = D / 16;
    const int b = blockIdx.z, g = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3;
    const PagedSeq s = paged_seq(a.kv, b);
    const int limit = min(s.len, a.row_cap);
    if (blockIdx.x == 0 && s.len > min(a.row_cap, a.kv.max_kv)) paged_report(a.kv, VTX_KERR_BOUND);
    const int k0 = blockIdx.x * 128 + warp * 32;
    if (k0 >= limit) return;

    // K rows of the warp's keys as B fragments.  The k index of the MMA is any
    // permutation of the head dim that Q shares: lane c of a quad takes dims
    // 32 i + 8 c ... + 7, one 16-byte load per row and 32 dims.  Q8_0: the
    // integers, and the scales of this lane's two columns of every block.
    uint32_t kb[NT][KC][2];
    float kd[NT][KVT == 8 ? D / 32 : 1][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int key = k0 + nt * 8 + (lane >> 2);
        const bool on = key < limit;
        const char *kr = a.kv.k + (on ? paged_row(a.kv, b, key, g) : 0);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const uint4 x = on ? paged_load8<KVT>(kr, 32 * i + 8 * c, 1.0f) : make_uint4(0u, 0u, 0u, 0u);
            kb[nt][2 * i][0] = x.x; kb[nt][2 * i][1] = x.y;
            kb[nt][2 * i + 1][0] = x.z; kb[nt][2 * i + 1][1] = x.w;
            if constexpr (KVT == 8) {
                const float d = on ? q8_scale(kr, 32 * i) : 0.f;
                kd[nt][i][0] = __shfl_sync(0xffffffffu, d, 8 * c);
                kd[nt][i][1] = __shfl_sync(0xffffffffu, d, 8 * c + 4);
            }
        }
    }
    float sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sum[nt][0] = sum[nt][1] = 0.f;

    const int off = s.len - s.n_new;
    int t0 = a.observe > 0 ? max(0, s.n_new - a.observe) : 0;
    if (a.causal) t0 = max(t0, k0 - off);                   // earlier tokens see none of these keys
    int t1 = s.n_new;
    if (a.window > 0) t1 = min(t1, k0 + 31 + a.window - off);   // nor do tokens past the window
    const int r_end = t1 * a.G;
    for (int r0 = t0 * a.G; r0 < r_end; r0 += 16) {
        int lo[2], hi[2];
        float ls[2];
        const char *qp[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = r0 + (lane >> 2) + 8 * u;
            const int tok = r / a.G, head = g * a.G + r % a.G;
            const bool on = r < r_end;
            hi[u] = on ? (a.causal ? min(off + tok, limit - 1) : limit - 1) : -1;
            lo[u] = a.window > 0 ? off + tok - a.window + 1 : 0;
            qp[u] = on ? a.q + (long long)(s.q0 + tok) * a.q_nbt + (long long)head * a.q_nbh : nullptr;
            const float x = on ? a.lse[(long long)(s.q0 + tok) * a.Hq + head] : INFINITY;
            ls[u] = x == -INFINITY ? INFINITY : x * kLog2e;
        }
        float x[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            uint32_t q[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) q[u][j] = qp[u] ? paged_q2(qp[u], a.q_f16, 32 * i + 8 * c + 2 * j) : 0u;
            const uint32_t a0[4] = {q[0][0], q[1][0], q[0][1], q[1][1]};
            const uint32_t a1[4] = {q[0][2], q[1][2], q[0][3], q[1][3]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if constexpr (KVT == 1) {
                    mma16816(x[nt], a0, kb[nt][2 * i][0], kb[nt][2 * i][1]);
                    mma16816(x[nt], a1, kb[nt][2 * i + 1][0], kb[nt][2 * i + 1][1]);
                } else {
                    float y[4] = {0.f, 0.f, 0.f, 0.f};
                    mma16816(y, a0, kb[nt][2 * i][0], kb[nt][2 * i][1]);
                    mma16816(y, a1, kb[nt][2 * i + 1][0], kb[nt][2 * i + 1][1]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[nt][j] = fmaf(kd[nt][i][j & 1], y[j], x[nt][j]);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int u = i >> 1, key = k0 + nt * 8 + 2 * c + (i & 1);
                const float p = ex2(paged_logit(x[nt][i], a.scale, a.softcap) - ls[u]);
                if (key >= lo[u] && key <= hi[u]) sum[nt][i & 1] += p;
            }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float x = sum[nt][i];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            const int key = k0 + nt * 8 + 2 * c + i;
            if (lane < 4 && key < limit) {
                const long long e = ((long long)b * a.kv.Hkv + g) * a.row_cap + key;
                a.score_out[e] = (a.decay != 0.f ? a.decay * a.score[e] : 0.f) + x;
            }
        }
}

}  // namespace vtx
