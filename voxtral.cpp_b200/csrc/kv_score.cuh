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
// Three kernels.  Few query rows per KV head (a decode step): bound by reading K
// once, kv_score_stream_kernel.  Many rows: bound by the exponentials (one per
// query row and key), kv_score_sm100_kernel.  Many rows with an F32 q, which TMA
// cannot round: kv_score_kernel, the description above.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>
#include "vtx_ptx.cuh"
#include "paged_kv.cuh"
#include "fa_paged.cuh"
#include "fa_paged_decode.cuh"

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

    const int off = s.off;
    int t0 = a.observe > 0 ? max(0, s.n_new - a.observe) : 0;
    const int lo_any = t0 < s.n_new ? (a.window > 0 ? off + t0 - a.window + 1 : 0) : limit;   // nobody sees keys below

    // K rows of the warp's keys as B fragments.  The k index of the MMA is any
    // permutation of the head dim that Q shares: lane c of a quad takes dims
    // 32 i + 8 c ... + 7, one 16-byte load per row and 32 dims.  Q8_0: the
    // integers, and the scales of this lane's two columns of every block.
    uint32_t kb[NT][KC][2];
    float kd[NT][KVT == 8 ? D / 32 : 1][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int key = k0 + nt * 8 + (lane >> 2);
        const bool on = key < limit && key >= lo_any;
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

// Streams with at most 16 query rows per KV head: the K half of the streaming
// attention kernel.  A CTA per (stream, KV head, key split), its 4 warps take
// tiles of 16 keys in turn through private rings of bulk copies; a tile's
// weights are summed over a quad's rows by shuffles and added to the old score,
// which was loaded before the wait for the tile.
template <int D, int KVT> struct ScoreStreamCfg {
    using P = PagedDecodeCfg<D, KVT>;
    static constexpr int STAGES = KVT == 1 ? 2 : 4;
    static constexpr int STAGE_BYTES = 16 * P::PITCH;
    static constexpr int WARP_BYTES = STAGES * STAGE_BYTES;
    static constexpr int BAR_OFF = 4 * WARP_BYTES;
    static constexpr int SMEM = BAR_OFF + 4 * STAGES * 8;
};

template <int D, int KVT, int ROWS, bool UF>
__global__ void __launch_bounds__(128)
kv_score_stream_kernel(const PagedScoreArgs a, const PagedSplit sp)
{
    grid_dep_wait();
    grid_dep_launch();
    using P = PagedDecodeCfg<D, KVT>;
    using C = ScoreStreamCfg<D, KVT>;
    constexpr int KC = D / 16, NC = ROWS / 8;
    extern __shared__ __align__(128) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3;
    char *ring = smem + warp * C::WARP_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::BAR_OFF) + warp * C::STAGES;
    const int g = blockIdx.x % a.kv.Hkv;
    const int split = (blockIdx.x / a.kv.Hkv) % sp.n_splits;
    const int b = blockIdx.x / (a.kv.Hkv * sp.n_splits);
    PagedSeq s = paged_seq(a.kv, b);
    if (threadIdx.x == 0 && split == 0 && (s.len > min(a.row_cap, a.kv.max_kv) || s.n_new > a.kv.max_new))
        paged_report(a.kv, VTX_KERR_BOUND);
    const int limit = min(s.len, a.row_cap);
    const int off = s.off;
    const int t0 = max(s.n_new - a.kv.max_new, a.observe > 0 ? max(0, s.n_new - a.observe) : 0);
    const int rows = (s.n_new - t0) * a.G;
    const int lo_any = rows == 0 ? limit : (a.window > 0 ? max(0, off + t0 - a.window + 1) : 0);
    const PagedCut cut = paged_cut(PagedSeq{s.q0, s.n_new, limit, off}, 0, 0, sp);
    if (split >= cut.n) return;
    const int t_end = min(cut.per * (split + 1), cut.nt);
    const int first = cut.per * split + warp;
    const int nt = t_end > first ? (t_end - first + 3) / 4 : 0;

    if (lane < C::STAGES) mbar_init(&full[lane], 1);
    __syncwarp();
    fence_mbar_init();
    __syncwarp();
    const char *kp = a.kv.k + (long long)g * a.kv.nb2;
    int pages = 0;
    auto issue = [&](int t) {
        if ((t & 31) == 0) {
            const int k = 16 * (first + (t + lane) * 4);
            pages = t + lane < nt && k + 16 > lo_any ? max(paged_page(a.kv, b, k), 0) : 0;
        }
        const int pg = __shfl_sync(0xffffffffu, pages, t & 31);
        const int k0 = 16 * (first + t * 4);
        if (t >= nt || k0 + 16 <= lo_any) return;               // nobody sees this tile: not read
        char *st = ring + (t % C::STAGES) * C::STAGE_BYTES;
        uint64_t *bar = &full[t % C::STAGES];
        const long long at = (long long)pg * a.kv.nb3 + (long long)(k0 & ((1 << a.kv.shift) - 1)) * a.kv.nb1;
        fence_proxy_async_smem();
        if (lane == 0) mbar_arrive_expect_tx(bar, 16 * P::ROW);
        __syncwarp();
        if constexpr (KVT == 1) {                               // rows behind kv_len are masked, whatever they hold
            if (lane < 16) bulk_g2s(st + lane * P::PITCH, kp + at + (long long)lane * a.kv.nb1, P::ROW, bar);
        } else {
            if (lane == 0) bulk_g2s(st, kp + at, 16 * P::ROW, bar);
        }
    };
#pragma unroll
    for (int t = 0; t < C::STAGES; ++t) issue(t);

    // Q fragments of the lane's column, limits and lse of the rows 8 nc + 2c + j that
    // its scores belong to
    uint32_t qb[NC][KC][2];
    int lo[NC][2], hi[NC][2];
    float ls[NC][2];
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
        const int r = 8 * nc + (lane >> 2);
        const bool on = r < rows;
        const char *qp = a.q + (long long)(s.q0 + t0 + (on ? r / a.G : 0)) * a.q_nbt +
                         (long long)(g * a.G + (on ? r % a.G : 0)) * a.q_nbh;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            const int d = paged_q_dim<KVT>(lane, kc);
            qb[nc][kc][0] = on ? paged_q2(qp, a.q_f16, d) : 0u;
            qb[nc][kc][1] = on ? paged_q2(qp, a.q_f16, d + (KVT == 1 ? 8 : 2)) : 0u;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r2 = 8 * nc + 2 * c + i;
            const bool on2 = r2 < rows;
            const int tok = t0 + (on2 ? r2 / a.G : 0), head = g * a.G + (on2 ? r2 % a.G : 0);
            hi[nc][i] = on2 ? (a.causal ? min(off + tok, limit - 1) : limit - 1) : -1;
            lo[nc][i] = a.window > 0 ? off + tok - a.window + 1 : 0;
            const float x = on2 ? a.lse[(long long)(s.q0 + tok) * a.Hq + head] : INFINITY;
            ls[nc][i] = x == -INFINITY ? INFINITY : x * kLog2e;
        }
    }
    // lanes c = 0, 1 end up with the sums of their two keys
    const int mine = paged_tile_key<KVT>(lane, c & 1);
    const long long base = ((long long)b * a.kv.Hkv + g) * a.row_cap;
    // tiles nobody sees come first and use no stage
    const int skip = min(nt, (lo_any >> 4) > first ? ((lo_any >> 4) - 1 - first) / 4 + 1 : 0);
    const float cx = a.scale * kLog2e;
    const int hi_all = a.causal ? off + t0 : limit - 1;        // every token sees [lo_all, hi_all]
    const int lo_all = a.window > 0 ? off + s.n_new - a.window : 0;
    // old scores of the next four tiles: their latency is a tile's whole time
    auto old_of = [&](int t) {
        const int key = 16 * (first + t * 4) + mine;
        return t < nt && c < 2 && key < limit && a.decay != 0.f ? a.decay * a.score[base + key] : 0.f;
    };
    constexpr int U = 4;
    float old[U];
#pragma unroll
    for (int i = 0; i < U; ++i) old[i] = old_of(i);
    bool ok = true;
    int done = 0;
    for (int tb = 0; tb < nt && ok; tb += U) {
#pragma unroll
        for (int ui = 0; ui < U; ++ui) {
            const int t = tb + ui;
            if (t >= nt || !ok) break;
            const int k0 = 16 * (first + t * 4), key = k0 + mine;
            const bool inner = k0 >= lo_all && k0 + 15 <= hi_all;
            float sum = 0.f;
            if (t >= skip) {
                ok = __all_sync(0xffffffffu,
                                mbar_wait(&full[t % C::STAGES], ((t - skip) / C::STAGES) & 1, a.kv.err, VTX_KERR_KV));
                if (!ok) break;
                float x[NC][4], w[2] = {0.f, 0.f};
                paged_tile_scores<D, KVT, NC>(ring + (t % C::STAGES) * C::STAGE_BYTES, qb, x, lane);
#pragma unroll
                for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k = k0 + paged_tile_key<KVT>(lane, i >> 1);
                        const float p = ex2(paged_logit_t<UF>(x[nc][i], cx, a.scale, a.softcap) - ls[nc][i & 1]);
                        w[i >> 1] += inner || (k >= lo[nc][i & 1] && k <= hi[nc][i & 1]) ? p : 0.f;
                    }
                // over the lanes of the quad; lane c keeps key c & 1
                sum = (c & 1 ? w[1] : w[0]) + __shfl_xor_sync(0xffffffffu, c & 1 ? w[0] : w[1], 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                __syncwarp();
            }
            if (c < 2 && key < limit) a.score_out[base + key] = old[ui] + sum;
            old[ui] = old_of(t + U);
            issue(t + C::STAGES);
            done = t + 1;
        }
    }
    for (int t = max(done, skip); t < min(nt, done + C::STAGES); ++t)   // after a failed wait: copies must land
        mbar_wait(&full[t % C::STAGES], ((t - skip) / C::STAGES) & 1, nullptr, 0);
}

}  // namespace vtx
