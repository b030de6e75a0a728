// fa_paged_decode.cuh — HBM-streaming attention of a few new tokens per stream
// over a paged cache (decode steps, short drafts): the decode node of
// src/voxtral.cpp:1802 for streams that bring at most 16 / G tokens.
//
// Every K and V row is read once and does 4 flops a byte per query row, so the
// call is bound by HBM.  One CTA per (stream, KV head, key split); its 4 warps
// take tiles of 16 keys in turn, each through a private ring of bulk copies
// (no CTA barrier in the loop), 16-key tiles never cross a page.  The n * G
// query rows (token * G + head of the group) are the M operand of mma.sync
// m16n8k16: S = Q K^T, then the S fragment becomes the A fragment of O += P V.
//   F16:  a lane copies one K or V row into a 16-byte padded pitch; ldmatrix.
//   Q8_0: the 16 rows of a tile are one contiguous block, copied as such.  K's
//         integers become halves exactly (0x64xx, minus 1152) and every block of
//         32 dims gets its scale in f32, so scores carry no rounding of K.  V's
//         integers are exact too: the scale of (row, block) multiplies P before P
//         is rounded to half, so P V has the one rounding that F16 has.  P stays
//         below 2^6 there, which bounds |scale| by 1023.  The k index of an MMA
//         may be any permutation: the lanes' words are chosen free of bank
//         conflicts (keys 2n + tile, words c and c + 4 of a block).
// Softmax in log2 units with a lazily moved reference m: O is rescaled only
// when the running maximum passes it by 2^8 (2^6).  The warps' (m, l, O) are
// merged in shared memory; with several splits every CTA leaves its result in the
// workspace, and the one that arrives last at the (stream, KV head)'s counter
// merges them in split order.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>
#include "vtx_ptx.cuh"
#include "paged_kv.cuh"
#include "fa_paged.cuh"

namespace vtx {

struct PagedSplit {
    int n_splits;             // splits of a stream's keys at most
    int tiles;                // 16-key tiles per split at least
    float *part_o, *part_ml;  // [n_seq][Hkv][n_splits][ROWS][D], ... [2] (m, l)
    unsigned *arrived;        // [n_seq][Hkv], zero between calls
    int beside;               // runs beside the kernel launched just before (see the kernel)
};

template <int D, int KVT> struct PagedDecodeCfg {
    static constexpr int KEYS = 16, WARPS = 4;
    static constexpr int ROW = KVT == 1 ? D * 2 : D / 32 * 34;
    static constexpr int PITCH = KVT == 1 ? ROW + 16 : ROW;
    static constexpr int STAGES = KVT == 1 ? 2 : 4;
    static constexpr int STAGE_BYTES = 2 * KEYS * PITCH;
    // the ring, reused for the warp's 16 x D floats at the end
    static constexpr int WARP_BYTES = STAGES * STAGE_BYTES > 16 * D * 4 ? STAGES * STAGE_BYTES : 16 * D * 4;
    static constexpr int BAR_OFF = WARPS * WARP_BYTES;
    static constexpr int ML_OFF = BAR_OFF + WARPS * STAGES * 8;
    static constexpr int SMEM = ML_OFF + WARPS * 16 * 8 + 16;
};

// How a stream's keys are cut: `lo` its first needed tile's row, nt tiles of 16
// keys from there, `per` tiles a split, n splits.
struct PagedCut {
    int lo, nt, per, n;
};
__device__ __forceinline__ PagedCut paged_cut(const PagedSeq &s, int causal, int window, const PagedSplit &sp) {
    PagedCut c;
    c.lo = window > 0 && causal ? max(0, s.len - s.n_new - window + 1) & ~15 : 0;
    c.nt = max(0, s.len - c.lo + 15) >> 4;
    c.per = max(sp.tiles, (c.nt + sp.n_splits - 1) / sp.n_splits);
    c.n = max(1, (c.nt + c.per - 1) / c.per);
    return c;
}

// The word at a byte offset of 2 mod 4 (HALF) or 0 mod 4 in shared memory.
template <bool HALF>
__device__ __forceinline__ uint32_t lds_word(const char *p) {
    if (!HALF) return *reinterpret_cast<const uint32_t *>(p);
    const uint32_t *w = reinterpret_cast<const uint32_t *>(p - 2);
    return __funnelshift_r(w[0], w[1], 16);
}
__device__ __forceinline__ float lds_half(const char *p) { return __half2float(*reinterpret_cast<const __half *>(p)); }

// S of 16 keys: x[nt] = columns of key tile nt (F16: keys 8 nt + col, Q8_0:
// keys 2 col + nt).
template <int D, int KVT>
__device__ __forceinline__ void paged_tile_scores(const char *ks, const uint32_t (&qa)[D / 16][4], float (&x)[2][4],
                                                  int lane)
{
    using C = PagedDecodeCfg<D, KVT>;
    constexpr int KC = D / 16;
    const int c = lane & 3, n = lane >> 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[0][i] = x[1][i] = 0.f;
    if constexpr (KVT == 1) {
        const int lrow = lane & 7, lmat = lane >> 3;
        float y[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[0][i] = y[1][i] = 0.f;
#pragma unroll
        for (int kc = 0; kc < KC; kc += 2) {
            uint32_t b0[4], b1[4];
            ldsm_x4(b0, ks + lrow * C::PITCH + (kc * 16 + lmat * 8) * 2);
            ldsm_x4(b1, ks + (8 + lrow) * C::PITCH + (kc * 16 + lmat * 8) * 2);
            mma16816(x[0], qa[kc], b0[0], b0[1]);
            mma16816(x[1], qa[kc], b1[0], b1[1]);
            mma16816(y[0], qa[kc + 1], b0[2], b0[3]);
            mma16816(y[1], qa[kc + 1], b1[2], b1[3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[0][i] += y[0][i];
            x[1][i] += y[1][i];
        }
    } else {
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                const char *p = ks + (2 * n + nt) * C::ROW + 34 * b + 2 + 4 * c;
                uint32_t w0, w1, k0, k1, k2, k3;
                if (b & 1) { w0 = lds_word<false>(p); w1 = lds_word<false>(p + 16); }
                else { w0 = lds_word<true>(p); w1 = lds_word<true>(p + 16); }
                q8_halves(w0, k0, k1);
                q8_halves(w1, k2, k3);
                float y[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816(y, qa[2 * b], k0, k1);
                mma16816(y, qa[2 * b + 1], k2, k3);
                const float d0 = lds_half(ks + (4 * c + nt) * C::ROW + 34 * b);
                const float d1 = lds_half(ks + (4 * c + 2 + nt) * C::ROW + 34 * b);
                x[nt][0] = fmaf(d0, y[0], x[nt][0]);
                x[nt][1] = fmaf(d1, y[1], x[nt][1]);
                x[nt][2] = fmaf(d0, y[2], x[nt][2]);
                x[nt][3] = fmaf(d1, y[3], x[nt][3]);
            }
        }
    }
}

// O += P V of 16 keys.  n0, n1: rows of the tile outside [n0, n1) hold anything
// (Q8_0: their scale is taken as 0; F16: the loader zeroed them).
template <int D, int KVT, int ROWS>
__device__ __forceinline__ void paged_tile_pv(const char *vs, const float (&p)[2][4], int n0, int n1,
                                              float (&o)[D / 8][4], int lane)
{
    using C = PagedDecodeCfg<D, KVT>;
    const int c = lane & 3;
    if constexpr (KVT == 1) {
        const int lrow = lane & 7, lmat = lane >> 3;
        const uint32_t pa[4] = {pack_half2(p[0][0], p[0][1]), ROWS > 8 ? pack_half2(p[0][2], p[0][3]) : 0u,
                                pack_half2(p[1][0], p[1][1]), ROWS > 8 ? pack_half2(p[1][2], p[1][3]) : 0u};
#pragma unroll
        for (int nb = 0; nb < D / 8; nb += 2) {
            uint32_t bv[4];
            ldsm_x4_t(bv, vs + ((lmat & 1) * 8 + lrow) * C::PITCH + (nb * 8 + (lmat >> 1) * 8) * 2);
            mma16816(o[nb], pa, bv[0], bv[1]);
            mma16816(o[nb + 1], pa, bv[2], bv[3]);
        }
    } else {
        const int n = lane >> 2;
        const char *v0 = vs + 4 * c * C::ROW;                   // this lane's keys 4c ... 4c + 3
        const bool all = n0 <= 0 && n1 >= 16;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            float d[4];
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                d[j] = lds_half(v0 + j * C::ROW + 34 * b);
                if (!all && (4 * c + j < n0 || 4 * c + j >= n1)) d[j] = 0.f;
                const char *q = v0 + j * C::ROW + 34 * b + 2 + 4 * n;
                w[j] = (b & 1) ? lds_word<false>(q) : lds_word<true>(q);
            }
            const uint32_t pa[4] = {pack_half2(p[0][0] * d[0], p[0][1] * d[2]),
                                    ROWS > 8 ? pack_half2(p[0][2] * d[0], p[0][3] * d[2]) : 0u,
                                    pack_half2(p[1][0] * d[1], p[1][1] * d[3]),
                                    ROWS > 8 ? pack_half2(p[1][2] * d[1], p[1][3] * d[3]) : 0u};
            uint32_t x[4], y[4];                                // dims 4n + i of keys (4c, 4c+2) and (4c+1, 4c+3)
            q8_halves(__byte_perm(w[0], w[2], 0x5140), x[0], x[1]);
            q8_halves(__byte_perm(w[0], w[2], 0x7362), x[2], x[3]);
            q8_halves(__byte_perm(w[1], w[3], 0x5140), y[0], y[1]);
            q8_halves(__byte_perm(w[1], w[3], 0x7362), y[2], y[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) mma16816(o[4 * b + i], pa, x[i], y[i]);
        }
    }
}

// The head dim of o[nb][j] in lane quad position c (j = 0, 1).
template <int KVT>
__device__ __forceinline__ int paged_o_dim(int nb, int j, int c) {
    return KVT == 1 ? nb * 8 + 2 * c + j : (nb >> 2) * 32 + 8 * c + 4 * j + (nb & 3);
}

// Normalises and writes 4 columns of query row r, and its lse with column 0.
template <int D>
__device__ __forceinline__ void paged_finish(const PagedAttnArgs &a, const PagedSeq &s, int g, int r, int d, float4 acc,
                                             float m, float l)
{
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int tok = s.q0 + r / a.G, head = g * a.G + r % a.G;
    paged_store2(a, tok, head, d, acc.x * inv, acc.y * inv);
    paged_store2(a, tok, head, d + 2, acc.z * inv, acc.w * inv);
    if (a.lse && d == 0) a.lse[(long long)tok * a.Hq + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <int D, int KVT, int ROWS, bool UF>
__device__ __forceinline__ void paged_decode_cta(const PagedAttnArgs &a, const PagedSplit &sp)
{
    using C = PagedDecodeCfg<D, KVT>;
    constexpr int KC = D / 16, NB = D / 8;
    extern __shared__ __align__(128) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3;
    char *ring = smem + warp * C::WARP_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::BAR_OFF) + warp * C::STAGES;
    const int g = blockIdx.x % a.kv.Hkv;
    const int split = (blockIdx.x / a.kv.Hkv) % sp.n_splits;
    const int b = blockIdx.x / (a.kv.Hkv * sp.n_splits);
    const PagedSeq s = paged_seq(a.kv, b);
    const int rows = s.n_new * a.G;
    if (s.n_new > a.kv.max_new && threadIdx.x == 0) paged_report(a.kv, VTX_KERR_BOUND);
    if (rows == 0 || rows > ROWS) return;
    const PagedCut cut = paged_cut(s, a.causal, a.window, sp);
    if (split >= cut.n) return;
    const int t_end = min(cut.per * (split + 1), cut.nt);
    const int first = cut.per * split + warp;                   // this warp's tiles: first, first + WARPS, ...
    const int nt = t_end > first ? (t_end - first + C::WARPS - 1) / C::WARPS : 0;
    const int off = s.len - s.n_new;
    const int lo_any = a.window > 0 ? max(0, off - a.window + 1) : 0;   // rows that some token sees

    if (lane < C::STAGES) mbar_init(&full[lane], 1);
    __syncwarp();
    fence_mbar_init();
    __syncwarp();
    const char *kp = a.kv.k + (long long)g * a.kv.nb2, *vp = a.kv.v + (long long)g * a.kv.nb2;
    int pages = 0;                                              // lane l: page of tile 32 (t / 32) + l
    auto issue = [&](int t) {
        if ((t & 31) == 0) {
            const int u = t + lane;
            pages = u < nt ? max(paged_page(a.kv, b, cut.lo + 16 * (first + u * C::WARPS)), 0) : 0;
        }
        const int pg = __shfl_sync(0xffffffffu, pages, t & 31);
        if (t >= nt) return;
        char *st = ring + (t % C::STAGES) * C::STAGE_BYTES;
        uint64_t *bar = &full[t % C::STAGES];
        const int k0 = cut.lo + 16 * (first + t * C::WARPS);
        const long long at = (long long)pg * a.kv.nb3 + (long long)(k0 & ((1 << a.kv.shift) - 1)) * a.kv.nb1;
        fence_proxy_async_smem();                               // our reads of this stage come first
        if constexpr (KVT == 1) {
            const int r = lane & 15, n0 = lo_any - k0, n1 = min(16, s.len - k0);
            if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(2 * (n1 - max(n0, 0)) * C::ROW));
            __syncwarp();
            char *dst = st + lane * C::PITCH;                   // K rows, then V rows
            if (r < n0 || r >= n1) {                            // rows no token sees may hold anything: zeros
#pragma unroll
                for (int i = 0; i < C::ROW / 16; ++i) reinterpret_cast<uint4 *>(dst)[i] = make_uint4(0u, 0u, 0u, 0u);
            } else {
                bulk_g2s(dst, (lane < 16 ? kp : vp) + at + (long long)r * a.kv.nb1, C::ROW, bar);
            }
            __syncwarp();
        } else {
            if (lane == 0) mbar_arrive_expect_tx(bar, 2 * C::KEYS * C::ROW);
            __syncwarp();
            if (lane < 2) bulk_g2s(st + lane * C::KEYS * C::ROW, (lane ? vp : kp) + at, C::KEYS * C::ROW, bar);
        }
    };
#pragma unroll
    for (int t = 0; t < C::STAGES; ++t) issue(t);

    uint32_t qa[KC][4];
    int lo[2], hi[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = (lane >> 2) + 8 * u;
        const bool on = r < rows && (u == 0 || ROWS > 8);
        const int tok = on ? r / a.G : 0;
        hi[u] = on ? (a.causal ? off + tok : s.len - 1) : -1;
        lo[u] = a.window > 0 ? off + tok - a.window + 1 : 0;
        const char *qp = a.q + (long long)(s.q0 + tok) * a.q_nbt + (long long)(g * a.G + (on ? r % a.G : 0)) * a.q_nbh;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            // F16: dims 16 kc + 2c and + 8; Q8_0: dims 32 b + 16 (kc odd) + 4c and + 2
            const int d = KVT == 1 ? kc * 16 + 2 * c : (kc >> 1) * 32 + (kc & 1) * 16 + 4 * c;
            qa[kc][u] = on ? paged_q2(qp, a.q_f16, d) : 0u;
            qa[kc][2 + u] = on ? paged_q2(qp, a.q_f16, d + (KVT == 1 ? 8 : 2)) : 0u;
        }
    }
    const int hi_all = a.causal ? off : s.len - 1;              // every token sees [lo_all, hi_all]
    const int lo_all = a.window > 0 ? off + s.n_new - a.window : 0;

    float o[NB][4];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const float cx = a.scale * kLog2e;
    constexpr float kJump = KVT == 1 ? 8.0f : 6.0f, kBack = KVT == 1 ? 0.0f : 4.0f;
    bool ok = true;
    int done = 0;
    for (int t = 0; t < nt; ++t) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full[t % C::STAGES], (t / C::STAGES) & 1, a.kv.err, VTX_KERR_KV));
        if (!ok) break;
        const char *ks = ring + (t % C::STAGES) * C::STAGE_BYTES, *vs = ks + C::KEYS * C::PITCH;
        const int k0 = cut.lo + 16 * (first + t * C::WARPS);
        float x[2][4];
        paged_tile_scores<D, KVT>(ks, qa, x, lane);
        const bool inner = k0 >= lo_all && k0 + 15 <= hi_all;
#pragma unroll
        for (int u = 0; u < (ROWS > 8 ? 2 : 1); ++u) {
            float mx = -INFINITY;
#pragma unroll
            for (int nt2 = 0; nt2 < 2; ++nt2)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float &y = x[nt2][2 * u + j];
                    y = paged_logit_t<UF>(y, cx, a.scale, a.softcap);
                    if (!inner) {
                        const int key = k0 + (KVT == 1 ? 8 * nt2 + 2 * c + j : 4 * c + 2 * j + nt2);
                        y = key < lo[u] || key > hi[u] ? -INFINITY : y;
                    }
                    mx = fmaxf(mx, y);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (mx > m[u] + kJump) {                            // uniform within the quad
                const float al = ex2(m[u] - (mx - kBack));
                m[u] = mx - kBack;
                l[u] *= al;
#pragma unroll
                for (int i = 0; i < NB; ++i) { o[i][2 * u] *= al; o[i][2 * u + 1] *= al; }
            }
            const float mu = m[u] == -INFINITY ? 0.f : m[u];
#pragma unroll
            for (int nt2 = 0; nt2 < 2; ++nt2)
#pragma unroll
                for (int j = 0; j < 2; ++j) x[nt2][2 * u + j] = ex2(x[nt2][2 * u + j] - mu);
            l[u] += (x[0][2 * u] + x[0][2 * u + 1]) + (x[1][2 * u] + x[1][2 * u + 1]);
        }
        paged_tile_pv<D, KVT, ROWS>(vs, x, lo_any - k0, s.len - k0, o, lane);
        __syncwarp();                                           // every lane has read this stage
        issue(t + C::STAGES);
        done = t + 1;
    }
    // after a failed wait: this warp's copies in flight must land (bounded)
    for (int t = done; t < min(nt, done + C::STAGES); ++t)
        mbar_wait(&full[t % C::STAGES], (t / C::STAGES) & 1, nullptr, 0);

    // ---- merge the warps: each scales its O to the common maximum -------------
    float2 *ml = reinterpret_cast<float2 *>(smem + C::ML_OFF);  // [WARPS][16]
#pragma unroll
    for (int u = 0; u < (ROWS > 8 ? 2 : 1); ++u) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
        if (c == 0) ml[warp * 16 + (lane >> 2) + 8 * u] = make_float2(m[u], l[u]);
    }
    __syncthreads();
    float *mine = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int u = 0; u < (ROWS > 8 ? 2 : 1); ++u) {
        const int r = (lane >> 2) + 8 * u;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) top = fmaxf(top, ml[w * 16 + r].x);
        const float f = m[u] == -INFINITY ? 0.f : ex2(m[u] - top);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < 2; ++j) mine[r * D + paged_o_dim<KVT>(nb, j, c)] = o[nb][2 * u + j] * f;
    }
    __syncthreads();
    const long long work = ((long long)b * a.kv.Hkv + g) * sp.n_splits + split;
    for (int i = threadIdx.x; i < rows * (D / 4); i += 128) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4;
        float top = -INFINITY, tot = 0.f;
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) top = fmaxf(top, ml[w * 16 + r].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) {
            const float2 y = ml[w * 16 + r];
            if (y.x != -INFINITY) tot += y.y * ex2(y.x - top);
            const float4 v = *reinterpret_cast<const float4 *>(smem + w * C::WARP_BYTES + (r * D + d) * 4);
            acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
        }
        if (cut.n > 1) {
            *reinterpret_cast<float4 *>(sp.part_o + (work * ROWS + r) * D + d) = acc;
            if (d == 0) reinterpret_cast<float2 *>(sp.part_ml)[work * ROWS + r] = make_float2(top, tot);
        } else {
            paged_finish<D>(a, s, g, r, d, acc, top, tot);
        }
    }
    if (cut.n == 1) return;

    // ---- merge the splits ---------------------------------------------------------
    int *last = reinterpret_cast<int *>(smem + C::ML_OFF + C::WARPS * 16 * 8);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned old;                                           // wraps to zero at the last arrival
        asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;" : "=r"(old)
                     : "l"(sp.arrived + (long long)b * a.kv.Hkv + g), "r"((unsigned)cut.n - 1) : "memory");
        *last = old == (unsigned)cut.n - 1;
    }
    __syncthreads();
    if (!*last) return;
    __threadfence();
    // a warp per query row, a lane per 4 dims (D = 64: two splits at a time),
    // eight splits' loads in flight
    constexpr int LPR = D / 4, SPW = 32 / LPR, U = 8 / SPW;
    const long long w0 = work - split;
    const int d = (lane % LPR) * 4;
    for (int r = warp; r < rows; r += C::WARPS) {
        float top = -INFINITY, tot = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = lane / LPR; i0 < cut.n; i0 += SPW * U) {
            float2 y[U];
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * SPW;
                y[u] = make_float2(-INFINITY, 0.f);
                v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < cut.n) {
                    y[u] = __ldcg(reinterpret_cast<const float2 *>(sp.part_ml) + (w0 + i) * ROWS + r);
                    v[u] = __ldcg(reinterpret_cast<const float4 *>(sp.part_o + ((w0 + i) * ROWS + r) * D + d));
                }
            }
            float mx = top;
#pragma unroll
            for (int u = 0; u < U; ++u) mx = fmaxf(mx, y[u].x);
            if (mx == -INFINITY) continue;
            const float f0 = ex2(top - mx);
            acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
            tot *= f0;
            top = mx;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float f = ex2(y[u].x - mx);
                tot = fmaf(f, y[u].y, tot);
                acc.x = fmaf(f, v[u].x, acc.x); acc.y = fmaf(f, v[u].y, acc.y);
                acc.z = fmaf(f, v[u].z, acc.z); acc.w = fmaf(f, v[u].w, acc.w);
            }
        }
        if (SPW == 2) {
            const float m2 = __shfl_xor_sync(0xffffffffu, top, 16), l2 = __shfl_xor_sync(0xffffffffu, tot, 16);
            const float4 o2 = make_float4(__shfl_xor_sync(0xffffffffu, acc.x, 16), __shfl_xor_sync(0xffffffffu, acc.y, 16),
                                          __shfl_xor_sync(0xffffffffu, acc.z, 16), __shfl_xor_sync(0xffffffffu, acc.w, 16));
            const float mx = fmaxf(top, m2);
            const float f = top == -INFINITY ? 0.f : ex2(top - mx), f2 = m2 == -INFINITY ? 0.f : ex2(m2 - mx);
            top = mx;
            tot = tot * f + l2 * f2;
            acc.x = acc.x * f + o2.x * f2; acc.y = acc.y * f + o2.y * f2;
            acc.z = acc.z * f + o2.z * f2; acc.w = acc.w * f + o2.w * f2;
        }
        if (lane < LPR) paged_finish<D>(a, s, g, r, d, acc, top, tot);
    }
}

// sp.beside: the kernel just before is the chunks' (fa_paged_sm100_kernel), which
// touches other streams' rows only.  It started once everything before it was
// complete, and this kernel starts once all of its CTAs have, so nothing needs to
// be waited for: the few-token streams fill the SMs that its last CTAs leave
// idle.  The wait comes last instead, so that this kernel's end is both ends.
template <int D, int KVT, int ROWS, bool UF>
__global__ void __launch_bounds__(128, 3)
fa_paged_decode_kernel(const PagedAttnArgs a, const PagedSplit sp)
{
    if (!sp.beside) grid_dep_wait();
    grid_dep_launch();
    paged_decode_cta<D, KVT, ROWS, UF>(a, sp);
    if (sp.beside) grid_dep_wait();
}

}  // namespace vtx
