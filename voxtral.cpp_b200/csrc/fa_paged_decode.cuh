// fa_paged_decode.cuh — HBM-streaming attention of a few new tokens per stream
// over a paged cache (decode steps, short drafts): the decode node of
// src/voxtral.cpp:1802 for streams that bring at most 16 / G tokens.
//
// Every K and V row is read once and does 4 flops a byte per query row, so the
// call is bound by HBM.  One CTA per (stream, KV head, key split); its 4 warps
// take tiles of 16 keys in turn, each through a private ring of bulk copies
// (no CTA barrier in the loop), 16-key tiles never cross a page.  The products run
// on mma.sync m16n8k16 turned round: S^T = K Q^T and O^T += V^T P^T, with the keys
// (the dims) as the 16 rows and the n * G query rows (token * G + head of the
// group), padded to 8 or 16, as the columns.  With the query rows as the MMA's
// rows half of it would be padding for G <= 8: twice the products and accumulator
// registers.
//   F16:  a lane copies one K or V row into a 16-byte padded pitch; ldmatrix.
//   Q8_0: the 16 rows of a tile are one contiguous block, copied as such.  K's
//         integers become halves exactly (0x64xx, minus 1152) and every block of
//         32 dims gets its scale in f32, so scores carry no rounding of K.  V's
//         integers are exact too: the scale of (row, block) multiplies P before P
//         is rounded to half, so P V has the one rounding that F16 has.  P stays
//         below 2^6 there, which bounds |scale| by 1023.  The k index of an MMA
//         may be any permutation: the lanes' words are chosen free of bank
//         conflicts (keys 2n and 2n + 1, words c and c + 4 of a block).
// Softmax in log2 units with a lazily moved reference m: O is rescaled only when
// some score passes it by 2^8 (2^6), which one vote per tile finds out.  The
// warps' (m, l, O) are merged in shared memory; with several splits every CTA
// leaves its result in the workspace, and the one that arrives last at the
// (stream, KV head)'s counter merges them in split order.
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
    static constexpr int STAGES = 2;
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
    c.lo = window > 0 && causal ? max(0, s.off - window + 1) & ~15 : 0;
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

// The transpose of an 8 x 8 matrix of halves held as an MMA fragment.
__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// The two keys of a tile whose scores a lane holds (which = 0, 1).
template <int KVT>
__device__ __forceinline__ int paged_tile_key(int lane, int which) {
    return KVT == 1 ? (lane >> 2) + 8 * which : 2 * (lane >> 2) + which;
}
// First dim of the pairs that a lane's Q fragment of k step kc takes (b0; b1: + 8,
// Q8_0: + 2).
template <int KVT>
__device__ __forceinline__ int paged_q_dim(int lane, int kc) {
    return KVT == 1 ? kc * 16 + 2 * (lane & 3) : (kc >> 1) * 32 + (kc & 1) * 16 + 4 * (lane & 3);
}

// S^T of 16 keys: x[nc][2 i + j] = key paged_tile_key(i), query row 8 nc + 2c + j.
template <int D, int KVT, int NC>
__device__ __forceinline__ void paged_tile_scores(const char *ks, const uint32_t (&qb)[NC][D / 16][2],
                                                  float (&x)[NC][4], int lane)
{
    using C = PagedDecodeCfg<D, KVT>;
    const int c = lane & 3, n = lane >> 2;
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[nc][i] = 0.f;
    if constexpr (KVT == 1) {
        const char *p = ks + ((lane & 7) + (lane & 8)) * C::PITCH + (lane >> 4) * 16;
        float y[NC][4];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[nc][i] = 0.f;
#pragma unroll
        for (int kc = 0; kc < D / 16; kc += 2) {            // two chains
            uint32_t k0[4], k1[4];
            ldsm_x4(k0, p + kc * 32);
            ldsm_x4(k1, p + kc * 32 + 32);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                mma16816(x[nc], k0, qb[nc][kc][0], qb[nc][kc][1]);
                mma16816(y[nc], k1, qb[nc][kc + 1][0], qb[nc][kc + 1][1]);
            }
        }
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[nc][i] += y[nc][i];
    } else {
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            const char *p = ks + 2 * n * C::ROW + 34 * b;
            uint32_t w[2][2];                               // [key][word]
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const char *q = p + i * C::ROW + 2 + 4 * c + 16 * j;
                    w[i][j] = (b & 1) ? lds_word<false>(q) : lds_word<true>(q);
                }
            const float d0 = lds_half(p), d1 = lds_half(p + C::ROW);
            uint32_t k0[4], k1[4];
            q8_halves(w[0][0], k0[0], k0[2]);
            q8_halves(w[1][0], k0[1], k0[3]);
            q8_halves(w[0][1], k1[0], k1[2]);
            q8_halves(w[1][1], k1[1], k1[3]);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                float y[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816(y, k0, qb[nc][2 * b][0], qb[nc][2 * b][1]);
                mma16816(y, k1, qb[nc][2 * b + 1][0], qb[nc][2 * b + 1][1]);
                x[nc][0] = fmaf(d0, y[0], x[nc][0]);
                x[nc][1] = fmaf(d0, y[1], x[nc][1]);
                x[nc][2] = fmaf(d1, y[2], x[nc][2]);
                x[nc][3] = fmaf(d1, y[3], x[nc][3]);
            }
        }
    }
}

// O^T += V^T P^T of 16 keys; o[nc][mt][2 i + j]: dim paged_o_dim(mt, i), query row
// 8 nc + 2c + j.  Rows of the tile outside [n0, n1) hold anything (Q8_0: their
// scale is taken as 0; F16: the loader zeroed them).
template <int D, int KVT, int NC>
__device__ __forceinline__ void paged_tile_pv(const char *vs, const float (&p)[NC][4], int n0, int n1,
                                              float (&o)[NC][D / 16][4], int lane)
{
    using C = PagedDecodeCfg<D, KVT>;
    const int c = lane & 3, n = lane >> 2;
    if constexpr (KVT == 1) {
        uint32_t pb[NC][2];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            pb[nc][0] = movm_t(pack_half2(p[nc][0], p[nc][1]));
            pb[nc][1] = movm_t(pack_half2(p[nc][2], p[nc][3]));
        }
        const char *q = vs + ((lane >> 4) * 8 + (lane & 7)) * C::PITCH + (lane & 8) * 2;
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
            uint32_t v[4];
            ldsm_x4_t(v, q + mt * 32);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) mma16816(o[nc][mt], v, pb[nc][0], pb[nc][1]);
        }
    } else {
        const char *v0 = vs + 4 * c * C::ROW;               // the k pairs: keys (4c, 4c + 2) and (4c + 1, 4c + 3)
        const char *s0 = vs + 2 * n * C::ROW;               // P's keys: 2n and 2n + 1
        const bool on0 = 2 * n >= n0 && 2 * n < n1, on1 = 2 * n + 1 >= n0 && 2 * n + 1 < n1;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            const float d0 = on0 ? lds_half(s0 + 34 * b) : 0.f, d1 = on1 ? lds_half(s0 + C::ROW + 34 * b) : 0.f;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const char *q = v0 + j * C::ROW + 34 * b + 2 + 4 * n;
                w[j] = (b & 1) ? lds_word<false>(q) : lds_word<true>(q);
            }
            uint32_t v[2][4];                               // bytes 2 mt and 2 mt + 1 of word n: rows n, n + 8
            q8_halves(__byte_perm(w[0], w[2], 0x5140), v[0][0], v[0][1]);
            q8_halves(__byte_perm(w[0], w[2], 0x7362), v[1][0], v[1][1]);
            q8_halves(__byte_perm(w[1], w[3], 0x5140), v[0][2], v[0][3]);
            q8_halves(__byte_perm(w[1], w[3], 0x7362), v[1][2], v[1][3]);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                const uint32_t b0 = movm_t(pack_half2(p[nc][0] * d0, p[nc][1] * d0));
                const uint32_t b1 = movm_t(pack_half2(p[nc][2] * d1, p[nc][3] * d1));
                mma16816(o[nc][2 * b], v[0], b0, b1);
                mma16816(o[nc][2 * b + 1], v[1], b0, b1);
            }
        }
    }
}

// The head dim of o[nc][mt][2 i + j].
template <int KVT>
__device__ __forceinline__ int paged_o_dim(int mt, int i, int lane) {
    return KVT == 1 ? mt * 16 + (lane >> 2) + 8 * i : (mt >> 1) * 32 + 4 * (lane >> 2) + 2 * (mt & 1) + i;
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
    constexpr int KC = D / 16, NC = ROWS / 8;
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
    const int off = s.off;
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

    // Q fragments: a lane's column is query row 8 nc + lane / 4; its scores are of
    // rows 8 nc + 2c + j, whose limits these are
    uint32_t qb[NC][KC][2];
    int lo[NC][2], hi[NC][2];
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
        const int r = 8 * nc + (lane >> 2);
        const bool on = r < rows;
        const int tok = on ? r / a.G : 0;
        const char *qp = a.q + (long long)(s.q0 + tok) * a.q_nbt + (long long)(g * a.G + (on ? r % a.G : 0)) * a.q_nbh;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            const int d = paged_q_dim<KVT>(lane, kc);
            qb[nc][kc][0] = on ? paged_q2(qp, a.q_f16, d) : 0u;
            qb[nc][kc][1] = on ? paged_q2(qp, a.q_f16, d + (KVT == 1 ? 8 : 2)) : 0u;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r2 = 8 * nc + 2 * c + j, tok2 = r2 / a.G;
            hi[nc][j] = r2 < rows ? (a.causal ? min(off + tok2, s.len - 1) : s.len - 1) : -1;
            lo[nc][j] = a.window > 0 ? off + tok2 - a.window + 1 : 0;
        }
    }
    // every token sees [lo_all, hi_all] (padding rows' results are not read)
    const int hi_all = a.causal ? min(off, s.len - 1) : s.len - 1;
    const int lo_all = a.window > 0 ? off + s.n_new - a.window : 0;

    float o[NC][KC][4];
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int i = 0; i < KC; ++i) o[nc][i][0] = o[nc][i][1] = o[nc][i][2] = o[nc][i][3] = 0.f;
    float m[NC][2], l[NC][2];
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
        m[nc][0] = m[nc][1] = -INFINITY;
        l[nc][0] = l[nc][1] = 0.f;
    }
    const float cx = a.scale * kLog2e;
    constexpr float kJump = KVT == 1 ? 8.0f : 6.0f, kBack = KVT == 1 ? 0.0f : 4.0f;
    bool ok = true;
    int done = 0;
    for (int t = 0; t < nt; ++t) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full[t % C::STAGES], (t / C::STAGES) & 1, a.kv.err, VTX_KERR_KV));
        if (!ok) break;
        const char *ks = ring + (t % C::STAGES) * C::STAGE_BYTES, *vs = ks + C::KEYS * C::PITCH;
        const int k0 = cut.lo + 16 * (first + t * C::WARPS);
        float x[NC][4];
        paged_tile_scores<D, KVT, NC>(ks, qb, x, lane);
        const bool inner = k0 >= lo_all && k0 + 15 <= hi_all;
        bool jump = false;
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float &y = x[nc][i];
                y = paged_logit_t<UF>(y, cx, a.scale, a.softcap);
                if (!inner) {
                    const int key = k0 + paged_tile_key<KVT>(lane, i >> 1);
                    y = key < lo[nc][i & 1] || key > hi[nc][i & 1] ? -INFINITY : y;
                }
                jump |= y > m[nc][i & 1] + kJump;
            }
        if (__any_sync(0xffffffffu, jump)) {
#pragma unroll
            for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float mx = fmaxf(x[nc][j], x[nc][2 + j]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    if (mx > m[nc][j] + kJump) {            // the same in every lane of this row
                        const float al = ex2(m[nc][j] - (mx - kBack));
                        m[nc][j] = mx - kBack;
                        l[nc][j] *= al;
#pragma unroll
                        for (int i = 0; i < KC; ++i) { o[nc][i][j] *= al; o[nc][i][2 + j] *= al; }
                    }
                }
        }
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float mu = m[nc][j] == -INFINITY ? 0.f : m[nc][j];
                x[nc][j] = ex2(x[nc][j] - mu);
                x[nc][2 + j] = ex2(x[nc][2 + j] - mu);
                l[nc][j] += x[nc][j] + x[nc][2 + j];
            }
        paged_tile_pv<D, KVT, NC>(vs, x, lo_any - k0, s.len - k0, o, lane);
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
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            l[nc][j] += __shfl_xor_sync(0xffffffffu, l[nc][j], 4);
            l[nc][j] += __shfl_xor_sync(0xffffffffu, l[nc][j], 8);
            l[nc][j] += __shfl_xor_sync(0xffffffffu, l[nc][j], 16);
            if (lane < 4) ml[warp * 16 + 8 * nc + 2 * c + j] = make_float2(m[nc][j], l[nc][j]);
        }
    __syncthreads();
    float *mine = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = 8 * nc + 2 * c + j;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < C::WARPS; ++w) top = fmaxf(top, ml[w * 16 + r].x);
            const float f = m[nc][j] == -INFINITY ? 0.f : ex2(m[nc][j] - top);
#pragma unroll
            for (int mt = 0; mt < KC; ++mt)
#pragma unroll
                for (int i = 0; i < 2; ++i) mine[r * D + paged_o_dim<KVT>(mt, i, lane)] = o[nc][mt][2 * i + j] * f;
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
            tot += y.x == -INFINITY ? y.y : y.y * ex2(y.x - top);       // NaN where all its scores were
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
            const float ref = mx == -INFINITY ? 0.f : mx;       // nothing seen, or NaN alone, which stays NaN
            const float f0 = ex2(top - ref);
            acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
            tot *= f0;
            top = mx;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float f = ex2(y[u].x - ref);
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
// Waiting is also what makes the memory of earlier kernels visible.  In its place a
// fence at the start keeps this SM's cache from answering with lengths, pages or
// queries of an earlier step (loads from L2 instead, in every launch: one stream of
// 1k rows 7.6 -> 8.5 us).
template <int D, int KVT, int ROWS, bool UF>
__global__ void __launch_bounds__(128, KVT == 8 && ROWS == 8 ? 5 : 3)
fa_paged_decode_kernel(const PagedAttnArgs a, const PagedSplit sp)
{
    if (sp.beside) asm volatile("fence.acq_rel.gpu;" ::: "memory");
    else grid_dep_wait();
    grid_dep_launch();
    paged_decode_cta<D, KVT, ROWS, UF>(a, sp);
    if (sp.beside) grid_dep_wait();
}

}  // namespace vtx
