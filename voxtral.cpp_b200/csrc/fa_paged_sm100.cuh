// fa_paged_sm100.cuh — tensor-core attention of chunks of new tokens over a
// paged F16 cache (tcgen05 / TMEM / TMA): the decoder prefill node of
// src/voxtral.cpp:1802 for ragged batches, bound by the tensor core and the
// exponentials (4 D flops and one exp per query row and visible key).
//
// A CTA owns a group of two 128-row Q tiles (one, when pairs would leave SMs idle)
// of one stream and KV head (row = token * G + head of the group, T = 128 / G
// tokens a tile) and one split of its key tiles of 128.  Two softmax warpgroups, one
// per Q tile (a thread per row = TMEM lane), take turns on the tensor core.  Of a
// group with one Q tile they take the key tiles in turn, each with its own (m, l, O),
// which the first one joins at the end: a prompt of 391 tokens 14.6 -> 13.3 us, 391
// more at 600 rows 24.3 -> 18.3.  A third warpgroup holds the TMA and the MMA warp and
// gives its registers away (setmaxnreg).  Per key tile and Q tile: S = Q K^T into
// TMEM, P = 2^(x - m) over S's first half columns, O += P V with P read from TMEM.
// Shared memory: both Q tiles, and rings of K and V tiles, all in the 128-byte
// swizzle.
//
// Pages: a tensor map (dim, row, head, page) per pool; a key tile is one box of
// 64 dims x min(page, 128) rows per page and half row, a lane of the TMA warp
// each.  Pages without a row that the group sees are not touched; rows of the
// other pages outside the group's key range may hold anything, so the softmax
// warps clear those V rows in shared memory before P V (masked P is 0, and
// 0 * NaN is not), while masked scores are replaced.
//
// LO: an unpacked Q8_0 cache, whose tiles hold 64 keys as 64 rows of hi and 64 of lo
// (value = hi + lo).  S's two halves are added before the softmax and P is stored
// twice, so both products stay as they are; 2048 tokens at 14k keys 833 us next to
// 502 over F16 pages, for twice the products.
//
// D = 64, twice the exponentials per flop: a quarter of them runs on the FMA pipe
// (2048 tokens at 14k keys 496-506 us without, 449-500 with, by how warm the board is;
// over Q8_0 652 and 631; D = 128 gained nothing, 519 us either way, and under the power
// cap it costs, 569 against 562 us).  2^x = 2^j p(f), j = round(x),
// with p the degree-4 polynomial of least relative error (2.6e-6) on
// [-1/2, 1/2], fitted here by an exchange.  The row sums are taken of the f32
// P, so lse carries neither P's rounding to half nor more than that error.
//
// Splits: with few groups the key tiles of a group are cut into up to n_splits
// ranges; their (m, l, O) are merged by fa_paged_tile_combine_kernel.  With one
// stream the first `whole` (group, head) items, full waves of CTAs, are not cut:
// only the rest is, so that the last wave is full too.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "vtx_ptx.cuh"
#include "paged_kv.cuh"
#include "fa_paged.cuh"
#include "fa_prefill_sm100.cuh"

namespace vtx {

struct PagedTile {
    int T;                    // tokens per Q tile: 128 / G
    int tokens;               // tokens per group: 2 T, or T when pairs would leave SMs idle
    int groups;               // bound on the groups of all streams
    int n_splits, min_tiles;  // splits of a group's key tiles at most, key tiles per split at least
    int whole;                // (group, head) items that are not split, the first ones
    int shift;                // log2 of the keys of a tile: 7, or 6 where a key has two rows
    float *part_o, *part_ml;  // [n_splits][n_tokens][Hq][D], ... [2] (m, l)
};

template <int D> struct PagedTileCfg {
    static constexpr int SUB = D / 64;
    static constexpr int TILE = 128 * D * 2;
    static constexpr int STAGES = D == 64 ? 4 : 2;
    static constexpr int Q_OFF = 0, K_OFF = 2 * TILE, V_OFF = K_OFF + STAGES * TILE;
    static constexpr int BAR_OFF = V_OFF + STAGES * TILE;
    static constexpr int NBARS = 1 + 4 * STAGES + 6;
    static constexpr int ML_OFF = BAR_OFF + NBARS * 8 + 32;            // (m, l) of the second warpgroup's rows
    static constexpr int SMEM = ML_OFF + 1024 + 1024;                  // + alignment slack
    static constexpr int NTHREADS = 384, TMA_WARP = 8, MMA_WARP = 9;
    static constexpr int REG_SOFTMAX = 224, REG_PRODUCER = 56;         // 256 x 224 + 128 x 56 = 384 x 168
    __host__ __device__ static constexpr int s_col(int t) { return t * 128; }
    __host__ __device__ static constexpr int o_col(int t) { return 256 + t * D; }
};

// Maximum that keeps a NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^x of a pair on the FMA pipe, x <= ~8; below -125, and for a NaN, the result is
// about 2^-125.
__device__ __forceinline__ void paged_exp2_pair(float &a, float &b) {
    const float kRound = 12582912.0f;                    // 1.5 * 2^23
    a = fmaxf(a, -125.0f);
    b = fmaxf(b, -125.0f);
    const uint64_t x = pk2(a, b);
    const uint64_t t = fadd2(x, pk2(kRound, kRound));
    const uint64_t f = fsub2(x, fadd2(t, pk2(-kRound, -kRound)));
    uint64_t p = ffma2(pk2(0.00957010191f, 0.00957010191f), f, pk2(0.0559178603f, 0.0559178603f));
    p = ffma2(p, f, pk2(0.240247448f, 0.240247448f));
    p = ffma2(p, f, pk2(0.693121815f, 0.693121815f));
    p = ffma2(p, f, pk2(0.999999261f, 0.999999261f));
    float pa, pb, ta, tb;
    upk2(p, pa, pb);
    upk2(t, ta, tb);
    a = __int_as_float(__float_as_int(pa) + (__float_as_int(ta) << 23));
    b = __int_as_float(__float_as_int(pb) + (__float_as_int(tb) << 23));
}

// Groups (pairs of Q tiles, or single ones) of a stream with n_new tokens.
__device__ __forceinline__ int paged_groups(int n_new, const PagedAttnArgs &a, const PagedTile &tl) {
    return n_new * a.G > a.min_rows ? (n_new + tl.tokens - 1) / tl.tokens : 0;
}

// Key tiles [j0, j1) of a group whose first token is tok0, and their splits.
struct PagedRange {
    int lo, hi;               // keys some token of the group sees
    int j0, j1, per, n;
};
__device__ __forceinline__ PagedRange paged_range(const PagedSeq &s, int tok0, const PagedAttnArgs &a,
                                                  const PagedTile &tl, bool cut) {
    PagedRange r;
    const int last = min(s.n_new, tok0 + tl.tokens) - 1;
    r.hi = a.causal ? min(s.off + last, s.len - 1) : s.len - 1;
    r.lo = a.window > 0 ? max(0, s.off + tok0 - a.window + 1) : 0;
    r.j0 = r.hi >= r.lo ? r.lo >> tl.shift : 0;
    r.j1 = r.hi >= r.lo ? (r.hi >> tl.shift) + 1 : 0;
    const int most = cut ? tl.n_splits : 1;
    r.per = max(tl.min_tiles, (r.j1 - r.j0 + most - 1) / most);
    r.n = max(1, (r.j1 - r.j0 + r.per - 1) / r.per);
    return r;
}

template <int D, bool UF, bool LO>
__global__ void __launch_bounds__(PagedTileCfg<D>::NTHREADS, 1)
fa_paged_sm100_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ CUtensorMap tmQ, const PagedAttnArgs a, const PagedTile tl)
{
    using C = PagedTileCfg<D>;
    constexpr int KEYS = LO ? 64 : 128;            // of a tile
    extern __shared__ __align__(1024) char smem_raw[];
    char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *q_full = reinterpret_cast<uint64_t *>(smem + C::BAR_OFF);
    uint64_t *k_full = q_full + 1;
    uint64_t *v_full = k_full + C::STAGES;
    uint64_t *k_empty = v_full + C::STAGES;
    uint64_t *v_empty = k_empty + C::STAGES;
    uint64_t *s_full = v_empty + C::STAGES;        // [2]
    uint64_t *p_full = s_full + 2;                 // [2]
    uint64_t *o_tile = p_full + 2;                 // [2]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(o_tile + 2);
    int *found = reinterpret_cast<int *>(tmem_slot + 2);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // item = group * Hkv + head; behind the whole ones n_splits CTAs each
    const int behind = (int)blockIdx.x - tl.whole;
    const int item = behind < 0 ? (int)blockIdx.x : tl.whole + behind / tl.n_splits;
    const int split = behind < 0 ? 0 : behind % tl.n_splits;
    const int g = item % a.kv.Hkv;

    if (tid == 32) {
        mbar_init(q_full, a.q_f16 ? 1 : 8);        // the TMA lane, or one arrival per softmax warp
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 4);
            mbar_init(&o_tile[t], 1);
        }
        fence_mbar_init();
    }
    if (warp == C::TMA_WARP && lane == 0) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        if (a.q_f16) tma_prefetch_desc(&tmQ);
    }
    grid_dep_wait();
    grid_dep_launch();
    if (warp == 0) {                               // the stream and group of this CTA
        const int want = item / a.kv.Hkv;
        int base = 0, b = -1, grp = 0;
        for (int i0 = 0; i0 < a.kv.n_seq && b < 0; i0 += 32) {
            const int i = i0 + lane;
            const int cnt = i < a.kv.n_seq ? paged_groups(min(paged_seq(a.kv, i).n_new, a.kv.max_new), a, tl) : 0;
            int inc = cnt;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += x;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, want < base + inc);
            if (hit) {
                const int l = __ffs(hit) - 1;
                b = i0 + l;
                // a stream's last group, whose key range is the longest, first
                grp = base + __shfl_sync(0xffffffffu, inc, l) - 1 - want;
            } else {
                base += __shfl_sync(0xffffffffu, inc, 31);
            }
        }
        if (lane == 0) {
            found[0] = b;
            found[1] = grp;
        }
    }
    __syncthreads();
    const int b = found[0];
    if (b < 0) return;
    PagedSeq s = paged_seq(a.kv, b);
    if (s.n_new > a.kv.max_new) {                  // what exceeds the bound is not served
        if (tid == 0) paged_report(a.kv, VTX_KERR_BOUND);
    }
    const int n_serve = min(s.n_new, a.kv.max_new);
    const int tok0 = found[1] * tl.tokens;
    const PagedRange rg = paged_range(s, tok0, a, tl, behind >= 0);
    if (split >= rg.n) return;
    const int jb = rg.j0 + split * rg.per;
    const int n_iter = max(0, min(jb + rg.per, rg.j1) - jb);
    const bool two = tl.tokens > tl.T && tok0 + tl.T < n_serve;        // the second Q tile holds tokens

    if (warp == C::MMA_WARP) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int off = s.off;

    if (warp < 8) {
        setmaxnreg_inc<C::REG_SOFTMAX>();
        // =================== softmax warpgroups ===============================
        // with two Q tiles a warpgroup each; with one the warpgroups take its key tiles in turn
        const int t = warp >> 2, r = tid & 127, step = two ? 1 : 2, it0 = two ? 0 : t;
        const int tok = tok0 + (two ? t * tl.T : 0) + r / a.G, head = g * a.G + r % a.G;
        const bool row_ok = r < tl.T * a.G && tok < n_serve;
        const int iters = (n_iter - it0 + step - 1) / step;
        bool ok = true;
        int lo = 1, hi = 0;
        if (row_ok) {
            hi = a.causal ? min(off + tok, s.len - 1) : s.len - 1;
            lo = a.window > 0 ? max(0, off + tok - a.window + 1) : 0;
        }
        char *qtile = smem + C::Q_OFF + t * C::TILE;
        if (!a.q_f16) {                            // F32 q: each thread rounds its row to half
            const char *src = a.q + (long long)(s.q0 + tok) * a.q_nbt + (long long)head * a.q_nbh;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                uint4 pk = make_uint4(0u, 0u, 0u, 0u);
                if (t == 1 && !two) break;
                if (row_ok) {
                    const float4 x = *reinterpret_cast<const float4 *>(src + c * 32);
                    const float4 y = *reinterpret_cast<const float4 *>(src + c * 32 + 16);
                    pk = make_uint4(pack_half2(x.x, x.y), pack_half2(x.z, x.w), pack_half2(y.x, y.y), pack_half2(y.z, y.w));
                }
                *reinterpret_cast<uint4 *>(qtile + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = pk;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + lane_base + C::s_col(t);
        const uint32_t o_addr = tmem + lane_base + C::o_col(t);
        const float cx = UF ? 1.0f : a.scale * kLog2e;
        float m_run = -INFINITY, l_run = 0.0f;

        for (int i0 = 0, it = it0; i0 < iters; ++i0, it += step) {
            ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], i0 & 1, a.kv.err, VTX_KERR_S));
            if (!ok) break;
            tc_fence_after();
            float x[KEYS];
            {
                uint32_t raw[128];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[c * 32]));
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < KEYS; ++i)
                    x[i] = LO ? __uint_as_float(raw[i]) + __uint_as_float(raw[(i + 64) % 128]) : __uint_as_float(raw[i]);
            }
            const int k0 = (jb + it) * KEYS;
            if (UF) {
#pragma unroll
                for (int i = 0; i < KEYS; ++i) x[i] = paged_logit(x[i], a.scale, a.softcap);
            }
            const bool full = !row_ok || (k0 >= lo && k0 + KEYS - 1 <= hi);
            if (__any_sync(0xffffffffu, !full)) {
#pragma unroll
                for (int i = 0; i < KEYS; ++i) x[i] = (k0 + i < lo || k0 + i > hi) ? -INFINITY : x[i];
            }
            // V rows outside the group's key range hold anything: clear them
            if (k0 < rg.lo || k0 + KEYS - 1 > rg.hi) {
                const int st = it % C::STAGES;
                ok = __all_sync(0xffffffffu, mbar_wait(&v_full[st], (it / C::STAGES) & 1, a.kv.err, VTX_KERR_KV));
                if (!ok) break;
                if (const int key = k0 + (r & (KEYS - 1)); key < rg.lo || key > rg.hi) {
                    char *v = smem + C::V_OFF + st * C::TILE + r * 128;
#pragma unroll
                    for (int i = 0; i < C::SUB * 8; ++i)
                        *reinterpret_cast<uint4 *>(v + (i >> 3) * 16384 + (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();
            }
            float mx8[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                constexpr int W = KEYS / 8;
                mx8[k] = max3_nan(x[W * k], x[W * k + 1], x[W * k + 1]);
#pragma unroll
                for (int i = 2; i < W; i += 2) mx8[k] = max3_nan(mx8[k], x[W * k + i], x[W * k + i + 1]);
            }
            const float mx = max3_nan(max3_nan(mx8[0], mx8[1], mx8[2]), max3_nan(mx8[3], mx8[4], mx8[5]),
                                      max3_nan(mx8[6], mx8[7], mx8[7])) * cx;
            bool rescale = false;
            float alpha = 1.0f;
            if (mx > m_run + 8.0f) {               // the reference moves only on a 2^8 jump
                if (m_run != -INFINITY) {
                    alpha = ex2(m_run - mx);
                    rescale = i0 > 0;
                }
                m_run = mx;
                l_run *= alpha;
            }
            const float neg_m = m_run == -INFINITY ? 0.0f : -m_run;
            const uint64_t cx2 = pk2(cx, cx), nm2 = pk2(neg_m, neg_m);
            uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
            uint32_t pk[KEYS / 2];
#pragma unroll
            for (int i = 0; i < KEYS / 2; ++i) {
                float e0, e1;
                upk2(ffma2(pk2(x[2 * i], x[2 * i + 1]), cx2, nm2), e0, e1);
                if (D == 64 && (i & 3) == 3) {     // every fourth pair off the MUFU
                    paged_exp2_pair(e0, e1);
                } else {
                    e0 = ex2(e0);
                    e1 = ex2(e1);
                }
                sum2[i & 3] = fadd2(sum2[i & 3], pk2(e0, e1));
                pk[i] = pack_half2(e0, e1);
            }
            {
                float sa, sb;
                upk2(fadd2(fadd2(sum2[0], sum2[1]), fadd2(sum2[2], sum2[3])), sa, sb);
                l_run += sa + sb;
            }
            if (!(mx < INFINITY)) l_run = NAN;     // a score of NaN or +inf, which the polynomial would lose
            tmem_st32(s_addr, *reinterpret_cast<const uint32_t(*)[32]>(&pk[0]));
            tmem_st32(s_addr + 32, *reinterpret_cast<const uint32_t(*)[32]>(&pk[LO ? 0 : 32]));
            // tcgen05.ld / st are warp-collective: the warp rescales when any row needs it
            if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(o_addr + c * 32, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                    tmem_st32(o_addr + c * 32, o);
                }
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t]);
        }
        // ---- write-back: rows staged in this tile's own Q tile
        if (iters > 0) {
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&o_tile[t], 0, a.kv.err, VTX_KERR_O));
            tc_fence_after();
        }
        // saw nothing: the sum holds 2^-125s (NaN where every score was, which stays)
        if (m_run == -INFINITY && l_run == l_run) l_run = 0.0f;
        float f0 = 1.0f, f1 = 0.0f;                // weights of this warpgroup's O and the other one's
        const bool join = !two && n_iter > 1;
        if (join) {                                // the first warpgroup takes the second one's sums in
            float2 *ml = reinterpret_cast<float2 *>(smem + C::ML_OFF);
            if (t == 1) ml[r] = make_float2(m_run, l_run);
            asm volatile("bar.sync 3, 256;" ::: "memory");
            if (t == 0) {
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&o_tile[1], 0, a.kv.err, VTX_KERR_O));
                tc_fence_after();
                const float2 y = ml[r];
                const float top = fmaxf(m_run, y.x);
                f0 = m_run == -INFINITY ? 0.0f : ex2(m_run - top);
                f1 = y.x == -INFINITY ? 0.0f : ex2(y.x - top);
                m_run = top;
                l_run = l_run * f0 + y.y * f1;
            }
        }
        const bool part = rg.n > 1;
        const float inv = part ? 1.0f : (l_run == 0.0f ? 0.0f : 1.0f / l_run);
        f0 *= inv;
        f1 *= inv;
        const long long row = (long long)(s.q0 + tok) * a.Hq + head;
        if (row_ok && ok && (t == 0 || two)) {
            if (part)
                reinterpret_cast<float2 *>(tl.part_ml)[(long long)split * a.kv.n_tokens * a.Hq + row] =
                    make_float2(m_run, l_run);
            else if (a.lse)
                a.lse[row] = l_run == 0.0f ? -INFINITY : (m_run + log2f(l_run)) * kLn2;
        }
        if (t == 0 || two) {
            // staged W bytes a row at a time (16-byte chunk c of row r at c ^ (r & 7))
            constexpr int W = C::TILE / 128, CH = W / 16;
            const bool f16 = !part && a.d_f16;
            const int bytes = D * (f16 ? 2 : 4);
            if (iters == 0) asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");   // after any Q rows written here
            for (int c0 = 0; c0 < bytes; c0 += W) {
                if (c0 > 0) asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");   // the staged rows were read
                if (ok) {
                    for (int c = 0; c < W / (f16 ? 64 : 128); ++c) {   // 32 columns
                        uint32_t o[32];
                        if (iters > 0) {
                            tmem_ld32(o_addr + c0 / (f16 ? 2 : 4) + c * 32, o);
                            tmem_ld_wait();
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = 0u;
                        }
                        float y[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(o[i]) * f0;
                        if (join) {
                            tmem_ld32(o_addr + D + c0 / (f16 ? 2 : 4) + c * 32, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) y[i] = fmaf(__uint_as_float(o[i]), f1, y[i]);
                        }
                        if (f16) {
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                *reinterpret_cast<uint4 *>(qtile + r * W + (((c * 4 + q) ^ (r & 7)) << 4)) =
                                    make_uint4(pack_half2(y[8 * q], y[8 * q + 1]), pack_half2(y[8 * q + 2], y[8 * q + 3]),
                                               pack_half2(y[8 * q + 4], y[8 * q + 5]), pack_half2(y[8 * q + 6], y[8 * q + 7]));
                        } else {
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                *reinterpret_cast<float4 *>(qtile + r * W + (((c * 8 + q) ^ (r & 7)) << 4)) =
                                    make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
                        }
                    }
                }
                asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");               // staged
                if (ok) {
                    for (int i = r; i < 128 * CH; i += 128) {
                        const int rr = i / CH, ch = i % CH;
                        const int tk = tok0 + t * tl.T + rr / a.G, hd = g * a.G + rr % a.G;
                        if (rr >= tl.T * a.G || tk >= n_serve) break;
                        const uint4 v = *reinterpret_cast<const uint4 *>(qtile + rr * W + ((ch ^ (rr & 7)) << 4));
                        char *p = part ? reinterpret_cast<char *>(tl.part_o + (((long long)split * a.kv.n_tokens + s.q0 + tk) * a.Hq + hd) * D)
                                       : a.dst + (long long)(s.q0 + tk) * a.d_nbt + (long long)hd * a.d_nbh;
                        *reinterpret_cast<uint4 *>(p + c0 + ch * 16) = v;
                    }
                }
            }
        }
    } else {
        setmaxnreg_dec<C::REG_PRODUCER>();
        if (warp == C::TMA_WARP) {
            // =================== TMA: Q, then K and V tile by tile ============
            if (a.q_f16 && n_iter > 0) {
                if (lane == 0) {
                    const int nq = two ? 2 : 1;
                    mbar_arrive_expect_tx(q_full, (uint32_t)(nq * C::SUB * 128 * tl.T * a.G));
                    for (int t = 0; t < nq; ++t)
                        for (int sub = 0; sub < C::SUB; ++sub)
                            tma_load_4d(smem + C::Q_OFF + t * C::TILE + sub * 16384, &tmQ, q_full, sub * 64, g * a.G,
                                        s.q0 + tok0 + t * tl.T, 0);
                }
                __syncwarp();
            }
            const int rows_box = LO ? 128 : min(128, 1 << a.kv.shift), per_tile = 128 / rows_box;   // boxes of a half-width tile
            const int mask = (1 << a.kv.shift) - 1, rows = LO ? 2 : 1;       // rows of a key
            // lane = box of a tile; 64 boxes at most (16-row pages: 8 pages x SUB x {K, V} = 32 for D = 128)
            const int kvsel = lane / (per_tile * C::SUB);                   // 0: K, 1: V, more: idle
            const int sub = (lane / per_tile) % C::SUB, pg = lane % per_tile;
            const bool mine = kvsel < 2;
            auto page_at = [&](int it) -> int {    // this lane's page of tile it, -1: none needed
                const int y = (jb + it) * KEYS + pg * rows_box;
                if (!mine || it >= n_iter || y > rg.hi || y + rows_box <= rg.lo) return -1;
                return max(paged_page(a.kv, b, y), 0);
            };
            // K's stage is free after Q K^T, V's after P V: K is loaded first
            int issued[2] = {0, 0}, next = page_at(0);
            for (int it = 0; it < n_iter; ++it) {
                const int st = it % C::STAGES, cur = next;
                next = page_at(it + 1);
                const unsigned live = __ballot_sync(0xffffffffu, cur >= 0);
                const uint32_t bytes = (uint32_t)(__popc(live) / 2 * rows_box * 128);       // of K's boxes; V has the same
                const int y = ((jb + it) * KEYS + pg * rows_box & mask) * rows;
                bool good = true;
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    if (it >= C::STAGES)
                        good = __all_sync(0xffffffffu, mbar_wait(kv ? &v_empty[st] : &k_empty[st],
                                                                 ((it / C::STAGES) - 1) & 1, a.kv.err, VTX_KERR_KV));
                    if (!good) break;
                    issued[kv] = it + 1;
                    uint64_t *bar = kv ? &v_full[st] : &k_full[st];
                    if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
                    __syncwarp();
                    if (cur >= 0 && kvsel == kv)
                        tma_load_4d(smem + (kv ? C::V_OFF : C::K_OFF) + st * C::TILE + sub * 16384 + pg * rows_box * 128,
                                    kv ? &tmV : &tmK, bar, sub * 64, y, g, cur);
                    __syncwarp();
                }
                if (!good) break;
            }
            // the last loads must have landed before shared memory is released
            for (int kv = 0; kv < 2; ++kv)
                for (int it = max(0, issued[kv] - C::STAGES); it < issued[kv]; ++it)
                    mbar_wait(kv ? &v_full[it % C::STAGES] : &k_full[it % C::STAGES], (it / C::STAGES) & 1, a.kv.err,
                              VTX_KERR_KV);
            if (a.q_f16 && n_iter > 0) mbar_wait(q_full, 0, a.kv.err, VTX_KERR_Q);
        } else if (warp == C::MMA_WARP && n_iter > 0) {
            // =================== MMA issuer (warp converged, one elected lane) =
            const uint32_t lead = elect_one();
            constexpr uint32_t IDESC_QK = idesc_f16_f32(128, 128, 0, 0);
            constexpr uint32_t IDESC_PV = idesc_f16_f32(128, D, 0, 1);
            constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);   // SBO 1024, v1, 128-byte swizzle
            const uint32_t sbase = smem_u32(smem);
            const uint32_t lo_q = ((sbase + C::Q_OFF) >> 4) | (1u << 16);
            const uint32_t lo_k = ((sbase + C::K_OFF) >> 4) | (1u << 16);
            const uint32_t lo_v = ((sbase + C::V_OFF) >> 4) | ((16384u >> 4) << 16);   // LBO: next 64 columns
            constexpr uint32_t T16 = C::TILE >> 4;
            const int nt = two ? 2 : min(2, n_iter);                    // warpgroups at work
            bool good = __all_sync(0xffffffffu, mbar_wait(q_full, 0, a.kv.err, VTX_KERR_Q));
            tc_fence_after();
            auto issue_qk = [&](int qt, int t, int st) {                // Q tile qt into warpgroup t's S
                const uint32_t d = tmem + C::s_col(t), q = lo_q + qt * T16, k = lo_k + st * T16;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t ko = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
                    mma_f16_ss_w(lead, d, desc64(q + ko, HI), desc64(k + ko, HI), IDESC_QK, kk > 0);
                }
                mma_commit_w(lead, &s_full[t]);
            };
            auto issue_pv = [&](int t, int st, uint32_t acc) {
                const uint32_t p = tmem + C::s_col(t), d = tmem + C::o_col(t), v = lo_v + st * T16;
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                    mma_f16_ts_w(lead, d, p + kk * 8, desc64(v + kk * (2048 >> 4), HI), IDESC_PV, kk > 0 ? 1u : acc);
            };
            auto wait_k = [&](int it) {
                return __all_sync(0xffffffffu, mbar_wait(&k_full[it % C::STAGES], (it / C::STAGES) & 1, a.kv.err, VTX_KERR_KV));
            };
            auto wait_v = [&](int it) {
                return __all_sync(0xffffffffu, mbar_wait(&v_full[it % C::STAGES], (it / C::STAGES) & 1, a.kv.err, VTX_KERR_KV));
            };
            auto wait_p = [&](int t, int i) {
                return __all_sync(0xffffffffu, mbar_wait(&p_full[t], i & 1, a.kv.err, VTX_KERR_P));
            };
            if (two) {
                for (int it = 0; it <= n_iter && good; ++it) {
                    for (int t = 0; t < 2 && good; ++t) {
                        if (it > 0) {
                            if (t == 0) good = wait_v(it - 1);
                            if (good) good = wait_p(t, it - 1);
                            if (!good) break;
                            tc_fence_after();
                            issue_pv(t, (it - 1) % C::STAGES, it > 1 ? 1u : 0u);
                            if (it == n_iter) mma_commit_w(lead, &o_tile[t]);
                        }
                        if (it < n_iter) {
                            if (t == 0) good = wait_k(it);
                            if (!good) break;
                            tc_fence_after();
                            issue_qk(t, t, it % C::STAGES);
                        }
                    }
                    if (good && it > 0) mma_commit_w(lead, &v_empty[(it - 1) % C::STAGES]);
                    if (good && it < n_iter) mma_commit_w(lead, &k_empty[it % C::STAGES]);
                }
            } else {                               // key tile i is warpgroup i % 2's
                for (int it = 0; it < n_iter + 2 && good; ++it) {
                    const int t = it & 1, j = it - 2;
                    if (j >= 0) {
                        good = wait_v(j) && wait_p(t, j >> 1);
                        if (!good) break;
                        tc_fence_after();
                        issue_pv(t, j % C::STAGES, j > 1 ? 1u : 0u);
                        if (j + 2 >= n_iter) mma_commit_w(lead, &o_tile[t]);
                        mma_commit_w(lead, &v_empty[j % C::STAGES]);
                    }
                    if (it < n_iter) {
                        good = wait_k(it);
                        if (!good) break;
                        tc_fence_after();
                        issue_qk(0, t, it % C::STAGES);
                        mma_commit_w(lead, &k_empty[it % C::STAGES]);
                    }
                }
            }
            if (!good) {                           // release the write-back after a failed wait
                for (int t = 0; t < nt; ++t) mma_commit_w(lead, &o_tile[t]);
            }
            // every MMA has retired before TMEM is released
            for (int t = 0; t < nt; ++t) mbar_wait(&o_tile[t], 0, a.kv.err, VTX_KERR_O);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == C::MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Merges the splits: grid (n_tokens, ceil(Hq / 8 H)), a warp per H query heads, a
// lane per 4 dims; at most 32 splits, whose (m, l) the lanes read at once.
template <int D, int H>
__global__ void __launch_bounds__(256)
fa_paged_tile_combine_kernel(const PagedAttnArgs a, const PagedTile tl)
{
    grid_dep_wait();
    grid_dep_launch();
    const int t = blockIdx.x;
    const int b = paged_find(a.kv, t, threadIdx.x & 31);
    if (b >= a.kv.n_seq) return;
    const PagedSeq s = paged_seq(a.kv, b);
    const int tok = t - s.q0, served = min(s.n_new, a.kv.max_new);
    if (tok < 0 || tok >= served || paged_groups(served, a, tl) == 0) return;
    const int lane = threadIdx.x & 31, d = lane * 4, h0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * H;
    const int grp = tok / tl.tokens, n = paged_range(s, grp * tl.tokens, a, tl, true).n;
    if (n == 1 || h0 >= a.Hq) return;
    const long long step = (long long)a.kv.n_tokens * a.Hq, row = (long long)t * a.Hq + h0;
    float2 ml[H];
    bool on[H];                                    // heads whose item was cut
#pragma unroll
    for (int j = 0; j < H; ++j) {
        // whole items exist with one stream only, whose last group comes first
        on[j] = h0 + j < a.Hq && (paged_groups(served, a, tl) - 1 - grp) * a.kv.Hkv + (h0 + j) / a.G >= tl.whole;
        ml[j] = make_float2(-INFINITY, 0.f);
        if (on[j] && lane < n) ml[j] = reinterpret_cast<const float2 *>(tl.part_ml)[lane * step + row + j];
    }
    float top[H], f[H], l[H];
    float4 acc[H];
#pragma unroll
    for (int j = 0; j < H; ++j) {
        top[j] = ml[j].x;
#pragma unroll
        for (int o = 16; o; o >>= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
        f[j] = ml[j].x == -INFINITY ? 0.f : ex2(ml[j].x - top[j]);
        l[j] = f[j] * ml[j].y;
#pragma unroll
        for (int o = 16; o; o >>= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
        acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll (8 / H)
    for (int i = 0; i < n; ++i) {
        float4 v[H];
#pragma unroll
        for (int j = 0; j < H; ++j)
            v[j] = on[j] && d < D ? *reinterpret_cast<const float4 *>(tl.part_o + (i * step + row + j) * D + d)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < H; ++j) {
            const float w = __shfl_sync(0xffffffffu, f[j], i);
            acc[j].x = fmaf(w, v[j].x, acc[j].x); acc[j].y = fmaf(w, v[j].y, acc[j].y);
            acc[j].z = fmaf(w, v[j].z, acc[j].z); acc[j].w = fmaf(w, v[j].w, acc[j].w);
        }
    }
#pragma unroll
    for (int j = 0; j < H; ++j) {
        if (!on[j]) continue;
        const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
        if (d < D) {
            paged_store2(a, t, h0 + j, d, acc[j].x * inv, acc[j].y * inv);
            paged_store2(a, t, h0 + j, d + 2, acc[j].z * inv, acc[j].w * inv);
        }
        if (a.lse && lane == 0) a.lse[row + j] = l[j] == 0.f ? -INFINITY : (top[j] + log2f(l[j])) * kLn2;
    }
}

}  // namespace vtx
