// kv_score_sm100.cuh — accumulated attention weight of many query rows on the
// tensor core (F16 q): kv_score.cuh's sum with the product turned
// round, S^T = K Q^T, so that a key is a TMEM lane and its thread adds up its
// own row of weights; nothing crosses threads.
//
// A CTA owns NT key tiles of 128 of one stream and KV head (A operands, loaded
// once) and walks the query rows 128 at a time (the B operand, T = 128 / G
// tokens, a ring of two tiles).  Four warpgroups: one per key tile (NT = 4), or
// two with half of the columns each (NT = 2, whose S^T is double-buffered); 4 x
// 128 TMEM columns either way, so the tensor core works ahead of the
// exponentials, which bound the kernel: 128 x 128 per tile at 16 a clock and SM.
// Every CTA of a head reads all of its Q from L2, so more key tiles per CTA are
// faster once the CTAs fill the GPU: 500 tokens x 16000 keys x 32 heads take 102
// us with four, 116 us with two (58 us of exponentials).  A degree-5 polynomial
// on the FMA pipe for 1/8, 1/4 or 1/2 of the exponentials: 100, 101, 114 us, so
// not kept.
// A column's -lse and last visible row are staged; (-inf, -1) makes a column
// count nothing (rows past the tokens, or T * G < 128).
// Q8_0: a K tile is made once by the threads, as two halves per value, d * q
// rounded and what that lost; two products per tile then carry about 22 bits of K
// (one rounded half would move a weight by 2^-12), and the tensor core has the
// time, since the exponentials bound the kernel.
// Key rows that do not exist or that nobody sees only affect their own lane.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "vtx_ptx.cuh"
#include "paged_kv.cuh"
#include "kv_score.cuh"
#include "fa_prefill_sm100.cuh"

namespace vtx {

template <int D, int KVT, int NT> struct ScoreTileCfg {
    static constexpr int SUB = D / 64, TILE = 128 * D * 2, STAGES = 2;
    static constexpr int PER = 4 / NT;             // warpgroups and TMEM buffers per key tile
    static constexpr int K_TILES = KVT == 1 ? NT : 2 * NT;             // Q8_0: high and low parts
    static constexpr int K_OFF = 0, Q_OFF = K_TILES * TILE;
    static constexpr int LSE_OFF = Q_OFF + STAGES * TILE;              // per stage: -lse, last visible row
    static constexpr int LSTAGES = 4;
    static constexpr int SUM_OFF = LSE_OFF + LSTAGES * 1024, BAR_OFF = SUM_OFF + 1024;
    static constexpr int NBARS = 2 + 2 * STAGES + 2 * LSTAGES + 8;
    static constexpr int SMEM = BAR_OFF + NBARS * 8 + 16 + 1024;
    static constexpr int NTHREADS = 608, TMA_WARP = 16, MMA_WARP = 17, LSE_WARP = 18;
};

// Grid (key ranges of 128 NT, Hkv, n_seq).
template <int D, int KVT, int NT, bool UF>
__global__ void __launch_bounds__(ScoreTileCfg<D, KVT, NT>::NTHREADS, 1)
kv_score_sm100_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmQ,
                      const PagedScoreArgs a, int T)
{
    using C = ScoreTileCfg<D, KVT, NT>;
    extern __shared__ __align__(1024) char smem_raw[];
    char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *k_full = reinterpret_cast<uint64_t *>(smem + C::BAR_OFF);
    uint64_t *q_full = k_full + 1;                 // [STAGES] the Q tile landed
    uint64_t *q_empty = q_full + C::STAGES;        // [STAGES] its products are done
    uint64_t *l_full = q_empty + C::STAGES;        // [LSTAGES] its columns' lse is staged
    uint64_t *l_empty = l_full + C::LSTAGES;       // [LSTAGES] ... and read
    uint64_t *s_full = l_empty + C::LSTAGES;       // [tile][buffer]
    uint64_t *s_free = s_full + 4;
    uint64_t *mma_done = s_free + 4;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_done + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = blockIdx.z, g = blockIdx.y;
    if (tid == 0) {
        mbar_init(k_full, KVT == 1 ? 1 : 16);      // the TMA lane, or the warps that make K
        mbar_init(mma_done, 1);
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < C::LSTAGES; ++i) {
            mbar_init(&l_full[i], 1);
            mbar_init(&l_empty[i], 16);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_free[i], 4 * C::PER);
        }
        fence_mbar_init();
    }
    grid_dep_wait();
    grid_dep_launch();
    const PagedSeq s = paged_seq(a.kv, b);
    const int limit = min(s.len, a.row_cap);
    if (blockIdx.x == 0 && tid == 0 && s.len > min(a.row_cap, a.kv.max_kv)) paged_report(a.kv, VTX_KERR_BOUND);
    const int k0 = blockIdx.x * 128 * NT;
    if (k0 >= limit) return;
    const int off = s.off;
    const int ta = a.observe > 0 ? max(0, s.n_new - a.observe) : 0;     // first token that counts
    const int lo_any = ta < s.n_new ? (a.window > 0 ? max(0, off + ta - a.window + 1) : 0) : limit;
    int t0 = ta, t1 = s.n_new;
    if (a.causal) t0 = max(t0, k0 - off);                               // earlier tokens see none of these keys
    if (a.window > 0) t1 = (int)min((long long)t1, (long long)k0 + 128 * NT - 1 + a.window - off);
    const int n_iter = t1 > t0 ? (t1 - t0 + T - 1) / T : 0;
    const int TG = T * a.G;

    if (warp == C::MMA_WARP) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    // columns no token fills stay zero: their -lse is -inf
    for (int i = tid; i < C::STAGES * (128 - TG) * C::SUB * 8; i += C::NTHREADS) {
        const int ch = i & 7, r = TG + (i >> 3) % (128 - TG), u = (i >> 3) / (128 - TG);
        *reinterpret_cast<uint4 *>(smem + C::Q_OFF + (u / C::SUB) * C::TILE + (u % C::SUB) * 16384 + r * 128 + ch * 16) =
            make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp < 16) {
        // =================== a thread per key (and half of the columns) ========
        constexpr int COLS = 128 / C::PER;
        const int half = warp / (4 * NT), kt = tid & (128 * NT - 1);    // kt = 128 tile + TMEM lane
        const int t = kt >> 7, key = k0 + kt;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const long long e = ((long long)b * a.kv.Hkv + g) * a.row_cap + key;
        const float old = half == 0 && key < limit && a.decay != 0.f ? a.decay * a.score[e] : 0.f;
        if constexpr (KVT == 8) {
            if (n_iter > 0) {
                for (int i = tid; i < NT * 128 * (D / 8); i += 512) {
                    const int r = i / (D / 8), c = i % (D / 8), ky = k0 + r;
                    if (ky >= limit || ky < lo_any) continue;           // affects its own lane only
                    const char *row = a.kv.k + paged_row(a.kv, b, ky, g);
                    const float d = q8_scale(row, c * 8);
                    const unsigned short *w = reinterpret_cast<const unsigned short *>(row + (c >> 2) * 34 + 2 + (c & 3) * 8);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float x = d * (float)(int8_t)(w[j] & 0xff), y = d * (float)(int8_t)(w[j] >> 8);
                        hi[j] = pack_half2(x, y);
                        const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi[j]));
                        lo[j] = pack_half2(x - h.x, y - h.y);
                    }
                    char *dst = smem + C::K_OFF + (r >> 7) * C::TILE + (c >> 3) * 16384 + (r & 127) * 128 +
                                (((c & 7) ^ (r & 7)) << 4);
                    *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4 *>(dst + NT * C::TILE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full);
            }
        }
        const float cx = a.scale * kLog2e;
        const unsigned reach = a.window > 0 ? (unsigned)a.window : 0x80000000u;
        float sum = 0.f;
        for (int it = 0; it < n_iter; ++it) {
            const int st = it % C::LSTAGES, buf = t * C::PER + it % C::PER;
            ok = __all_sync(0xffffffffu, mbar_wait(&s_full[buf], (it / C::PER) & 1, a.kv.err, VTX_KERR_S));
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&l_full[st], (it / C::LSTAGES) & 1, a.kv.err, VTX_KERR_Q));
            if (!ok) break;
            tc_fence_after();
            const float *ls = reinterpret_cast<const float *>(smem + C::LSE_OFF + st * 1024) + half * COLS;
            const int *pos = reinterpret_cast<const int *>(ls + 128);
            // every column is a token, and sees every key of this warp
            const int tok = t0 + it * T, kw = k0 + (kt & ~31);
            const bool inner = tok + T <= t1 && (!a.causal || kw + 31 <= off + tok) &&
                               (a.window == 0 || kw > off + min(tok + T, t1) - 1 - a.window);
            uint64_t acc[2] = {0ull, 0ull};
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) {
                uint32_t raw[32];
                tmem_ld32(tmem + lane_base + buf * 128 + half * COLS + c * 32, raw);
                tmem_ld_wait();
                if (c == COLS / 32 - 1) {                               // this warp has read its part of S
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[buf]);
                }
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 l = *reinterpret_cast<const float4 *>(ls + c * 32 + i);
                    float x[4];
                    if (UF) {
                        x[0] = paged_logit(__uint_as_float(raw[i]), a.scale, a.softcap) + l.x;
                        x[1] = paged_logit(__uint_as_float(raw[i + 1]), a.scale, a.softcap) + l.y;
                        x[2] = paged_logit(__uint_as_float(raw[i + 2]), a.scale, a.softcap) + l.z;
                        x[3] = paged_logit(__uint_as_float(raw[i + 3]), a.scale, a.softcap) + l.w;
                    } else {
                        upk2(ffma2(pk2(__uint_as_float(raw[i]), __uint_as_float(raw[i + 1])), pk2(cx, cx), pk2(l.x, l.y)),
                             x[0], x[1]);
                        upk2(ffma2(pk2(__uint_as_float(raw[i + 2]), __uint_as_float(raw[i + 3])), pk2(cx, cx), pk2(l.z, l.w)),
                             x[2], x[3]);
                    }
                    if (!inner) {                                       // visible: 0 <= pos - key < window
                        const int4 p = *reinterpret_cast<const int4 *>(pos + c * 32 + i);
                        x[0] = (unsigned)(p.x - key) < reach ? x[0] : -INFINITY;
                        x[1] = (unsigned)(p.y - key) < reach ? x[1] : -INFINITY;
                        x[2] = (unsigned)(p.z - key) < reach ? x[2] : -INFINITY;
                        x[3] = (unsigned)(p.w - key) < reach ? x[3] : -INFINITY;
                    }
                    acc[0] = fadd2(acc[0], pk2(ex2(x[0]), ex2(x[1])));
                    acc[1] = fadd2(acc[1], pk2(ex2(x[2]), ex2(x[3])));
                }
            }
            if (lane == 0) mbar_arrive(&l_empty[st]);
            float y0, y1;
            upk2(fadd2(acc[0], acc[1]), y0, y1);
            sum += y0 + y1;
        }
        if constexpr (C::PER == 2) {                                    // the halves' sums meet in shared memory
            float *part = reinterpret_cast<float *>(smem + C::SUM_OFF);
            if (half == 1) part[kt] = sum;
            asm volatile("bar.sync 1, 512;" ::: "memory");
            if (half == 0) sum += part[kt];
        }
        if (half == 0 && key < limit) a.score_out[e] = old + (key >= lo_any ? sum : 0.f);
    } else if (warp == C::TMA_WARP) {
        // =================== TMA: the K tiles, then Q tile by tile =========
        if (n_iter > 0) {
            if constexpr (KVT == 1) {
                // boxes of a half-width tile row range: 16 a tile at most, two tiles a round
                const int rows_box = min(128, 1 << a.kv.shift), per = 128 / rows_box * C::SUB;
                unsigned need = 0;                     // bit u: this lane's box of round u is loaded
                int n = 0;
#pragma unroll
                for (int u = 0; u < NT / 2; ++u) {
                    const int j = lane / per, y = k0 + (2 * u + j) * 128 + (lane % per) / C::SUB * rows_box;
                    const bool on = j < 2 && y < limit && y + rows_box > lo_any;
                    n += __popc(__ballot_sync(0xffffffffu, on));
                    need |= (unsigned)on << u;
                }
                if (lane == 0) mbar_arrive_expect_tx(k_full, (uint32_t)(n * rows_box * 128));
                __syncwarp();
#pragma unroll
                for (int u = 0; u < NT / 2; ++u) {
                    const int j = 2 * u + lane / per, r = (lane % per) / C::SUB * rows_box, sub = lane % C::SUB;
                    if ((need >> u) & 1u)
                        tma_load_4d(smem + C::K_OFF + j * C::TILE + sub * 16384 + r * 128, &tmK, k_full, sub * 64,
                                    (k0 + j * 128 + r) & ((1 << a.kv.shift) - 1), g,
                                    max(paged_page(a.kv, b, k0 + j * 128 + r), 0));
                }
                __syncwarp();
            }
            int issued = 0;
            if (lane == 0) {
                for (int it = 0; it < n_iter; ++it) {
                    const int st = it % C::STAGES;
                    if (it >= C::STAGES && !mbar_wait(&q_empty[st], ((it / C::STAGES) - 1) & 1, a.kv.err, VTX_KERR_Q)) break;
                    issued = it + 1;
                    mbar_arrive_expect_tx(&q_full[st], (uint32_t)(C::SUB * TG * 128));
#pragma unroll
                    for (int u = 0; u < C::SUB; ++u)
                        tma_load_4d(smem + C::Q_OFF + st * C::TILE + u * 16384, &tmQ, &q_full[st], u * 64, g * a.G,
                                    s.q0 + t0 + it * T, 0);
                }
                // everything must have landed before shared memory is released
                mbar_wait(k_full, 0, a.kv.err, VTX_KERR_KV);
                for (int it = max(0, issued - C::STAGES); it < issued; ++it)
                    mbar_wait(&q_full[it % C::STAGES], (it / C::STAGES) & 1, a.kv.err, VTX_KERR_Q);
            }
            __syncwarp();
        }
    } else if (warp == C::LSE_WARP) {
        // =================== lse and row position of a tile's columns ==========
        float next[4];
        auto load = [&](int it) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = lane + 32 * i, tok = t0 + it * T + r / a.G;
                next[i] = -INFINITY;                                    // minus lse in log2 units
                if (it < n_iter && r < TG && tok < t1) {
                    const float x = a.lse[(long long)(s.q0 + tok) * a.Hq + g * a.G + r % a.G];
                    next[i] = x == -INFINITY ? x : -x * kLog2e;
                }
            }
        };
        load(0);
        for (int it = 0; it < n_iter; ++it) {
            const int st = it % C::LSTAGES;
            if (it >= C::LSTAGES &&
                !__all_sync(0xffffffffu, mbar_wait(&l_empty[st], ((it / C::LSTAGES) - 1) & 1, a.kv.err, VTX_KERR_Q)))
                break;
            float *ls = reinterpret_cast<float *>(smem + C::LSE_OFF + st * 1024);
            int *pos = reinterpret_cast<int *>(ls + 128);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ls[lane + 32 * i] = next[i];
                // the last row this column's token sees; none where it counts nothing
                const int p = a.causal ? off + t0 + it * T + (lane + 32 * i) / a.G : s.len - 1;
                pos[lane + 32 * i] = next[i] == -INFINITY ? -1 : p;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&l_full[st]);
            load(it + 1);
        }
    } else if (warp == C::MMA_WARP && n_iter > 0) {
        // =================== MMA issuer =========================================
        const uint32_t lead = elect_one();
        constexpr uint32_t IDESC = idesc_f16_f32(128, 128, 0, 0);
        constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);       // SBO 1024, v1, 128-byte swizzle
        const uint32_t sbase = smem_u32(smem);
        const uint32_t lo_k = ((sbase + C::K_OFF) >> 4) | (1u << 16), lo_q = ((sbase + C::Q_OFF) >> 4) | (1u << 16);
        constexpr uint32_t T16 = C::TILE >> 4;
        bool good = __all_sync(0xffffffffu, mbar_wait(k_full, 0, a.kv.err, VTX_KERR_KV));
        for (int it = 0; it < n_iter && good; ++it) {
            const int st = it % C::STAGES;
            good = __all_sync(0xffffffffu, mbar_wait(&q_full[st], (it / C::STAGES) & 1, a.kv.err, VTX_KERR_Q));
            for (int t = 0; t < NT && good; ++t) {
                const int buf = t * C::PER + it % C::PER;
                if (it >= C::PER)
                    good = __all_sync(0xffffffffu,
                                      mbar_wait(&s_free[buf], ((it / C::PER) - 1) & 1, a.kv.err, VTX_KERR_S));
                if (!good) break;
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t ko = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
                    mma_f16_ss_w(lead, tmem + buf * 128, desc64(lo_k + t * T16 + ko, HI), desc64(lo_q + st * T16 + ko, HI),
                                 IDESC, kk > 0);
                    if constexpr (KVT == 8)
                        mma_f16_ss_w(lead, tmem + buf * 128, desc64(lo_k + (NT + t) * T16 + ko, HI),
                                     desc64(lo_q + st * T16 + ko, HI), IDESC, 1);
                }
                mma_commit_w(lead, &s_full[buf]);
            }
            mma_commit_w(lead, &q_empty[st]);
        }
        mma_commit_w(lead, mma_done);                                         // all retired before TMEM is released
        mbar_wait(mma_done, 0, a.kv.err, VTX_KERR_S);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == C::MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace vtx
