// fa_paged.cuh — attention of ragged chunks of new tokens over a paged cache: what
// its kernels share, and the one for chunks over short Q8_0 caches (mma.sync): the
// decoder node of src/voxtral.cpp:1802 over pages.
//
//   x_ij = scale * q_i . k_j  (softcap c: c * tanh(x / c)),  j visible to i
//   O_i  = sum_j e^(x_ij - m_i) v_j / sum_j e^(x_ij - m_i)
//
// in one pass over the keys with the running maximum m and sum l of each row in
// registers.  Three kernels: few query rows per stream, bound by HBM
// (fa_paged_decode.cuh); chunks on the tensor core (fa_paged_sm100.cuh), over F16
// pages or over Q8_0 ones that paged_unpack_kernel has split into pairs of halves;
// and here chunks over short Q8_0 caches.  A CTA owns 64 query rows (row = token * G
// + head of the group, so every K/V row is read once for the whole group) of one KV
// head: 4 warps of 16 rows, tiles of 32 keys in shared memory.  K and V as their
// integers (exact halves): K's scales are applied to each block's f32 sum, V's to P
// before its one rounding to half, 64-fold so that a small scale keeps P out of the
// subnormals.  So only P (and a F32 q) is rounded.  Loads are not overlapped with
// the products: over the 95 keys at most that it is meant for there is little to
// overlap.  Chunks over longer caches come here too where their unpacked copy would
// be too large (vtx_paged.cu), and pay for it: 128 tokens at 14k keys 1630 us, 109 on
// the tensor-core kernel.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>
#include "vtx_ptx.cuh"
#include "paged_kv.cuh"
#include "fa_prefill_sm100.cuh"
#include "fa_decode_mma.cuh"

namespace vtx {

struct PagedAttnArgs {
    PagedView kv;
    const char *q; int q_f16; long long q_nbt, q_nbh;       // token and head strides (bytes)
    char *dst; int d_f16; long long d_nbt, d_nbh;
    float *lse;
    int Hq, G;
    float scale, softcap;                                   // logits: scale * s, or softcap * tanh(scale / softcap * s)
    int causal, window;
    int min_rows;             // streams with at most so many query rows per KV head are another kernel's
};

// Logit in log2 units of a dot product.
__device__ __forceinline__ float paged_logit(float s, float scale, float softcap) {
    return softcap != 0.0f ? softcap * kLog2e * tanhf(s * (scale / softcap)) : s * (scale * kLog2e);
}

// The same with the choice made by the instantiation (UF: softcap).
template <bool UF>
__device__ __forceinline__ float paged_logit_t(float s, float cx, float scale, float softcap) {
    return UF ? softcap * kLog2e * tanhf(s * (scale / softcap)) : s * cx;
}

// Two adjacent columns (d even) of a query row, rounded to half.
__device__ __forceinline__ uint32_t paged_q2(const char *row, int f16, int d) {
    if (f16) return *reinterpret_cast<const uint32_t *>(row + d * 2);
    const float2 x = *reinterpret_cast<const float2 *>(row + d * 4);
    return pack_half2(x.x, x.y);
}

// Scale of the Q8_0 block that holds column d of a cache row.
__device__ __forceinline__ float q8_scale(const char *row, int d) {
    return __half2float(*reinterpret_cast<const __half *>(row + (d >> 5) * 34));
}
// 8 consecutive values of a cache row as halves.  Q8_0: s * q rounded once,
// exact for s = 1 (the bare integers).
template <int KVT>
__device__ __forceinline__ uint4 paged_load8(const char *row, int d, float s) {
    if (KVT == 1) return *reinterpret_cast<const uint4 *>(row + d * 2);
    const unsigned short *w = reinterpret_cast<const unsigned short *>(row + (d >> 5) * 34 + 2 + (d & 31));
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned short u = w[i];
        r[i] = pack_half2(s * (float)(int8_t)(u & 0xff), s * (float)(int8_t)(u >> 8));
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// Four int8 of a word as two pairs of halves, exactly.
__device__ __forceinline__ void q8_halves(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
    w ^= 0x80808080u;
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), off);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
    lo = *reinterpret_cast<const uint32_t *>(&x);
    hi = *reinterpret_cast<const uint32_t *>(&y);
}
// Writes two adjacent columns of an output row.
__device__ __forceinline__ void paged_store2(const PagedAttnArgs &a, int tok, int head, int d, float x, float y) {
    char *p = a.dst + (long long)tok * a.d_nbt + (long long)head * a.d_nbh;
    if (a.d_f16) *reinterpret_cast<uint32_t *>(p + d * 2) = pack_half2(x, y);
    else *reinterpret_cast<float2 *>(p + d * 4) = make_float2(x, y);
}

constexpr float kLn2 = 0.6931471805599453f;

template <int D>
__global__ void __launch_bounds__(128)
fa_paged_q8_kernel(const PagedAttnArgs a)
{
    grid_dep_wait();
    grid_dep_launch();
    constexpr int KEYS = 32, P = D + 8, KC = D / 16, NB = D / 8;
    __shared__ __align__(16) __half ks[KEYS * P];
    __shared__ __align__(16) __half vs[KEYS * P];
    __shared__ float kd[D / 32][KEYS], vd[D / 32][KEYS];    // scales of K, 64 times V's
    const int b = blockIdx.z, g = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PagedSeq s = paged_seq(a.kv, b);
    if (blockIdx.x == 0 && s.n_new > a.kv.max_new) paged_report(a.kv, VTX_KERR_BOUND);
    const int rows = min(s.n_new, a.kv.max_new) * a.G;
    const int r_first = blockIdx.x * 64;
    if (r_first >= rows || rows <= a.min_rows) return;

    const int off = s.off;                                  // row of token 0
    int row[2], tok[2], lo[2], hi[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        row[u] = r_first + warp * 16 + (lane >> 2) + 8 * u;
        tok[u] = row[u] / a.G;
        hi[u] = row[u] < rows ? (a.causal ? min(off + tok[u], s.len - 1) : s.len - 1) : -1;
        lo[u] = a.window > 0 ? off + tok[u] - a.window + 1 : 0;
    }
    const int t_first = r_first / a.G, t_last = (min(r_first + 64, rows) - 1) / a.G;
    const int k_hi = a.causal ? min(off + t_last, s.len - 1) : s.len - 1;
    const int k_lo = a.window > 0 ? max(0, off + t_first - a.window + 1) : 0;

    uint32_t qa[KC][4];
    {
        const char *q0 = a.q + (long long)(s.q0 + tok[0]) * a.q_nbt + (long long)(g * a.G + row[0] % a.G) * a.q_nbh;
        const char *q1 = a.q + (long long)(s.q0 + tok[1]) * a.q_nbt + (long long)(g * a.G + row[1] % a.G) * a.q_nbh;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            const int c = kc * 16 + 2 * (lane & 3);
            qa[kc][0] = row[0] < rows ? paged_q2(q0, a.q_f16, c) : 0u;
            qa[kc][1] = row[1] < rows ? paged_q2(q1, a.q_f16, c) : 0u;
            qa[kc][2] = row[0] < rows ? paged_q2(q0, a.q_f16, c + 8) : 0u;
            qa[kc][3] = row[1] < rows ? paged_q2(q1, a.q_f16, c + 8) : 0u;
        }
    }
    float o[NB][4];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int lrow = lane & 7, lmat = lane >> 3;

    for (int k0 = k_lo & ~(KEYS - 1); k0 <= k_hi; k0 += KEYS) {
        __syncthreads();
        for (int i = threadIdx.x; i < KEYS * (D / 8); i += 128) {
            const int r = i / (D / 8), c = (i % (D / 8)) * 8;
            uint4 kx = make_uint4(0u, 0u, 0u, 0u), vx = kx;
            if (k0 + r >= k_lo && k0 + r <= k_hi) {         // other rows may hold anything: zeros instead
                const long long at = paged_row(a.kv, b, k0 + r, g);
                kx = paged_load8<8>(a.kv.k + at, c, 1.0f);
                vx = paged_load8<8>(a.kv.v + at, c, 1.0f);
            }
            if ((c & 31) == 0) {
                const bool in = k0 + r >= k_lo && k0 + r <= k_hi;
                const long long at = in ? paged_row(a.kv, b, k0 + r, g) : 0;
                kd[c >> 5][r] = in ? q8_scale(a.kv.k + at, c) : 0.f;
                vd[c >> 5][r] = in ? 64.0f * q8_scale(a.kv.v + at, c) : 0.f;
            }
            *reinterpret_cast<uint4 *>(ks + r * P + c) = kx;
            *reinterpret_cast<uint4 *>(vs + r * P + c) = vx;
        }
        __syncthreads();
        float x[KEYS / 8][4];
#pragma unroll
        for (int nt = 0; nt < KEYS / 8; ++nt) {
            x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
#pragma unroll
            for (int kc = 0; kc < KC; kc += 2) {
                uint32_t bk[4];
                ldsm_x4(bk, ks + (nt * 8 + lrow) * P + kc * 16 + lmat * 8);
                // a block of 32 dims, then its scale
                float y[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816(y, qa[kc], bk[0], bk[1]);
                mma16816(y, qa[kc + 1], bk[2], bk[3]);
                const float2 d = *reinterpret_cast<const float2 *>(&kd[kc / 2][nt * 8 + 2 * (lane & 3)]);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[nt][i] = fmaf(i & 1 ? d.y : d.x, y[i], x[nt][i]);
            }
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int nt = 0; nt < KEYS / 8; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int u = i >> 1, key = k0 + nt * 8 + 2 * (lane & 3) + (i & 1);
                x[nt][i] = key >= lo[u] && key <= hi[u] ? paged_logit(x[nt][i], a.scale, a.softcap) : -INFINITY;
                mx[u] = fmaxf(mx[u], x[nt][i]);
            }
        float mu[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
            mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2));
            const float mn = fmaxf(m[u], mx[u]);
            mu[u] = mn == -INFINITY ? 0.f : mn;
            const float al = ex2(m[u] - mu[u]);
            m[u] = mn;
            l[u] *= al;
#pragma unroll
            for (int i = 0; i < NB; ++i) { o[i][2 * u] *= al; o[i][2 * u + 1] *= al; }
        }
#pragma unroll
        for (int nt = 0; nt < KEYS / 8; ++nt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[nt][i] = ex2(x[nt][i] - mu[i >> 1]);
            l[0] += x[nt][0] + x[nt][1];
            l[1] += x[nt][2] + x[nt][3];
        }
#pragma unroll
        for (int kk = 0; kk < KEYS / 16; ++kk)
#pragma unroll
            for (int nb = 0; nb < NB; nb += 4) {            // a block of 32 dims: its scales go into P
                uint32_t pa[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 d = *reinterpret_cast<const float2 *>(&vd[nb / 4][kk * 16 + h * 8 + 2 * (lane & 3)]);
                    const float *p = x[kk * 2 + h];
                    pa[2 * h] = pack_half2(p[0] * d.x, p[1] * d.y);
                    pa[2 * h + 1] = pack_half2(p[2] * d.x, p[3] * d.y);
                }
#pragma unroll
                for (int n2 = nb; n2 < nb + 4; n2 += 2) {
                    uint32_t bv[4];
                    ldsm_x4_t(bv, vs + (kk * 16 + (lmat & 1) * 8 + lrow) * P + n2 * 8 + (lmat >> 1) * 8);
                    mma16816(o[n2], pa, bv[0], bv[1]);
                    mma16816(o[n2 + 1], pa, bv[2], bv[3]);
                }
            }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
        if (row[u] >= rows) continue;
        const float inv = l[u] == 0.f ? 0.f : 0.015625f / l[u];
        const int head = g * a.G + row[u] % a.G, t = s.q0 + tok[u];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
            paged_store2(a, t, head, nb * 8 + 2 * (lane & 3), o[nb][2 * u] * inv, o[nb][2 * u + 1] * inv);
        if (a.lse && (lane & 3) == 0)
            a.lse[(long long)t * a.Hq + head] = l[u] == 0.f ? -INFINITY : (m[u] + log2f(l[u])) * kLn2;
    }
}

// 8 values at 2-byte aligned shared memory as exact halves.
__device__ __forceinline__ void q8_lds8(const char *p, uint32_t (&h)[4]) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3));
    const uint32_t sh = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 2) * 8;
    const uint32_t x = w[0], y = w[1], z = sh ? w[2] : 0u;
    q8_halves(__funnelshift_r(x, y, sh), h[0], h[1]);
    q8_halves(__funnelshift_r(y, z, sh), h[2], h[3]);
}

// Copies the Q8_0 pages of the streams that bring more than a.min_rows query rows
// into pages of 128 keys in `out` (stream s, page p: page s * out.max_pages + p).  A
// value d * q of 18 bits becomes hi = it rounded to half and lo = the rest, exact
// down to 2^-25; 64 rows of hi, then the same keys' 64 rows of lo, so that a tile of
// 128 rows is a product over hi and lo at once.  (hi alone halves the products, but
// its rounding of V doubles the output's squared error and K's grows with the
// logits: 2.2 times the error of an F32 computation rounded to half at 1400 keys,
// with lo 1.2 times.)  272 bytes read and 1024 written per row and KV head, next to
// 8 * 128 flops per query row for each of those rows.
// Grid (32-row ranges, Hkv, n_seq), 128 threads.
template <int D>
__global__ void __launch_bounds__(128)
paged_unpack_kernel(const PagedAttnArgs a, const PagedView out)
{
    grid_dep_wait();
    grid_dep_launch();
    constexpr int ROW = D / 32 * 34;
    __shared__ __align__(16) char raw[2 * 32 * ROW];
    const int b = blockIdx.z, g = blockIdx.y, r0 = blockIdx.x * 32;
    const PagedSeq s = paged_seq(a.kv, b);
    const int end = min(s.len, out.cap);
    const int lo = a.window > 0 ? s.off - a.window + 1 : 0;
    if (s.n_new * a.G <= a.min_rows || r0 >= end || r0 + 32 <= lo) return;
    // groups of 16 rows are contiguous in a page
    constexpr int CH = 16 * ROW / 16;
    for (int i = threadIdx.x; i < 4 * CH; i += 128) {
        const int grp = i / CH, r = r0 + (grp & 1) * 16;
        if (r >= end || r + 16 <= lo) continue;
        const char *src = (grp < 2 ? a.kv.k : a.kv.v) + paged_row(a.kv, b, r, g);
        reinterpret_cast<uint4 *>(raw)[i] = reinterpret_cast<const uint4 *>(src)[i % CH];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * 32 * (D / 8); i += 128) {
        const int sel = i / (32 * (D / 8)), r = i / (D / 8) % 32, c = i % (D / 8);
        const int grp = r0 + (r & 16);
        if (grp >= end || grp + 16 <= lo) continue;
        const char *blk = raw + (sel * 32 + r) * ROW + (c >> 2) * 34;
        const __half d = *reinterpret_cast<const __half *>(blk);
        uint32_t h[4];
        q8_lds8(blk + 2 + (c & 3) * 8, h);
        const __half2 d2 = __half2half2(d);
        uint32_t rest[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __half2 q = *reinterpret_cast<const __half2 *>(&h[j]);
            const __half2 x = __hmul2(q, d2), y = __hfma2(q, d2, __hneg2(x));
            h[j] = *reinterpret_cast<const uint32_t *>(&x);
            rest[j] = *reinterpret_cast<const uint32_t *>(&y);
        }
        const int row = r0 + r;
        char *dst = (sel ? out.v : out.k) + (long long)paged_page(out, b, row) * out.nb3 + (long long)g * out.nb2 +
                    (long long)((row & 64) * 2 + (row & 63)) * out.nb1 + c * 16;
        *reinterpret_cast<uint4 *>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(dst + 64 * out.nb1) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
    }
}

}  // namespace vtx
