// vtx_paged.cu — C ABI entry points of the paged decoder cache: append,
// attention over ragged chunks, accumulated attention weight, eviction.
// Operand checks, launch geometry and workspace accounting; nothing here
// allocates, synchronises or aborts.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "../../include/vtx_fa.h"
#include "vtx_ptx.cuh"
#include "vtx_host.cuh"
#include "fa_prefill_sm100.cuh"
#include "paged_kv.cuh"
#include "fa_paged.cuh"
#include "fa_paged_decode.cuh"
#include "fa_paged_sm100.cuh"
#include "kv_score.cuh"
#include "kv_score_sm100.cuh"
#include "kv_evict.cuh"

using namespace vtx;

namespace {

constexpr int kMaxGroup = 16;             // query heads per KV head

int check_pool(const vtx_tensor &t, int row) {
    if (!t.data) return VTX_ERR_NULL;
    if (t.nb[1] < (size_t)row || (t.ne[2] > 1 && !t.nb[2]) || (t.ne[3] > 1 && !t.nb[3])) return VTX_ERR_STRIDE;
    if (reinterpret_cast<uintptr_t>(t.data) % 16 || t.nb[2] % 16 || t.nb[3] % 16) return VTX_ERR_STRIDE;
    if (t.type == VTX_TYPE_Q8_0) return t.nb[0] == 34 && t.nb[1] == (size_t)row ? VTX_OK : VTX_ERR_STRIDE;
    return t.nb[0] == 2 && t.nb[1] % 16 == 0 ? VTX_OK : VTX_ERR_STRIDE;
}

// Sizes and strides of a paged cache, as every call needs them.
int check_paged(const vtx_paged_kv *p) {
    if (!p) return VTX_ERR_NULL;
    const vtx_tensor &k = p->k, &v = p->v;
    if (k.type != v.type || (k.type != VTX_TYPE_F16 && k.type != VTX_TYPE_Q8_0)) return VTX_ERR_TYPE;
    for (int i = 0; i < 4; ++i)
        if (k.ne[i] != v.ne[i] || k.ne[i] < 1) return VTX_ERR_SHAPE;
    if (k.ne[0] != 64 && k.ne[0] != 128) return VTX_ERR_UNSUPPORTED;
    if (k.ne[1] < 16 || k.ne[1] > 256 || (k.ne[1] & (k.ne[1] - 1))) return VTX_ERR_UNSUPPORTED;
    if (k.ne[2] > 65535 || k.ne[3] > INT32_MAX) return VTX_ERR_SHAPE;
    if (p->n_seq < 0 || p->n_seq > 65535 || p->max_pages < 0 || p->n_tokens < 0 || p->max_new < 0 ||
        p->max_kv_len < 0)
        return VTX_ERR_SHAPE;
    if ((long long)p->max_pages * k.ne[1] > INT32_MAX || p->n_tokens > (1 << 24)) return VTX_ERR_SHAPE;
    if (p->max_kv_len > (long long)p->max_pages * k.ne[1] || p->max_new > p->n_tokens) return VTX_ERR_SHAPE;
    for (int i = 1; i < 4; ++i)
        if (k.nb[i] != v.nb[i] || k.nb[i] >= (1ULL << 40)) return VTX_ERR_STRIDE;
    const int row = row_bytes(k.type, k.ne[0]);
    int rc = check_pool(k, row);
    if (rc == VTX_OK) rc = check_pool(v, row);
    if (rc != VTX_OK) return rc;
    if (p->n_seq > 0 && (!p->kv_len || (p->max_pages > 0 && !p->page_table))) return VTX_ERR_NULL;
    return VTX_OK;
}

PagedView view_of(const vtx_paged_kv *p, const DeviceState *ds) {
    PagedView v{};
    v.k = static_cast<char *>(p->k.data);
    v.v = static_cast<char *>(p->v.data);
    v.nb1 = (long long)p->k.nb[1]; v.nb2 = (long long)p->k.nb[2]; v.nb3 = (long long)p->k.nb[3];
    v.table = p->page_table; v.kv_len = p->kv_len; v.q_start = p->q_start;
    v.n_seq = p->n_seq; v.n_tokens = p->n_tokens; v.max_new = p->max_new; v.max_kv = p->max_kv_len;
    v.max_pages = p->max_pages; v.n_pages = (int)p->k.ne[3];
    while ((1 << v.shift) < (int)p->k.ne[1]) ++v.shift;
    v.cap = v.max_pages << v.shift;
    v.Hkv = (int)p->k.ne[2];
    v.err = ds->err;
    return v;
}

// q [D, n_tokens, Hq, 1] of the attention and score calls.
int check_q(const vtx_paged_kv *p, const vtx_tensor *q) {
    if (!q) return VTX_ERR_NULL;
    if (q->type != VTX_TYPE_F32 && q->type != VTX_TYPE_F16) return VTX_ERR_TYPE;
    if (q->ne[0] != p->k.ne[0] || q->ne[1] != p->n_tokens || q->ne[3] != 1) return VTX_ERR_SHAPE;
    if (q->ne[2] < 1 || q->ne[2] % p->k.ne[2]) return VTX_ERR_SHAPE;
    if (q->ne[2] / p->k.ne[2] > kMaxGroup) return VTX_ERR_UNSUPPORTED;
    if (q->nb[0] != (size_t)elem_size(q->type)) return VTX_ERR_STRIDE;
    if (p->n_tokens == 0) return VTX_OK;
    if (!q->data || !p->q_start) return VTX_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(q->data) % 16 || q->nb[1] % 16 || q->nb[2] % 16) return VTX_ERR_STRIDE;
    if (q->nb[1] >= (1ULL << 40) || q->nb[2] >= (1ULL << 40)) return VTX_ERR_STRIDE;
    return VTX_OK;
}

int check_params(const vtx_fa_params *p) {
    if (!p) return VTX_ERR_NULL;
    if (p->window < 0 || (p->window > 0 && !p->causal) || p->max_bias != 0.0f) return VTX_ERR_UNSUPPORTED;
    if (!std::isfinite(p->scale) || !std::isfinite(p->logit_softcap)) return VTX_ERR_UNSUPPORTED;
    return VTX_OK;
}

// Allows a kernel its shared memory, once per device (`done`: one flag each).
template <typename K>
int allow_smem(K kernel, int bytes, std::atomic<int> (&done)[kMaxDevices]) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (done[dev].load(std::memory_order_acquire)) return VTX_OK;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
        return VTX_ERR_CUDA;
    done[dev].store(1, std::memory_order_release);
    return VTX_OK;
}

int current_sms() {
    int sms = 148, dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cudaGetLastError();
    return sms;
}

// Streams of at most kFewRows query rows per KV head go to the streaming kernel.
constexpr int kFewRows = 16;

struct DecodePlan {
    bool use;                 // the streaming kernel is launched
    int rows;                 // its row count, 8 or 16
    PagedSplit split;
    size_t o_bytes, bytes;    // partial O, with (m, l)
};

// Splits over (streams x KV heads): one wave of three CTAs per SM for one stream,
// or where two would leave fewer than 40 tiles each (8 streams of 4000: 39.8 -> 30.2
// us); else two, which spreads ragged lengths more evenly; at most 128 tiles (2048
// keys) each, and at least one tile per warp.
DecodePlan plan_decode(const vtx_paged_kv *p, int G, int sms) {
    DecodePlan d{};
    // the only stream may bring more tokens than fit: then all go one way
    d.use = p->max_new * (long long)G <= kFewRows || p->n_seq > 1;
    if (!d.use || G > kFewRows || p->n_seq == 0) {
        d.use = false;
        return d;
    }
    d.rows = p->max_new * (long long)G <= 8 ? 8 : 16;
    const long long base = (long long)p->n_seq * p->k.ne[2];
    const int tiles = std::max(1, (p->max_kv_len + 15) / 16);
    long long want = (6LL * sms + base - 1) / base;
    if (p->n_seq == 1 || tiles < 40 * want) want = 3LL * sms / base;
    want = std::max<long long>(std::max<long long>(want, 1), (tiles + 127) / 128);
    want = std::min<long long>(want, (tiles + 3) / 4);
    d.split.n_splits = (int)want;
    d.split.tiles = (int)((tiles + want - 1) / want);
    if (want > 1) {
        const size_t rows = (size_t)base * want * d.rows;
        d.o_bytes = align_up(rows * p->k.ne[0] * 4, 256);
        d.bytes = d.o_bytes + align_up(rows * 8, 256);
    }
    return d;
}

// The attention workspace begins with the arrival counters of the streaming kernel's
// splits, a word per stream and KV head, at least kArrivals of them whatever the plan:
// nothing else is ever put there, so they stay zero between calls of any sizes.
constexpr size_t kArrivals = 65536;

size_t arrival_bytes(const vtx_paged_kv *p, size_t rest) {
    return rest ? align_up(std::max((size_t)p->n_seq * (size_t)p->k.ne[2], kArrivals) * 4, 256) : 0;
}

template <int D, int KVT, int ROWS, bool UF>
int launch_decode(const PagedAttnArgs &a, const PagedSplit &sp, cudaStream_t st) {
    using C = PagedDecodeCfg<D, KVT>;
    static std::atomic<int> done[kMaxDevices];
    int rc = allow_smem(fa_paged_decode_kernel<D, KVT, ROWS, UF>, C::SMEM, done);
    if (rc != VTX_OK) return rc;
    const long long ctas = (long long)a.kv.n_seq * a.kv.Hkv * sp.n_splits;
    if (ctas > 0x7fffffffLL) return VTX_ERR_UNSUPPORTED;
    return launch_pdl(fa_paged_decode_kernel<D, KVT, ROWS, UF>, dim3((unsigned)ctas), dim3(128), C::SMEM, st, a, sp);
}

template <int D, int KVT>
int launch_decode_rows(const PagedAttnArgs &a, const DecodePlan &d, cudaStream_t st) {
    if (a.softcap != 0.0f)
        return d.rows == 8 ? launch_decode<D, KVT, 8, true>(a, d.split, st)
                           : launch_decode<D, KVT, 16, true>(a, d.split, st);
    return d.rows == 8 ? launch_decode<D, KVT, 8, false>(a, d.split, st)
                       : launch_decode<D, KVT, 16, false>(a, d.split, st);
}

template <int D>
int launch_attn_q8(const PagedAttnArgs &a, cudaStream_t st) {
    const long long tiles = ((long long)a.kv.max_new * a.G + 63) / 64;
    return launch_pdl(fa_paged_q8_kernel<D>, dim3((unsigned)tiles, (unsigned)a.kv.Hkv, (unsigned)a.kv.n_seq),
                      dim3(128), 0, st, a);
}

// The tensor-core kernel, when a stream may bring more rows than the streaming
// kernel takes: F16 caches, and Q8_0 caches of kUnpackFrom rows or more, whose
// pages it reads as pairs of halves (value = hi + lo) in the workspace.  Over
// shorter ones mma.sync on the pages is as fast and takes no workspace (prompts of
// 32, 64, 96 and 128 tokens, 8 KV heads: 8.3, 12.0, 15.7 and 19.3 us there, 13.7,
// 13.6, 15.0 and 15.1 unpacked; 391: 52 and 22).  It also takes what would need
// more than kUnpackBytes of workspace (128 tokens at 14k: 1630 and 109 us).
constexpr int kUnpackFrom = 96, kUnpackPage = 128;
constexpr size_t kUnpackBytes = size_t(4) << 30;

struct TilePlan {
    bool use;
    PagedTile tile;
    int unpack;               // pages of kUnpackPage keys per stream, 0: none
    size_t o_bytes, u_bytes, bytes;   // partial O, one unpacked pool, all
};

TilePlan plan_tile(const vtx_paged_kv *p, int G, int Hq, int min_rows, int sms) {
    TilePlan t{};
    const int Hkv = (int)p->k.ne[2], D = (int)p->k.ne[0];
    if (p->k.type == VTX_TYPE_Q8_0 && p->max_kv_len >= kUnpackFrom) {
        t.unpack = (p->max_kv_len + kUnpackPage - 1) / kUnpackPage;
        t.u_bytes = (size_t)p->n_seq * t.unpack * kUnpackPage * Hkv * D * 4;
        if (2 * t.u_bytes > kUnpackBytes) t.unpack = 0;
    }
    t.use = (p->k.type == VTX_TYPE_F16 || t.unpack) && p->max_new * (long long)G > min_rows && p->n_seq > 0;
    if (!t.use || !t.unpack) t.u_bytes = 0;
    if (!t.use) return t;
    t.tile.T = 128 / G;
    // streams with more than min_rows rows, and what rounding each up to whole groups adds
    const long long streams = std::min<long long>(p->n_seq, p->n_tokens / (min_rows / G + 1));
    auto groups_of = [&](long long tokens) { return (p->n_tokens + streams * (tokens - 1)) / tokens; };
    // single Q tiles while they fit on the SMs at once (a prompt of 391 tokens, 8 KV
    // heads: 104 CTAs instead of 56, 13.3 us instead of 15.9; 391 at 1600 rows 27 and
    // 36, 512 at 13.8k 133 and 139); beyond that pairs, which share K and V
    const long long pair = groups_of(t.tile.T) * Hkv <= sms ? t.tile.T : 2 * t.tile.T;
    t.tile.tokens = (int)pair;
    t.tile.groups = (int)groups_of(pair);
    t.tile.min_tiles = 2;
    // Splits of a group's key tiles: the number of least estimated time.  A key
    // tile of a group takes about 2.1 us (D = 128), half of that where the group is
    // one Q tile (32 tokens at 700 rows: 17.9 us by 2.1, 15.0 by 1.0), a CTA's start
    // and end 6; a merge writes and reads a split's rows at about 5 TB/s and costs a
    // launch.
    // One stream: its groups are about equal, so whole waves count, and full waves
    // are left whole.  Several: lengths spread, so the average load plus half a
    // CTA's time.
    t.tile.shift = t.unpack ? 6 : 7;
    const int tiles = std::max(1, (p->max_kv_len + (1 << t.tile.shift) - 1) >> t.tile.shift);
    const bool one_tile = pair == t.tile.T || p->max_new <= t.tile.T;
    const double tile_us = (one_tile ? 1.0 : 2.1) * (D == 128 ? 1.0 : 0.76), cta_us = 6.0;
    const double row_us = (double)D * 8 / 5e6;               // one row, one split
    const long long items = (long long)t.tile.groups * Hkv;
    double best = 1e30, one = 1e30;
    t.tile.n_splits = 1;
    for (int s = 1; s <= 32 && s <= (tiles + 1) / 2; ++s) {
        const double each = (double)((tiles + s - 1) / s) * tile_us + cta_us;
        if (p->n_seq == 1) {
            for (long long whole = 0; whole <= (s > 1 ? items : 0); whole += sms) {
                const double us = (double)(whole / sms) * (tiles * tile_us + cta_us) +
                                  (double)(((items - whole) * s + sms - 1) / sms) * each +
                                  (s > 1 ? (items - whole) * 256.0 * s * row_us + 3.0 : 0.0);
                if (s == 1) one = us;
                // launches of full waves are short of power, not of SMs: a small gain
                // is none there (2048 tokens at 14k: 501 us whole, 516 with the last
                // wave split; 1184 tokens: 360 and 287)
                if (us < best && (s == 1 || items < sms || us < 0.85 * one)) {
                    best = us;
                    t.tile.n_splits = s;
                    t.tile.whole = (int)whole;
                }
            }
        } else {
            const double ctas = (double)p->n_tokens / pair * Hkv;
            const double us = ctas * tiles * 0.5 / sms * tile_us + 0.5 * each +
                              (s > 1 ? (double)p->n_tokens * Hq * s * row_us + 3.0 : 0.0);
            if (us < best) { best = us; t.tile.n_splits = s; }
        }
    }
    if (t.tile.n_splits > 1) {
        // every split that long, so that shorter streams have fewer
        t.tile.min_tiles = std::max(2, (tiles + t.tile.n_splits - 1) / t.tile.n_splits);
        const size_t rows = (size_t)p->n_tokens * Hq * t.tile.n_splits;
        t.o_bytes = align_up(rows * D * 4, 256);
        t.bytes = t.o_bytes + align_up(rows * 8, 256);
    }
    t.bytes += 2 * t.u_bytes;                                // pages are multiples of 256 bytes
    return t;
}

// The unpacked copy of a Q8_0 cache, two rows of halves for each of its own, at the end of the tile plan's workspace.
PagedView unpacked_view(const PagedView &kv, const TilePlan &t, int D, char *ws) {
    PagedView u = kv;
    u.k = ws + t.bytes - 2 * t.u_bytes;
    u.v = u.k + t.u_bytes;
    u.nb1 = D * 2; u.nb2 = (long long)kUnpackPage * D * 4; u.nb3 = u.nb2 * kv.Hkv;
    u.table = nullptr;
    u.max_pages = t.unpack; u.n_pages = kv.n_seq * t.unpack;
    u.shift = 7;
    u.cap = (int)std::min<long long>(kv.cap, (long long)t.unpack << 7);       // what was unpacked
    return u;
}

template <int D>
int launch_unpack(const PagedAttnArgs &a, const PagedView &out, cudaStream_t st) {
    return launch_pdl(paged_unpack_kernel<D>,
                      dim3((unsigned)(out.max_pages * (kUnpackPage / 32)), (unsigned)a.kv.Hkv, (unsigned)a.kv.n_seq),
                      dim3(128), 0, st, a, out);
}

// Map of an F16 pool: (dim, row, head, page), boxes of 64 dims x min(page, 128) rows.
// key_rows: rows that a key has (2 in an unpacked copy).
int encode_pool_map(CUtensorMap *m, const PagedView &kv, void *pool, int D, int key_rows = 1) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
    if (!enc) return VTX_ERR_CUDA;
    const long long page = (long long)key_rows << kv.shift;                   // extent-1 axes: any legal stride
    const long long s2 = kv.Hkv > 1 ? kv.nb2 : kv.nb1 * page, s3 = kv.n_pages > 1 ? kv.nb3 : s2 * kv.Hkv;
    cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)page, (cuuint64_t)kv.Hkv, (cuuint64_t)kv.n_pages};
    cuuint64_t strides[3] = {(cuuint64_t)kv.nb1, (cuuint64_t)s2, (cuuint64_t)s3};
    cuuint32_t box[4] = {64, (cuuint32_t)std::min<long long>(page, 128), 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, pool, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? VTX_OK : VTX_ERR_STRIDE;
}

// Map of an F16 q: (dim, head, token), boxes of 64 dims x G heads x T tokens.
int encode_paged_q_map(CUtensorMap *m, const vtx_tensor *q, int G, int T) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
    if (!enc) return VTX_ERR_CUDA;
    const size_t s1 = q->ne[2] > 1 ? q->nb[2] : (size_t)q->ne[0] * 2;
    const size_t s2 = q->ne[1] > 1 ? q->nb[1] : s1 * (size_t)q->ne[2];
    cuuint64_t dims[4] = {(cuuint64_t)q->ne[0], (cuuint64_t)q->ne[2], (cuuint64_t)q->ne[1], 1};
    cuuint64_t strides[3] = {(cuuint64_t)s1, (cuuint64_t)s2, (cuuint64_t)(s2 * (size_t)q->ne[1])};
    cuuint32_t box[4] = {64, (cuuint32_t)G, (cuuint32_t)T, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, q->data, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? VTX_OK : VTX_ERR_STRIDE;
}

template <int D, bool UF, bool LO>
int launch_tile(const CUtensorMap (&m)[3], const PagedAttnArgs &a, const PagedTile &tl, cudaStream_t st) {
    using C = PagedTileCfg<D>;
    static std::atomic<int> done[kMaxDevices];
    int rc = allow_smem(fa_paged_sm100_kernel<D, UF, LO>, C::SMEM, done);
    if (rc != VTX_OK) return rc;
    const long long items = (long long)tl.groups * a.kv.Hkv;
    const long long ctas = tl.whole + (items - tl.whole) * tl.n_splits;
    if (ctas > 0x7fffffffLL) return VTX_ERR_UNSUPPORTED;
    if (ctas == 0) return VTX_OK;
    return launch_pdl(fa_paged_sm100_kernel<D, UF, LO>, dim3((unsigned)ctas), dim3(C::NTHREADS), C::SMEM, st, m[0], m[1],
                      m[2], a, tl);
}

template <int D>
int launch_tile_any(const CUtensorMap (&m)[3], const PagedAttnArgs &a, const TilePlan &t, bool uf, cudaStream_t st) {
    if (t.unpack) return uf ? launch_tile<D, true, true>(m, a, t.tile, st) : launch_tile<D, false, true>(m, a, t.tile, st);
    return uf ? launch_tile<D, true, false>(m, a, t.tile, st) : launch_tile<D, false, false>(m, a, t.tile, st);
}

// A warp per query row for few rows (20 tokens of 32 heads at 12k rows 28.3 -> 24.3
// us, 70 at 6k 29.9 -> 27.5), else per four of them, which look the stream up once
// (192 tokens: 32.8 us, a warp per row 33.9).
template <int D>
int launch_tile_combine(const PagedAttnArgs &a, const PagedTile &tl, int sms, cudaStream_t st) {
    const unsigned T = (unsigned)a.kv.n_tokens, Hq = (unsigned)a.Hq;
    if ((long long)T * Hq <= 16LL * sms)
        return launch_pdl(fa_paged_tile_combine_kernel<D, 1>, dim3(T, (Hq + 7) / 8), dim3(256), 0, st, a, tl);
    return launch_pdl(fa_paged_tile_combine_kernel<D, 4>, dim3(T, (Hq + 31) / 32), dim3(256), 0, st, a, tl);
}

template <int D, int KVT>
int launch_score(const PagedScoreArgs &a, cudaStream_t st) {
    return launch_pdl(kv_score_kernel<D, KVT>,
                      dim3((unsigned)((a.kv.max_kv + 127) / 128), (unsigned)a.kv.Hkv, (unsigned)a.kv.n_seq), dim3(128),
                      0, st, a);
}

// Few query rows: the splits of the streaming attention kernel (whose K half
// this is), without partials.
template <int D, int KVT, int ROWS, bool UF>
int launch_score_stream_t(const PagedScoreArgs &a, const PagedSplit &sp, cudaStream_t st) {
    using C = ScoreStreamCfg<D, KVT>;
    static std::atomic<int> done[kMaxDevices];
    int rc = allow_smem(kv_score_stream_kernel<D, KVT, ROWS, UF>, C::SMEM, done);
    if (rc != VTX_OK) return rc;
    const long long ctas = (long long)a.kv.n_seq * a.kv.Hkv * sp.n_splits;
    if (ctas > 0x7fffffffLL) return VTX_ERR_UNSUPPORTED;
    return launch_pdl(kv_score_stream_kernel<D, KVT, ROWS, UF>, dim3((unsigned)ctas), dim3(128), C::SMEM, st, a, sp);
}

template <int D, int KVT>
int launch_score_stream(const PagedScoreArgs &a, int rows, int sms, cudaStream_t st) {
    const long long base = (long long)a.kv.n_seq * a.kv.Hkv;
    const int tiles = std::max(1, (a.kv.max_kv + 15) / 16);
    PagedSplit sp{};
    const long long want = std::max<long long>((4LL * sms + base - 1) / base, (tiles + 63) / 64);
    sp.n_splits = (int)std::min<long long>(want, (tiles + 3) / 4);
    sp.tiles = (tiles + sp.n_splits - 1) / sp.n_splits;
    if (a.softcap != 0.0f)
        return rows <= 8 ? launch_score_stream_t<D, KVT, 8, true>(a, sp, st)
                         : launch_score_stream_t<D, KVT, 16, true>(a, sp, st);
    return rows <= 8 ? launch_score_stream_t<D, KVT, 8, false>(a, sp, st)
                     : launch_score_stream_t<D, KVT, 16, false>(a, sp, st);
}

template <int D, int KVT, int NT, bool UF>
int launch_score_tile_n(const CUtensorMap (&m)[2], const PagedScoreArgs &a, int T, cudaStream_t st) {
    using C = ScoreTileCfg<D, KVT, NT>;
    static std::atomic<int> done[kMaxDevices];
    int rc = allow_smem(kv_score_sm100_kernel<D, KVT, NT, UF>, C::SMEM, done);
    if (rc != VTX_OK) return rc;
    return launch_pdl(kv_score_sm100_kernel<D, KVT, NT, UF>,
                      dim3((unsigned)((a.kv.max_kv + 128 * NT - 1) / (128 * NT)), (unsigned)a.kv.Hkv,
                           (unsigned)a.kv.n_seq),
                      dim3(C::NTHREADS), C::SMEM, st, m[0], m[1], a, T);
}

// F16: four key tiles per CTA halve the reads of Q from L2, two spread over more
// SMs: four once they fill the GPU (500 tokens: 16000 keys 102 us with four, 116
// with two; 4000 keys 51 and 31 us).  Q8_0: two (shared memory).
template <int D, bool UF>
int launch_score_tile(const CUtensorMap (&m)[2], const PagedScoreArgs &a, bool f16, int T, int sms, cudaStream_t st) {
    const long long ctas4 = ((long long)a.kv.max_kv + 511) / 512 * a.kv.Hkv * a.kv.n_seq;
    if (!f16) return launch_score_tile_n<D, 8, 2, UF>(m, a, T, st);
    return ctas4 >= sms ? launch_score_tile_n<D, 1, 4, UF>(m, a, T, st) : launch_score_tile_n<D, 1, 2, UF>(m, a, T, st);
}

struct EvictPlan {
    long long items;
    int max_moves;
    size_t moves_bytes, bytes;
};

EvictPlan plan_evict(const vtx_paged_kv *p) {
    EvictPlan e{};
    e.items = (long long)p->n_seq * p->k.ne[2];
    e.max_moves = std::max(1, p->max_kv_len / 2);        // min(m, n - m) rows move at most
    e.moves_bytes = align_up((size_t)e.items * e.max_moves * sizeof(int2), 256);
    e.bytes = e.moves_bytes + align_up((size_t)e.items * sizeof(int2), 256);
    return e;
}

template <bool SMEM, int UNIT>
int launch_evict_select(const PagedEvictArgs &a, long long items, int sms, cudaStream_t st) {
    size_t keys = SMEM ? align_up((size_t)a.kv.max_kv * 4, 16) : 0;
    // Two CTAs fit on an SM.  Up to an item per SM, shared memory for one alone: a
    // launch that begins while the one before still runs would put two on some SMs (64
    // items of 1500 to 8192 rows, call after call: 27.1 -> 22.6 us with the moves).
    if (SMEM && UNIT == 0 && items <= sms) keys = std::max(keys, size_t(116) << 10);
    if (SMEM) {
        static std::atomic<int> done[kMaxDevices];
        const int rc = allow_smem(kv_evict_select_kernel<SMEM, UNIT>, kEvictKeysInSmem * 4, done);
        if (rc != VTX_OK) return rc;
    }
    return launch_pdl(kv_evict_select_kernel<SMEM, UNIT>, dim3((unsigned)items), dim3(kEvictThreads), keys, st, a);
}

}  // namespace

extern "C" {

int vtx_kv_append_paged(const vtx_kv_append_paged_args *p, void *stream) {
    if (!p) return VTX_ERR_NULL;
    int rc = check_paged(p->kv);
    if (rc != VTX_OK) return rc;
    const vtx_paged_kv *kv = p->kv;
    const int D = (int)kv->k.ne[0];
    if (p->q_out && p->q_out_type != VTX_TYPE_F32 && p->q_out_type != VTX_TYPE_F16) return VTX_ERR_TYPE;
    if (p->q_out && p->n_head_q < 1) return VTX_ERR_SHAPE;
    if (!(p->freq_base > 0.0f) || !std::isfinite(p->freq_base)) return VTX_ERR_UNSUPPORTED;
    if ((p->row_pos || p->score) && p->row_cap < kv->max_kv_len) return VTX_ERR_SHAPE;
    if (kv->n_tokens == 0) return VTX_OK;
    if (!p->k || !p->v || !p->positions || (kv->n_seq > 0 && !kv->q_start) || (p->q_out && !p->q)) return VTX_ERR_NULL;
    const size_t kvrow = (size_t)kv->k.ne[2] * D * 4, qrow = (size_t)p->n_head_q * D;
    if (p->k_nb1 < kvrow || p->v_nb1 < kvrow) return VTX_ERR_STRIDE;
    const unsigned long long rows =
        reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v) | p->k_nb1 | p->v_nb1 |
        (p->q_out ? reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->q_out) | p->q_nb1 |
                        p->q_out_nb1 : 0);
    if (rows % 8) return VTX_ERR_STRIDE;
    if (p->q_out && (p->q_nb1 < qrow * 4 || p->q_out_nb1 < qrow * elem_size(p->q_out_type))) return VTX_ERR_STRIDE;
    DeviceState *ds = nullptr;
    rc = ensure_device(&ds);
    if (rc != VTX_OK) return rc;
    KvAppendPagedArgs a{};
    a.kv = view_of(kv, ds);
    a.Hq = p->q_out ? p->n_head_q : 0;
    a.q8 = kv->k.type == VTX_TYPE_Q8_0;
    a.qo_f16 = p->q_out_type == VTX_TYPE_F16;
    a.q = p->q; a.q_nb1 = (long long)(p->q_nb1 / 4);
    a.k = p->k; a.k_nb1 = (long long)(p->k_nb1 / 4);
    a.v = p->v; a.v_nb1 = (long long)(p->v_nb1 / 4);
    a.q_out = p->q_out; a.qo_nb1 = (long long)(p->q_out_nb1 / (a.qo_f16 ? 2 : 4));
    a.positions = p->positions;
    a.row_pos = p->row_pos; a.score = p->score; a.row_cap = p->row_cap;
    for (int i = 0; i < D / 2; ++i)
        a.turns[i] = std::pow((double)p->freq_base, -2.0 * i / D) / (2.0 * 3.14159265358979323846);
    // few tokens: a warp's rows (two or four) at once per CTA and warp, so that all
    // rows are in flight together; many: one CTA and one cos/sin table per token
    const int per_tok = a.Hq + 2 * a.kv.Hkv;
    a.rows_per_cta = kv->n_tokens >= 2 * ds->sms ? per_tok : D == 64 ? 32 : 16;
    const dim3 grid((unsigned)kv->n_tokens, (unsigned)((per_tok + a.rows_per_cta - 1) / a.rows_per_cta));
    if (grid.y > 65535) return VTX_ERR_SHAPE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows % 16 == 0)
        return D == 64 ? launch_pdl(kv_append_paged_kernel<64, true>, grid, dim3(256), 0, st, a)
                       : launch_pdl(kv_append_paged_kernel<128, true>, grid, dim3(256), 0, st, a);
    return D == 64 ? launch_pdl(kv_append_paged_kernel<64, false>, grid, dim3(256), 0, st, a)
                   : launch_pdl(kv_append_paged_kernel<128, false>, grid, dim3(256), 0, st, a);
}

size_t vtx_flash_attn_paged_workspace(const vtx_paged_kv *kv, int32_t n_head_q) {
    if (check_paged(kv) != VTX_OK || n_head_q < 1 || n_head_q % kv->k.ne[2] ||
        n_head_q / kv->k.ne[2] > kMaxGroup)
        return (size_t)-1;
    const int G = n_head_q / (int)kv->k.ne[2], sms = current_sms();
    const DecodePlan d = plan_decode(kv, G, sms);
    const size_t rest = d.bytes + plan_tile(kv, G, n_head_q, d.use ? d.rows : 0, sms).bytes;
    return arrival_bytes(kv, rest) + rest;
}

int vtx_flash_attn_paged(const vtx_flash_attn_paged_args *p, void *workspace, size_t workspace_bytes, void *stream) {
    if (!p) return VTX_ERR_NULL;
    int rc = check_paged(p->kv);
    if (rc == VTX_OK) rc = check_q(p->kv, p->q);
    if (rc == VTX_OK) rc = check_params(p->params);
    if (rc != VTX_OK) return rc;
    const vtx_paged_kv *kv = p->kv;
    const vtx_tensor *q = p->q, *d = p->dst;
    if (!d) return VTX_ERR_NULL;
    if (d->type != VTX_TYPE_F32 && d->type != VTX_TYPE_F16) return VTX_ERR_TYPE;
    if (d->ne[0] != q->ne[0] || d->ne[1] != q->ne[2] || d->ne[2] != q->ne[1] || d->ne[3] != 1) return VTX_ERR_SHAPE;
    if (d->nb[0] != (size_t)elem_size(d->type)) return VTX_ERR_STRIDE;
    for (int i = 1; i < 3; ++i)                               // rows of dst must not overlap
        if (d->ne[i] > 1 && d->nb[i] < (size_t)d->ne[0] * d->nb[0]) return VTX_ERR_STRIDE;
    if (kv->n_tokens == 0 || kv->n_seq == 0) return VTX_OK;
    if (!d->data) return VTX_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(d->data) % 16 || d->nb[1] % 16 || d->nb[2] % 16) return VTX_ERR_STRIDE;
    const int Hq = (int)q->ne[2];
    DeviceState *ds = nullptr;
    rc = ensure_device(&ds);
    if (rc != VTX_OK) return rc;
    DecodePlan dp = plan_decode(kv, Hq / (int)kv->k.ne[2], ds->sms);
    TilePlan tp = plan_tile(kv, Hq / (int)kv->k.ne[2], Hq, dp.use ? dp.rows : 0, ds->sms);
    const size_t first = arrival_bytes(kv, dp.bytes + tp.bytes), need = first + dp.bytes + tp.bytes;
    if (workspace_bytes < need || (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256)))
        return VTX_ERR_WORKSPACE;
    PagedAttnArgs a{};
    a.kv = view_of(kv, ds);
    a.q = static_cast<const char *>(q->data); a.q_f16 = q->type == VTX_TYPE_F16;
    a.q_nbt = (long long)q->nb[1]; a.q_nbh = (long long)q->nb[2];
    a.dst = static_cast<char *>(d->data); a.d_f16 = d->type == VTX_TYPE_F16;
    a.d_nbt = (long long)d->nb[2]; a.d_nbh = (long long)d->nb[1];
    a.lse = p->lse;
    a.Hq = Hq; a.G = Hq / a.kv.Hkv;
    a.scale = p->params->scale; a.softcap = p->params->logit_softcap;
    a.causal = p->params->causal != 0;
    a.window = std::min(p->params->window, 1 << 30);          // sums with lengths stay in range
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool f16 = kv->k.type == VTX_TYPE_F16, d64 = kv->k.ne[0] == 64;
    // chunks first (their CTAs are long), few-token streams beside them
    a.min_rows = dp.use ? dp.rows : 0;
    PagedAttnArgs ta = a;                                     // what the tensor-core kernel reads
    if (tp.use) {
        char *ws = static_cast<char *>(workspace) + first + dp.bytes;
        tp.tile.part_o = reinterpret_cast<float *>(ws);
        tp.tile.part_ml = reinterpret_cast<float *>(ws + tp.o_bytes);
        const int D = (int)kv->k.ne[0];
        if (tp.unpack) {
            ta.kv = unpacked_view(a.kv, tp, D, ws);
            rc = d64 ? launch_unpack<64>(a, ta.kv, st) : launch_unpack<128>(a, ta.kv, st);
            if (rc != VTX_OK) return rc;
        }
        CUtensorMap m[3];
        rc = encode_pool_map(&m[0], ta.kv, ta.kv.k, D, tp.unpack ? 2 : 1);
        if (rc == VTX_OK) rc = encode_pool_map(&m[1], ta.kv, ta.kv.v, D, tp.unpack ? 2 : 1);
        m[2] = m[0];                                          // an F32 q is read by the softmax warps
        if (rc == VTX_OK && a.q_f16) rc = encode_paged_q_map(&m[2], q, a.G, tp.tile.T);
        if (rc != VTX_OK) return rc;
        // tanh, or a scale that the row maximum cannot carry: logits formed first
        const bool uf = a.softcap != 0.0f || !(a.scale > 0.0f);
        if (d64) rc = launch_tile_any<64>(m, ta, tp, uf, st);
        else rc = launch_tile_any<128>(m, ta, tp, uf, st);
    } else if (kv->max_new * (long long)a.G > a.min_rows) {
        rc = d64 ? launch_attn_q8<64>(a, st) : launch_attn_q8<128>(a, st);
    }
    if (rc != VTX_OK) return rc;
    if (dp.use) {
        char *ws = static_cast<char *>(workspace);
        dp.split.arrived = reinterpret_cast<unsigned *>(ws);
        dp.split.part_o = reinterpret_cast<float *>(ws + first);
        dp.split.part_ml = reinterpret_cast<float *>(ws + first + dp.o_bytes);
        dp.split.beside = kv->max_new * (long long)a.G > a.min_rows;
        rc = d64 ? (f16 ? launch_decode_rows<64, 1>(a, dp, st) : launch_decode_rows<64, 8>(a, dp, st))
                 : (f16 ? launch_decode_rows<128, 1>(a, dp, st) : launch_decode_rows<128, 8>(a, dp, st));
        if (rc != VTX_OK) return rc;
    }
    if (!tp.use || tp.tile.n_splits == 1) return VTX_OK;
    return d64 ? launch_tile_combine<64>(ta, tp.tile, ds->sms, st) : launch_tile_combine<128>(ta, tp.tile, ds->sms, st);
}

int vtx_kv_score_paged(const vtx_kv_score_paged_args *p, void *stream) {
    if (!p) return VTX_ERR_NULL;
    int rc = check_paged(p->kv);
    if (rc == VTX_OK) rc = check_q(p->kv, p->q);
    if (rc == VTX_OK) rc = check_params(p->params);
    if (rc != VTX_OK) return rc;
    const vtx_paged_kv *kv = p->kv;
    if (!std::isfinite(p->decay)) return VTX_ERR_UNSUPPORTED;
    if (p->observe < 0 || p->row_cap < kv->max_kv_len) return VTX_ERR_SHAPE;
    if (kv->n_seq == 0 || kv->max_kv_len == 0) return VTX_OK;
    if (!p->score_out || !kv->q_start || (kv->n_tokens > 0 && !p->lse) || (p->decay != 0.0f && !p->score))
        return VTX_ERR_NULL;
    DeviceState *ds = nullptr;
    rc = ensure_device(&ds);
    if (rc != VTX_OK) return rc;
    PagedScoreArgs a{};
    a.kv = view_of(kv, ds);
    a.q = static_cast<const char *>(p->q->data); a.q_f16 = p->q->type == VTX_TYPE_F16;
    a.q_nbt = (long long)p->q->nb[1]; a.q_nbh = (long long)p->q->nb[2];
    a.lse = p->lse; a.score = p->score; a.score_out = p->score_out; a.row_cap = p->row_cap;
    a.decay = p->decay; a.observe = p->observe;
    a.Hq = (int)p->q->ne[2]; a.G = a.Hq / a.kv.Hkv;
    a.scale = p->params->scale; a.softcap = p->params->logit_softcap;
    a.causal = p->params->causal != 0;
    a.window = std::min(p->params->window, 1 << 30);          // sums with lengths stay in range
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool f16 = kv->k.type == VTX_TYPE_F16, d64 = kv->k.ne[0] == 64;
    const long long rows = (long long)(p->observe > 0 ? std::min(p->observe, kv->max_new) : kv->max_new) * a.G;
    if (rows <= kFewRows) {
        const int r = (int)rows, n = ds->sms;
        if (d64) return f16 ? launch_score_stream<64, 1>(a, r, n, st) : launch_score_stream<64, 8>(a, r, n, st);
        return f16 ? launch_score_stream<128, 1>(a, r, n, st) : launch_score_stream<128, 8>(a, r, n, st);
    }
    if (a.q_f16) {
        CUtensorMap m[2];
        const int T = 128 / a.G;
        rc = encode_paged_q_map(&m[1], p->q, a.G, T);
        m[0] = m[1];                                          // Q8_0 pages are read by the threads
        if (rc == VTX_OK && f16) rc = encode_pool_map(&m[0], a.kv, a.kv.k, (int)kv->k.ne[0]);
        if (rc != VTX_OK) return rc;
        if (a.softcap != 0.0f)
            return d64 ? launch_score_tile<64, true>(m, a, f16, T, ds->sms, st)
                       : launch_score_tile<128, true>(m, a, f16, T, ds->sms, st);
        return d64 ? launch_score_tile<64, false>(m, a, f16, T, ds->sms, st)
                   : launch_score_tile<128, false>(m, a, f16, T, ds->sms, st);
    }
    if (d64) return f16 ? launch_score<64, 1>(a, st) : launch_score<64, 8>(a, st);
    return f16 ? launch_score<128, 1>(a, st) : launch_score<128, 8>(a, st);
}

size_t vtx_kv_evict_paged_workspace(const vtx_paged_kv *kv) {
    return check_paged(kv) == VTX_OK ? plan_evict(kv).bytes : (size_t)-1;
}

int vtx_kv_evict_paged(const vtx_kv_evict_paged_args *p, void *workspace, size_t workspace_bytes, void *stream) {
    if (!p) return VTX_ERR_NULL;
    int rc = check_paged(p->kv);
    if (rc != VTX_OK) return rc;
    const vtx_paged_kv *kv = p->kv;
    if (p->keep < 0 || p->n_sink < 0 || p->n_recent < 0 || (long long)p->n_sink + p->n_recent > p->keep)
        return VTX_ERR_SHAPE;
    if (p->row_cap < kv->max_kv_len) return VTX_ERR_SHAPE;
    if ((p->score_out || p->pos_out || p->src_out) && p->out_cap < p->keep) return VTX_ERR_SHAPE;
    if (((p->score_out && p->score_out == p->score) || (p->pos_out && p->pos_out == p->row_pos)) &&
        p->out_cap != p->row_cap)
        return VTX_ERR_SHAPE;
    if (kv->n_seq == 0) return VTX_OK;
    if (!p->kv_len_out || (kv->max_kv_len > 0 && !p->score) || (p->row_pos && !p->next_pos)) return VTX_ERR_NULL;
    const EvictPlan e = plan_evict(kv);
    if (e.items > (1 << 24)) return VTX_ERR_UNSUPPORTED;
    if (workspace_bytes < e.bytes || !workspace || reinterpret_cast<uintptr_t>(workspace) % 256)
        return VTX_ERR_WORKSPACE;
    DeviceState *ds = nullptr;
    rc = ensure_device(&ds);
    if (rc != VTX_OK) return rc;
    PagedEvictArgs a{};
    a.kv = view_of(kv, ds);
    a.score = p->score; a.row_pos = p->row_pos; a.next_pos = p->next_pos;
    a.score_out = p->score_out; a.pos_out = p->pos_out; a.src_out = p->src_out; a.kv_len_out = p->kv_len_out;
    a.keep = p->keep; a.n_sink = p->n_sink; a.n_recent = p->n_recent;
    a.row_cap = p->row_cap; a.out_cap = p->out_cap;
    a.max_moves = e.max_moves;
    a.moves = static_cast<int2 *>(workspace);
    a.counts = reinterpret_cast<int2 *>(static_cast<char *>(workspace) + e.moves_bytes);
    a.row_bytes = row_bytes(kv->k.type, kv->k.ne[0]);
    // a CTA per 64 moves at most (8 warps of 8), about eight CTAs per SM over all
    a.slices = (int)std::max<long long>(1, std::min<long long>((8LL * ds->sms + e.items - 1) / e.items,
                                                               (e.max_moves + 63) / 64));
    // rows of 256 or 128 (F16), 136 or 68 bytes (Q8_0: 8- and 4-byte aligned)
    const int unit = kv->k.type == VTX_TYPE_F16 ? 16 : a.row_bytes % 8 == 0 ? 8 : 4;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Few moves: one kernel, a launch less.  A (stream, head) is one CTA there, too
    // little for many moves, and with enough items the two kernels take as long as
    // one (256 items of 1500 to 8192 rows: 87 against 91 us; 71 by now).  Not in place on kv_len
    // or next_pos, which the other heads' CTAs may not have read yet.
    if (e.max_moves <= 512 && p->kv_len_out != kv->kv_len && p->kv_len_out != p->next_pos) {
        if (unit == 16) return launch_evict_select<true, 16>(a, e.items, ds->sms, st);
        return unit == 8 ? launch_evict_select<true, 8>(a, e.items, ds->sms, st)
                         : launch_evict_select<true, 4>(a, e.items, ds->sms, st);
    }
    rc = kv->max_kv_len <= kEvictKeysInSmem ? launch_evict_select<true, 0>(a, e.items, ds->sms, st)
                                            : launch_evict_select<false, 0>(a, e.items, ds->sms, st);
    if (rc != VTX_OK) return rc;
    const dim3 grid((unsigned)(e.items * a.slices));
    if (unit == 16) return launch_pdl(kv_evict_move_kernel<16>, grid, dim3(256), 0, st, a);
    return unit == 8 ? launch_pdl(kv_evict_move_kernel<8>, grid, dim3(256), 0, st, a)
                     : launch_pdl(kv_evict_move_kernel<4>, grid, dim3(256), 0, st, a);
}

}  // extern "C"
