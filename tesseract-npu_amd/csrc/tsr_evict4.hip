// tsr_evict4.hip -- host side of eviction by attention weight: the weights that cells of a 4-bit K cache gather, the cells that
// are kept, and their move (caches of every type).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "kernels.hpp"
#include "kv4.hpp"
#include "runtime.hpp"
#include "tsr_hip.h"
#include "weights4_plan.hpp"

static bool heads_ok(uint32_t D, uint32_t n_head, uint32_t n_head_kv) {
    return (D == 64u || D == 128u || D == 256u || D == 512u) && n_head_kv != 0u && n_head != 0u && n_head % n_head_kv == 0u &&
           n_head / n_head_kv <= 64u && (uint64_t)n_head * D <= 32768u;
}

// A call's workspace: the caller's, or eagerly the context's scratch, which orders calls across streams; a graph's replays
// are ordered by nobody, so that a captured call brings its own. The caller holds the context's mutex.
static int workspace(tsr_hip_ctx * ctx, size_t need, void * ws_dev, hipStream_t s, void ** ws) {
    *ws = ws_dev;
    if (ws_dev != nullptr || need == 0u) return TSR_HIP_OK;
    if (tsr_capturing(s)) return TSR_HIP_E_ARG;
    const int rc = ctx->scratch.reserve(need, s);
    *ws = ctx->scratch.ptr;
    return rc;
}

size_t tsr_hip_attn_weights_kv4_ws(tsr_hip_ctx * ctx, uint32_t T, uint32_t D, uint32_t n_head, uint32_t n_head_kv, uint32_t n_kv) {
    if (ctx == nullptr || T == 0u || T > 65535u || !heads_ok(D, n_head, n_head_kv) || n_kv == 0u || n_kv > 0x7FFFFFFFu) return 0u;
    return tsr::weights4_ws(T, D, n_head, n_head_kv, n_kv, (uint32_t)ctx->n_cu);
}

int tsr_hip_attn_weights_kv4(tsr_hip_ctx * ctx, const float * q_dev, uint32_t T, uint64_t q_stride, const tsr_hip_kv * kc, uint32_t D,
                             uint32_t n_head, uint32_t n_head_kv, float scale, uint32_t n_kv, const uint32_t * runs_dev,
                             const float * before_dev, float decay, float * out_dev, void * ws_dev, size_t ws_bytes, void * stream) {
    if (ctx == nullptr || q_dev == nullptr || kc == nullptr || out_dev == nullptr || T == 0u || T > 65535u) return TSR_HIP_E_ARG;
    if (!heads_ok(D, n_head, n_head_kv)) return TSR_HIP_E_SHAPE;
    if (!(scale > 0.0f) || !std::isnormal(scale) || !std::isfinite(decay)) return TSR_HIP_E_SHAPE;
    if (kc->type == TSR_HIP_KV_Q8_0) return TSR_HIP_E_FMT;
    if (kc->E != n_head_kv * D) return TSR_HIP_E_SHAPE;
    if (n_kv > kc->kv_size) return TSR_HIP_E_RANGE;
    if ((((uintptr_t)q_dev | (uintptr_t)runs_dev) & 15u) != 0u || (((uintptr_t)before_dev | (uintptr_t)out_dev) & 3u) != 0u ||
        (T > 1u && (q_stride % 4u != 0u || q_stride < (uint64_t)n_head * D)))
        return TSR_HIP_E_ARG;
    if (n_kv == 0u) return TSR_HIP_OK;
    const tsr::Weights4Plan p = tsr::weights4_plan(T, D, n_head, n_head_kv, n_kv, (uint32_t)ctx->n_cu);
    if (ws_dev != nullptr && (ws_bytes < tsr::weights4_ws(T, D, n_head, n_head_kv, n_kv, (uint32_t)ctx->n_cu) || ((uintptr_t)ws_dev & 15u) != 0u))
        return TSR_HIP_E_ARG;
    tsr::Attn4Args a{};
    a.q_stride = q_stride;
    a.k = kc->dev;
    a.out = out_dev;
    a.type = kc->type;
    a.D = D;
    a.G = n_head / n_head_kv;
    a.inv_G = a.G == 1u ? 0u : (uint32_t)((1ull << 32) / a.G) + 1u;
    a.n_head_kv = n_head_kv;
    a.n_kv = n_kv;
    a.n_tiles = tsr::kv4_tiles(kc->kv_size);
    a.S = p.S;
    a.scale = scale;
    std::lock_guard<std::mutex> lk(ctx->mtx);
    (void)hipSetDevice(ctx->device);
    hipStream_t s = ctx->pick(stream);
    void * ws = nullptr;
    const int rc = workspace(ctx, p.ws_bytes, ws_dev, s, &ws);
    if (rc) return rc;
    a.part = (float *)ws;
    ctx->ctr.flash_attn_calls++;
    ctx->ctr.flash_attn_kv_bytes += (uint64_t)n_kv * (kc->E / 32u) * tsr::kv4_block_bytes(kc->type);
    const float * before = decay != 0.0f ? before_dev : nullptr;
    for (uint32_t t0 = 0; t0 < T; t0 += p.tokens) {               // (a launch adds to what those before it left)
        tsr::Weights4Plan q = p;
        a.T = std::min(T - t0, p.tokens);
        q.n_rg = (a.T * a.G + 16u * p.NT - 1u) / (16u * p.NT);
        a.q = q_dev + t0 * q_stride;
        a.runs = runs_dev ? runs_dev + 4u * (size_t)t0 : nullptr;
        if (tsr_launch_attn4_weights(a, q, before, t0 == 0u ? decay : 1.0f, s)) return TSR_HIP_E_HIP;
        before = out_dev;
    }
    return TSR_HIP_OK;
}

int tsr_hip_kv_pick(tsr_hip_ctx * ctx, const float * weights_dev, uint32_t n_kv, uint32_t n_keep, uint32_t n_first, uint32_t n_last,
                    int64_t * idx_dev, float * kept_dev, void * stream) {
    if (ctx == nullptr || weights_dev == nullptr || idx_dev == nullptr) return TSR_HIP_E_ARG;
    if (n_keep > n_kv || n_kv > 0x7FFFFFFFu) return TSR_HIP_E_RANGE;
    if (n_first > n_keep || n_last > n_keep - n_first) return TSR_HIP_E_SHAPE;
    if ((((uintptr_t)weights_dev | (uintptr_t)kept_dev) & 3u) != 0u || ((uintptr_t)idx_dev & 7u) != 0u || kept_dev == weights_dev)
        return TSR_HIP_E_ARG;
    if (n_keep == 0u) return TSR_HIP_OK;
    std::lock_guard<std::mutex> lk(ctx->mtx);
    (void)hipSetDevice(ctx->device);
    return tsr_launch_kv_pick(weights_dev, n_kv, n_keep, n_first, n_last, idx_dev, kept_dev, ctx->pick(stream)) ? TSR_HIP_E_HIP : TSR_HIP_OK;
}

// A plane's first n cells by themselves: bytes, and where q8_0's quants begin.
static size_t part_bytes(const tsr_hip_kv * kv, uint32_t n, size_t * quants) {
    *quants = 0u;
    if (kv->type != TSR_HIP_KV_Q8_0) return (size_t)(kv->E / 64u) * tsr::kv4_tiles(n) * tsr::kv4_tile_bytes(kv->type);
    const size_t ng = ((size_t)n + 15u) / 16u;
    *quants = (ng * 16u * kv->meta_row + 255u) & ~(size_t)255u;
    return *quants + ng * 16u * kv->E;
}

size_t tsr_hip_kv_gather_ws(tsr_hip_ctx * ctx, const tsr_hip_kv * kv, uint32_t n) {
    if (ctx == nullptr || kv == nullptr || n == 0u || n > kv->kv_size) return 0u;
    size_t quants;
    return part_bytes(kv, n, &quants);
}

int tsr_hip_kv_gather(tsr_hip_ctx * ctx, tsr_hip_kv * dst, const tsr_hip_kv * src, uint32_t which, const int64_t * idx_dev, uint32_t n,
                      int32_t * bad_dev, void * ws_dev, size_t ws_bytes, void * stream) {
    if (ctx == nullptr || dst == nullptr || src == nullptr || idx_dev == nullptr || which > 1u) return TSR_HIP_E_ARG;
    if (dst->type != src->type) return TSR_HIP_E_FMT;
    if (dst->E != src->E) return TSR_HIP_E_SHAPE;
    if (n > dst->kv_size) return TSR_HIP_E_RANGE;
    if (((uintptr_t)idx_dev & 7u) != 0u || ((uintptr_t)bad_dev & 3u) != 0u) return TSR_HIP_E_ARG;
    if (n == 0u) return TSR_HIP_OK;
    const bool self = dst == src, q8 = dst->type == TSR_HIP_KV_Q8_0;
    size_t quants = 0u;
    const size_t need = self ? part_bytes(dst, n, &quants) : 0u;
    if (ws_dev != nullptr && (ws_bytes < need || ((uintptr_t)ws_dev & 15u) != 0u)) return TSR_HIP_E_ARG;
    tsr::KvGatherArgs a{};
    a.src = src->dev;
    a.idx = idx_dev;
    a.n = n;
    a.E = dst->E;
    a.src_size = src->kv_size;
    if (q8) a.src_off = src->quant_off;
    else a.src_tiles = tsr::kv4_tiles(src->kv_size);
    std::lock_guard<std::mutex> lk(ctx->mtx);
    (void)hipSetDevice(ctx->device);
    hipStream_t s = ctx->pick(stream);
    a.bad = ctx->flag(bad_dev);
    if (!self) {
        a.dst = dst->dev;
        if (q8) a.dst_off = dst->quant_off;
        else a.dst_tiles = tsr::kv4_tiles(dst->kv_size);
        return tsr_launch_kv_gather(a, dst->type, which, s) ? TSR_HIP_E_HIP : TSR_HIP_OK;
    }
    void * ws = nullptr;
    const int rc = workspace(ctx, need, ws_dev, s, &ws);
    if (rc) return rc;
    a.dst = (uint8_t *)ws;
    // (cells stay that have no source, and those behind the last of the part's tiles)
    if (q8) {
        a.dst_off = quants;
        a.stay_size = (uint32_t)std::min<uint64_t>(((uint64_t)dst->kv_size + 15u) & ~(uint64_t)15u, 0xFFFFFFF0u);
    } else {
        a.dst_tiles = tsr::kv4_tiles(n);
        a.stay_size = 32u * a.src_tiles;
    }
    if (tsr_launch_kv_gather(a, dst->type, which, s)) return TSR_HIP_E_HIP;
    int e = 0;
    if (q8) {
        const size_t ng = ((size_t)n + 15u) / 16u;
        e = tsr_launch_kv_rows_copy(dst->dev, 0u, a.dst, 0u, ng * 16u * dst->meta_row, 1u, s);
        if (e == 0) e = tsr_launch_kv_rows_copy(dst->dev + dst->quant_off, 0u, a.dst + quants, 0u, ng * 16u * dst->E, 1u, s);
    } else {
        const size_t tb = tsr::kv4_tile_bytes(dst->type);
        e = tsr_launch_kv_rows_copy(dst->dev + tsr::kKv4Header, a.src_tiles * tb, a.dst + tsr::kKv4Header, a.dst_tiles * tb, a.dst_tiles * tb,
                                    dst->E / 64u, s);
    }
    return e ? TSR_HIP_E_HIP : TSR_HIP_OK;
}
