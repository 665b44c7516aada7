// tsr_sparse4.hip -- host side of the sparse attention over 4-bit KV caches: the bounds of a K cache's blocks,
// their selection and the attention over them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "kernels.hpp"
#include "kv4.hpp"
#include "runtime.hpp"
#include "sparse4_plan.hpp"
#include "tsr_hip.h"

static bool block_ok(uint32_t block) { return block != 0u && block % 32u == 0u && block <= 1024u; }
static bool head_ok(uint32_t D) { return D == 64u || D == 128u || D == 256u || D == 512u; }

int tsr_hip_kv4_bounds(tsr_hip_ctx * ctx, const tsr_hip_kv * kc, uint32_t D, uint32_t block, uint32_t n_kv, uint32_t * bounds_dev,
                       const uint32_t * cells_dev, uint32_t n_new, void * stream) {
    if (ctx == nullptr || kc == nullptr || bounds_dev == nullptr) return TSR_HIP_E_ARG;
    if (!head_ok(D) || !block_ok(block) || kc->E % D != 0u) return TSR_HIP_E_SHAPE;
    if (kc->type == TSR_HIP_KV_Q8_0) return TSR_HIP_E_FMT;
    if (n_kv > kc->kv_size) return TSR_HIP_E_RANGE;
    if (((uintptr_t)bounds_dev & 15u) != 0u || ((uintptr_t)cells_dev & 3u) != 0u || (cells_dev != nullptr && n_new == 0u))
        return TSR_HIP_E_ARG;
    if (n_kv == 0u) return TSR_HIP_OK;
    tsr::Kv4BoundsArgs a{};
    a.k = kc->dev;
    a.cells = cells_dev;
    a.bounds = bounds_dev;
    a.type = kc->type;
    a.E = kc->E;
    a.D = D;
    a.n_tiles = tsr::kv4_tiles(kc->kv_size);
    a.block = block;
    a.n_kv = n_kv;
    a.stride = (uint32_t)(((uint64_t)kc->kv_size + block - 1u) / block);
    a.n_blocks = (n_kv + block - 1u) / block;                      // (cells stay below 2^31)
    if (cells_dev != nullptr) a.n_blocks = (uint32_t)std::min<uint64_t>(a.n_blocks, ((uint64_t)n_new + block - 2u) / block + 1u);
    std::lock_guard<std::mutex> lk(ctx->mtx);
    (void)hipSetDevice(ctx->device);
    return tsr_launch_kv4_bounds(a, ctx->pick(stream)) ? TSR_HIP_E_HIP : TSR_HIP_OK;
}

static bool heads_ok(uint32_t D, uint32_t n_head, uint32_t n_head_kv) {
    return head_ok(D) && n_head_kv != 0u && n_head != 0u && n_head % n_head_kv == 0u && n_head / n_head_kv <= 64u &&
           (uint64_t)n_head * D <= 32768u;
}
static uint32_t blocks_of(uint32_t n_kv, uint32_t block) { return (uint32_t)(((uint64_t)n_kv + block - 1u) / block); }

// A call's workspace: the caller's, or eagerly the context's scratch, which orders calls across streams; a graph's replays
// are ordered by nobody, so that a captured call brings its own. `lk` holds the context.
static int workspace(tsr_hip_ctx * ctx, size_t need, void * ws_dev, hipStream_t s, void ** ws) {
    *ws = ws_dev;
    if (ws_dev != nullptr || need == 0u) return TSR_HIP_OK;
    if (tsr_capturing(s)) return TSR_HIP_E_ARG;
    const int rc = ctx->scratch.reserve(need, s);
    *ws = ctx->scratch.ptr;
    return rc;
}

size_t tsr_hip_kv4_select_ws(tsr_hip_ctx * ctx, uint32_t T, uint32_t n_head_kv, uint32_t block, uint32_t n_kv) {
    if (ctx == nullptr || T == 0u || T > 65535u || n_head_kv == 0u || n_head_kv > 512u || !block_ok(block) || n_kv > 0x7FFFFFFFu)
        return 0u;
    return tsr::kv4_select_ws(T, n_head_kv, blocks_of(n_kv, block));
}

int tsr_hip_kv4_select(tsr_hip_ctx * ctx, const float * q_dev, uint32_t T, uint64_t q_stride, const uint32_t * bounds_dev,
                       uint32_t bounds_blocks, uint32_t D, uint32_t n_head, uint32_t n_head_kv, uint32_t block, uint32_t n_kv,
                       const uint32_t * runs_dev, uint32_t n_sel, uint32_t n_first, uint32_t n_last, int32_t * blocks_dev,
                       void * ws_dev, size_t ws_bytes, void * stream) {
    if (ctx == nullptr || q_dev == nullptr || bounds_dev == nullptr || blocks_dev == nullptr || T == 0u || T > 65535u)
        return TSR_HIP_E_ARG;
    if (!heads_ok(D, n_head, n_head_kv) || !block_ok(block) || n_sel == 0u || n_sel > 65536u || n_first > n_sel || n_last > n_sel - n_first)
        return TSR_HIP_E_SHAPE;
    if (n_kv > 0x7FFFFFFFu || bounds_blocks < blocks_of(n_kv, block)) return TSR_HIP_E_RANGE;
    if ((((uintptr_t)q_dev | (uintptr_t)bounds_dev | (uintptr_t)runs_dev) & 15u) != 0u || ((uintptr_t)blocks_dev & 3u) != 0u ||
        (T > 1u && (q_stride % 4u != 0u || q_stride < (uint64_t)n_head * D)))
        return TSR_HIP_E_ARG;
    const uint32_t nb = blocks_of(n_kv, block);
    const size_t need = tsr::kv4_select_ws(T, n_head_kv, nb);
    if (ws_dev != nullptr && (ws_bytes < need || ((uintptr_t)ws_dev & 15u) != 0u)) return TSR_HIP_E_ARG;
    tsr::Kv4SelectArgs a{};
    a.q_stride = q_stride;
    a.bounds = bounds_dev;
    a.stride = bounds_blocks;
    a.D = D;
    a.G = n_head / n_head_kv;
    a.n_head_kv = n_head_kv;
    a.n_kv = n_kv;
    a.block = block;
    a.n_blocks = nb;
    a.n_sel = n_sel;
    a.n_first = n_first;
    a.n_last = n_last;
    std::lock_guard<std::mutex> lk(ctx->mtx);
    (void)hipSetDevice(ctx->device);
    hipStream_t s = ctx->pick(stream);
    void * ws = nullptr;
    const int rc = workspace(ctx, need, ws_dev, s, &ws);
    if (rc) return rc;
    a.keys = (uint64_t *)ws;
    const uint32_t step = tsr::kv4_select_tokens(T, n_head_kv, nb);
    for (uint32_t t0 = 0; t0 < T; t0 += step) {
        a.T = std::min(T - t0, step);
        a.q = q_dev + t0 * q_stride;
        a.runs = runs_dev ? runs_dev + 4u * (size_t)t0 : nullptr;
        a.blocks = blocks_dev + (size_t)t0 * n_head_kv * n_sel;
        if (tsr_launch_kv4_select(a, s)) return TSR_HIP_E_HIP;
    }
    return TSR_HIP_OK;
}

constexpr uint32_t kBlockTokens = 16000u;   // of one launch: at most 65535 tokens' groups of rows along its third axis

static bool list_ok(uint32_t n_sel, uint32_t block) { return block_ok(block) && n_sel != 0u && n_sel <= 65536u; }

size_t tsr_hip_flash_attn_kv4_blocks_ws(tsr_hip_ctx * ctx, uint32_t T, uint32_t D, uint32_t n_head, uint32_t n_head_kv, uint32_t n_sel,
                                        uint32_t block) {
    if (ctx == nullptr || T == 0u || T > 65535u || !heads_ok(D, n_head, n_head_kv) || !list_ok(n_sel, block)) return 0u;
    return tsr::attn4_blocks_plan(T, D, n_head, n_head_kv, n_sel, block, (uint32_t)ctx->n_cu).ws_bytes;
}

int tsr_hip_flash_attn_kv4_blocks(tsr_hip_ctx * ctx, const float * q_dev, uint32_t T, uint64_t q_stride, const tsr_hip_kv * kc,
                                  const tsr_hip_kv * vc, uint32_t D, uint32_t n_head, uint32_t n_head_kv, float scale, uint32_t n_kv,
                                  const uint32_t * runs_dev, const int32_t * blocks_dev, uint32_t n_sel, uint32_t block, float * out_dev,
                                  uint64_t out_stride, void * ws_dev, size_t ws_bytes, void * stream) {
    if (ctx == nullptr || q_dev == nullptr || kc == nullptr || vc == nullptr || out_dev == nullptr || blocks_dev == nullptr ||
        T == 0u || T > 65535u)
        return TSR_HIP_E_ARG;
    if (!heads_ok(D, n_head, n_head_kv) || !list_ok(n_sel, block)) return TSR_HIP_E_SHAPE;
    if (!(scale > 0.0f) || !std::isnormal(scale)) return TSR_HIP_E_SHAPE;
    if (kc->type == TSR_HIP_KV_Q8_0 || kc->type != vc->type) return TSR_HIP_E_FMT;
    const uint32_t E = n_head_kv * D, K = n_head * D;
    if (kc->E != E || vc->E != E || kc->kv_size != vc->kv_size) return TSR_HIP_E_SHAPE;
    if (n_kv > kc->kv_size) return TSR_HIP_E_RANGE;
    if ((((uintptr_t)q_dev | (uintptr_t)out_dev | (uintptr_t)runs_dev) & 15u) != 0u || ((uintptr_t)blocks_dev & 3u) != 0u ||
        (T > 1u && (q_stride % 4u != 0u || q_stride < K || out_stride % 4u != 0u || out_stride < K)))
        return TSR_HIP_E_ARG;
    const tsr::Attn4BlocksPlan p = tsr::attn4_blocks_plan(T, D, n_head, n_head_kv, n_sel, block, (uint32_t)ctx->n_cu);
    if (ws_dev != nullptr && (ws_bytes < p.ws_bytes || ((uintptr_t)ws_dev & 15u) != 0u)) return TSR_HIP_E_ARG;
    tsr::Attn4BlocksArgs b{};
    tsr::Attn4Args & a = b.a;
    a.q_stride = q_stride;
    a.k = kc->dev;
    a.v = vc->dev;
    a.out_stride = out_stride;
    a.type = kc->type;
    a.D = D;
    a.G = n_head / n_head_kv;
    a.n_head_kv = n_head_kv;
    a.n_kv = n_kv;
    a.n_tiles = tsr::kv4_tiles(kc->kv_size);
    a.S = p.S;
    a.scale = scale;
    b.n_sel = n_sel;
    b.block = block;
    std::lock_guard<std::mutex> lk(ctx->mtx);
    (void)hipSetDevice(ctx->device);
    hipStream_t s = ctx->pick(stream);
    void * ws = nullptr;
    const int rc = workspace(ctx, p.ws_bytes, ws_dev, s, &ws);
    if (rc) return rc;
    a.part = (float *)ws;
    ctx->ctr.flash_attn_calls++;
    ctx->ctr.flash_attn_kv_bytes += (uint64_t)std::min<uint64_t>(n_kv, (uint64_t)n_sel * block) * (E / 32u) * tsr::kv4_block_bytes(kc->type) * 2u;
    for (uint32_t t0 = 0; t0 < T; t0 += kBlockTokens) {            // (S is 1 where there are several)
        a.T = std::min(T - t0, kBlockTokens);
        a.q = q_dev + t0 * q_stride;
        a.out = out_dev + t0 * out_stride;
        a.runs = runs_dev ? runs_dev + 4u * (size_t)t0 : nullptr;
        b.blocks = blocks_dev + (size_t)t0 * n_head_kv * n_sel;
        if (tsr_launch_attn4_blocks(b, p.C, s)) return TSR_HIP_E_HIP;
    }
    return TSR_HIP_OK;
}
