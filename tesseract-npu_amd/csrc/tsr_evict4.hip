// tsr_evict4.hip -- host side of eviction by attention weight: the weights that cells of a 4-bit K cache gather.
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
    return tsr::weights4_plan(T, D, n_head, n_head_kv, n_kv, (uint32_t)ctx->n_cu).ws_bytes;
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
    if (ws_dev != nullptr && (ws_bytes < p.ws_bytes || ((uintptr_t)ws_dev & 15u) != 0u)) return TSR_HIP_E_ARG;
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
