// tsr_kv4.hip -- host side of the attention over 4-bit KV caches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "attn4_plan.hpp"
#include "kernels.hpp"
#include "kv4.hpp"
#include "runtime.hpp"
#include "tsr_hip.h"

constexpr uint32_t kTokens = 16000u;     // of one launch

static bool shape_ok(uint32_t D, uint32_t n_head, uint32_t n_head_kv) {
    return (D == 64u || D == 128u || D == 256u || D == 512u) && n_head_kv != 0u && n_head != 0u && n_head % n_head_kv == 0u &&
           n_head / n_head_kv <= 64u && (uint64_t)n_head * D <= 32768u;
}

size_t tsr_hip_flash_attn_kv4_ws(tsr_hip_ctx * ctx, uint32_t T, uint32_t D, uint32_t n_head, uint32_t n_head_kv,
                                 uint32_t n_kv) {
    if (ctx == nullptr || T == 0u || T > 65535u || !shape_ok(D, n_head, n_head_kv)) return 0u;
    return tsr::attn4_plan(T, D, n_head, n_head_kv, n_kv, (uint32_t)ctx->n_cu).ws_bytes;
}

int tsr_hip_flash_attn_kv4(tsr_hip_ctx * ctx, const float * q_dev, uint32_t T, uint64_t q_stride, const tsr_hip_kv * kc,
                           const tsr_hip_kv * vc, uint32_t D, uint32_t n_head, uint32_t n_head_kv, float scale,
                           uint32_t n_kv, const uint32_t * runs_dev, const uint16_t * mask_f16_dev, uint64_t mask_stride,
                           float * out_dev, uint64_t out_stride, void * ws_dev, size_t ws_bytes, void * stream) {
    if (ctx == nullptr || q_dev == nullptr || kc == nullptr || vc == nullptr || out_dev == nullptr || T == 0u)
        return TSR_HIP_E_ARG;
    if (!shape_ok(D, n_head, n_head_kv)) return TSR_HIP_E_SHAPE;
    if (!(scale > 0.0f) || !std::isnormal(scale)) return TSR_HIP_E_SHAPE;
    if (kc->type == TSR_HIP_KV_Q8_0 || kc->type != vc->type) return TSR_HIP_E_FMT;
    const uint32_t E = n_head_kv * D, K = n_head * D;
    if (kc->E != E || vc->E != E || kc->kv_size != vc->kv_size) return TSR_HIP_E_SHAPE;
    if (n_kv > kc->kv_size) return TSR_HIP_E_RANGE;
    if (T > 65535u || (((uintptr_t)q_dev | (uintptr_t)out_dev | (uintptr_t)runs_dev) & 15u) != 0u ||
        ((uintptr_t)mask_f16_dev & 1u) != 0u || (T > 1u && (q_stride % 4u != 0u || q_stride < K || out_stride % 4u != 0u ||
                                                            out_stride < K || (mask_f16_dev && mask_stride < n_kv))))
        return TSR_HIP_E_ARG;
    const tsr::Attn4Plan p = tsr::attn4_plan(T, D, n_head, n_head_kv, n_kv, (uint32_t)ctx->n_cu);   // (S 1 beyond kTokens)
    if (ws_dev != nullptr && (ws_bytes < p.ws_bytes || ((uintptr_t)ws_dev & 15u) != 0u)) return TSR_HIP_E_ARG;
    tsr::Attn4Args a{};
    a.q = q_dev;
    a.q_stride = q_stride;
    a.k = kc->dev;
    a.v = vc->dev;
    a.runs = runs_dev;
    a.mask = mask_f16_dev;
    a.mask_stride = mask_stride;
    a.mask_by4 = (((uintptr_t)mask_f16_dev | (T > 1u ? 2u * mask_stride : 0u)) & 7u) == 0u ? 1u : 0u;
    a.out = out_dev;
    a.out_stride = out_stride;
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
    a.part = (float *)ws_dev;
    if (ws_dev == nullptr && p.ws_bytes != 0u) {
        // the context's scratch orders eager calls across streams; a graph's replays are ordered by nobody, so that a
        // captured call brings its own workspace
        if (tsr_capturing(s)) return TSR_HIP_E_ARG;
        const int rc = ctx->scratch.reserve(p.ws_bytes, s);
        if (rc) return rc;
        a.part = (float *)ctx->scratch.ptr;
    }
    ctx->ctr.flash_attn_calls++;
    ctx->ctr.flash_attn_kv_bytes += (uint64_t)n_kv * (E / 32u) * tsr::kv4_block_bytes(kc->type) * 2u;
    // (a launch holds 65535 groups of at least 16 rows along its third axis: 16000 tokens of up to 64 query heads)
    for (uint32_t t0 = 0; t0 < T; t0 += kTokens) {
        a.T = std::min(T - t0, kTokens);
        a.q = q_dev + t0 * q_stride;
        a.out = out_dev + t0 * out_stride;
        if (runs_dev) a.runs = runs_dev + 4u * (size_t)t0;
        if (mask_f16_dev) a.mask = mask_f16_dev + t0 * mask_stride;
        if (tsr_launch_attn4(a, p, s)) return TSR_HIP_E_HIP;
    }
    return TSR_HIP_OK;
}
