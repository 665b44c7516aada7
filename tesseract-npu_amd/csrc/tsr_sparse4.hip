// tsr_sparse4.hip -- host side of the sparse attention over 4-bit KV caches: the bounds of a K cache's blocks.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <mutex>

#include "kernels.hpp"
#include "kv4.hpp"
#include "runtime.hpp"
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
