// attn4_plan.hpp -- how an attention call over a 4-bit cache is cut into workgroups. Plain C++.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace tsr {

constexpr uint32_t kSplitsMax = 256u;

struct Attn4Plan {
    bool split_waves;        // the four waves of a workgroup share 16 rows and take different cells; else 64 rows
    uint32_t C;              // split_waves: columns of the matrix instruction a row (k_attn4.hip)
    uint32_t S;              // splits of the cells, joined by a second launch
    size_t ws_bytes;         // partial rows of S > 1
};

// T tokens of G query heads a KV head over at most n_kv cells (tiles of 32).
inline Attn4Plan attn4_plan(uint32_t T, uint32_t D, uint32_t n_head, uint32_t n_head_kv, uint32_t n_kv, uint32_t n_cu) {
    Attn4Plan p{};
    const uint64_t R = (uint64_t)T * (n_head / n_head_kv), tiles = std::max<uint64_t>(1u, ((uint64_t)n_kv + 31u) / 32u);
    p.split_waves = (R + 63u) / 64u * n_head_kv < n_cu;
    p.C = !p.split_waves || R > 8u ? 1u : R > 4u || D == 64u ? 2u : 4u;
    const uint64_t rows = p.split_waves ? 16u / p.C : 64u, wgs = (R + rows - 1u) / rows * n_head_kv;
    const uint64_t share = p.split_waves ? 4u : 1u, most = (tiles + share - 1u) / share;
    p.S = (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>({ 2u * (uint64_t)n_cu / wgs, most, kSplitsMax }));
#ifdef TSR_TUNE
    if (getenv("TS")) p.S = atoi(getenv("TS"));
#endif
    p.ws_bytes = p.S > 1u ? 4u * (size_t)p.S * T * n_head * (2u + D) : 0u;
    return p;
}

}  // namespace tsr
