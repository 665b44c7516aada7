// weights4_plan.hpp -- how a call that sums attention weights a cell is cut, and its workspace. Plain C++.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace tsr {

constexpr uint32_t kWeightsSplits = 64u;
constexpr uint32_t kWeightsTokens = 16000u;           // of a launch: row sets of 16 fit a grid
constexpr uint32_t kTwoGroups = 64u, kFourGroups = 256u;   // products a SIMD from which a workgroup has two, four groups of rows
constexpr uint64_t kWeightsSums = (uint64_t)64 << 20; // bytes of a launch's sums, or one token's

struct Weights4Plan {
    uint32_t NT;             // groups of 16 rows of a workgroup
    uint32_t tokens;         // of a launch
    uint32_t n_rg;           // workgroups' row sets of a KV head
    uint32_t S;              // splits of the cells
    uint32_t n_pad;          // cells in whole tiles
    uint32_t one;            // workgroups of the form with a wave a KV head (0: not that form)
    size_t sums;             // byte offset of the sums behind the (maximum, sum) pairs
    size_t ws_bytes;
};

// (maximum, sum) of row r of a KV head's row set in one split, and the sums over a row set's rows for every cell.
constexpr size_t weights4_pair(const Weights4Plan & p, uint32_t n_head_kv, uint32_t split, uint32_t h, uint32_t rg, uint32_t r) {
    return ((size_t)split * n_head_kv * p.n_rg + (size_t)h * p.n_rg + rg) * (16u * p.NT) + r;
}

inline Weights4Plan weights4_plan(uint32_t T, uint32_t D, uint32_t n_head, uint32_t n_head_kv, uint32_t n_kv, uint32_t n_cu) {
    Weights4Plan p{};
    const uint64_t G = n_head / n_head_kv, tiles = std::max<uint64_t>(1u, ((uint64_t)n_kv + 31u) / 32u);
    // More groups of rows share the unpacking of a tile's codes, fewer start sooner (their queries' pieces are made by every workgroup).
    // By the products that a SIMD has (of 16 rows, a tile and 32 values): two groups from 64, four from 256. Microseconds of 1, 2 and 4
    // groups, 32 heads of 128 over 8 KV heads: 64 tokens behind 2048 cells 21.7, 22.9, 30.5, behind 8192 45.5, 41.4, 44.6, behind 32768 129,
    // 105, 98; 16 tokens behind 8192 22.2, 24.8, 36.0. Heads of 256 keep to one (64 tokens of 8 heads over 4, 32768 cells: 72.6, 91.1).
    const uint64_t R = T * G, groups = (R + 15u) / 16u, products = groups * n_head_kv * tiles * (D / 32u) / (4u * n_cu);
    p.NT = D > 128u || groups == 1u || products < kTwoGroups ? 1u : groups == 2u || products < kFourGroups ? 2u : 4u;
    // One group of rows of few heads: the heads' weights meet in a workgroup, a launch less, but a KV head's codes no longer come from the
    // L2 that its first pass filled. 14 heads of 64 over 2, 512 and 32768 cells: 10.1 -> 7.7 and 13.1 -> 11.1 us; 8 of 256 over 4, 4096 cells:
    // 17.6 -> 16.3; 32 of 128 over 8, 2048, 8192 and 32768 cells: 10.3 -> 9.9, 13.1 -> 12.1 to 14.4, 19.0 -> 19.9.
    p.one = groups == 1u && n_head_kv * D <= 1024u && (uint64_t)n_head_kv * D * n_kv <= (1u << 22) ? (uint32_t)std::min<uint64_t>(tiles, 2u * n_cu) : 0u;
    p.n_pad = (uint32_t)(32u * tiles);
    const uint64_t rows = 16u * p.NT, most = std::max<uint64_t>(1u, kWeightsSums / (4u * (uint64_t)p.n_pad * n_head_kv));   // row sets of a KV head
    p.tokens = (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>({ T, most * rows / G, kWeightsTokens }));
    p.n_rg = (uint32_t)((p.tokens * G + rows - 1u) / rows);
    const uint64_t n = (uint64_t)n_head_kv * p.n_rg;
    p.S = (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>({ (2u * (uint64_t)n_cu + n - 1u) / n, (tiles + 3u) / 4u, kWeightsSplits }));
    p.sums = 8u * (size_t)p.S * n * rows;
    p.ws_bytes = p.sums + 4u * (size_t)n * p.n_pad;
    return p;
}

// The workspace that callers bring: what the cut of any number of cells up to n_kv needs at most, so that one for the largest context
// does for all. The cut itself needs less where more cells make it give a workgroup more groups of rows or a launch fewer tokens.
inline size_t weights4_ws(uint32_t T, uint32_t D, uint32_t n_head, uint32_t n_head_kv, uint32_t n_kv, uint32_t n_cu) {
    const uint64_t G = n_head / n_head_kv, R = std::min(T, kWeightsTokens) * G, groups = (T * G + 15u) / 16u, all = ((uint64_t)n_kv + 31u) / 32u;
    const uint64_t a_tile = groups * n_head_kv * (D / 32u), most = D > 128u || groups == 1u ? 1u : groups == 2u ? 2u : 4u;
    size_t need = 0u;
    uint64_t below = 0u;                                           // tiles up to here are cut with fewer groups
    for (uint64_t NT = 1u; NT <= most && (need == 0u || below < all); NT *= 2u) {
        const uint64_t tiles = NT == most ? all : std::min(all, ((NT == 1u ? kTwoGroups : kFourGroups) * 4u * (uint64_t)n_cu - 1u) / a_tile);
        below = tiles;
        if (tiles == 0u) continue;
        // S n <= 2 n_cu + n of every cut; row sets as the largest launch has them, or as many as 64 MiB hold
        const uint64_t rows = 16u * NT, sets = (R + rows - 1u) / rows * n_head_kv, one = (G + rows - 1u) / rows * n_head_kv;
        const uint64_t pairs = rows * std::min(sets * std::min<uint64_t>(kWeightsSplits, (tiles + 3u) / 4u), 2u * (uint64_t)n_cu + sets);
        need = std::max<size_t>(need, 8u * pairs + std::min(128u * tiles * sets, std::max(kWeightsSums, 128u * tiles * one)));
    }
    return need;
}

}  // namespace tsr
