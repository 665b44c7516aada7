// attn4_plan.hpp -- how an attention call over a 4-bit cache is cut into workgroups. Plain C++.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace tsr {

constexpr uint32_t kSplitsMax = 256u;

// The workspace of S splits of nr rows, in floats: the splits' rows of D values, which are read and written 16 bytes at a
// time and so come first, behind them a (maximum, sum) each.
constexpr size_t attn4_part_row(uint64_t nr, uint32_t D, uint32_t split, uint64_t row) { return (split * nr + row) * D; }
constexpr size_t attn4_part_sum(uint64_t nr, uint32_t D, uint32_t S, uint32_t split, uint64_t row) {
    return attn4_part_row(nr, D, S, 0u) + 2u * (split * nr + row);
}

struct Attn4Plan {
    uint32_t C;              // columns of the matrix instruction a row (k_attn4.hip): 16 / C rows a group
    uint32_t NT;             // groups of rows of a workgroup
    uint32_t S;              // splits of the cells, joined by a second launch
    size_t ws_bytes;         // partial rows of S > 1
};

// T tokens of n_head query heads over at most n_kv cells (tiles of 32).
inline Attn4Plan attn4_plan(uint32_t T, uint32_t D, uint32_t n_head, uint32_t n_head_kv, uint32_t n_kv, uint32_t n_cu) {
    Attn4Plan p{};
    const uint64_t G = n_head / n_head_kv, R = T * G, tiles = std::max<uint64_t>(1u, ((uint64_t)n_kv + 31u) / 32u);
    auto wgs = [&](uint64_t rows) { return (R + rows - 1u) / rows * n_head_kv; };
    // Several columns a row take a third less work a tile, but a group is then 4 or 8 rows and not 16. That pays for a
    // token's own query heads, and for several tokens while every group has a compute unit (the host does not know whether
    // tokens share their cells; 32 heads of 8, D 128, us with 4 and 16 rows a group): 8 tokens behind 4000 cells of one
    // sequence 15.2 / 12.6, of 8 sequences with 2000 cells each 12.4 / 16.6; 32 tokens 29.4 / 19.2 and 18.9 / 31.6; 64
    // tokens 46.9 / 29.3 and 28.1 / 51.9.
    const uint32_t C = G <= 4u && D >= 128u ? 4u : G <= 8u ? 2u : 1u;
    p.C = C > 1u && (R <= 16u / C || wgs(16u / C) <= n_cu) ? C : 1u;
    // Two groups a workgroup share the unpacking of the codes, once that leaves every compute unit two workgroups (512
    // tokens behind 1536 cells 58.9 -> 54.2 us, 2048 behind 6144 685 -> 574; 100 tokens 9.1 -> 12.9). D 256 has no
    // registers for it.
    p.NT = p.C == 1u && D <= 128u && wgs(32u) >= 2u * (uint64_t)n_cu ? 2u : 1u;
    // Splits fill the compute units with one workgroup each (a token behind 8192 cells: 16, 32, 64 splits 12.4, 11.1, 11.0
    // us), with two where a wave then still has eight tiles (131072 cells: 32, 64, 96 splits 37.3, 34.7, 35.4). A split is
    // a second launch and a pass through memory, about the time of five tiles of a wave: none below 20 tiles (512 cells 7.7
    // us in one piece, 8.5 in four), and none where half the compute units have work (300 tokens 35 -> 41). Several
    // tokens behind many cells are mostly sequences of their own and of all lengths, and a group waits for its longest:
    // two workgroups a compute unit from 8192 cells on (64 tokens of up to 2000 cells, 128 groups: 2, 4, 8 splits 52.2,
    // 43.4, 40.8; 96, 192 groups: 1, 2, 4 splits 83, 70, 57; 64 tokens of one sequence behind 1000 cells 15.8, 18.8, 20.9
    // with 1, 2, 4), but not where a group is one token's and each unit has one (32 tokens of up to 1000 cells: 11.4, 15.4).
    const uint64_t n = wgs(16u / p.C * p.NT), fill = n_cu / n;
    const bool twice = n <= n_cu && (p.C == 1u || n < n_cu) && tiles >= std::max<uint64_t>(T <= 2u ? 0u : 256u, 64u * fill);
    const uint64_t S = tiles <= 20u ? 1u : twice ? (2u * (uint64_t)n_cu + n - 1u) / n : fill;
    p.S = (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>({ S, (tiles + 3u) / 4u, kSplitsMax }));
    p.ws_bytes = p.S > 1u ? 4u * (size_t)p.S * T * n_head * (2u + D) : 0u;
    return p;
}

}  // namespace tsr
