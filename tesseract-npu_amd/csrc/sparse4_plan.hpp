// sparse4_plan.hpp -- how the calls of sparse attention over a 4-bit cache are cut. Plain C++.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace tsr {

// Block selection: a key of 8 bytes a KV head and block. The tokens of a launch, so that their keys take at most 64 MiB (or are one
// token's) and its grid's second axis fits, and the workspace, which never falls with more tokens or blocks.
constexpr uint64_t kSelectKeys = (uint64_t)64 << 20;
constexpr uint32_t kSelectTokens = 32768u;
constexpr uint64_t kv4_token_keys(uint32_t n_head_kv, uint64_t n_blocks) { return 8u * std::max<uint64_t>(1u, n_blocks) * n_head_kv; }
inline uint32_t kv4_select_tokens(uint32_t T, uint32_t n_head_kv, uint64_t n_blocks) {
    return (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>({ T, kSelectKeys / kv4_token_keys(n_head_kv, n_blocks), kSelectTokens }));
}
inline size_t kv4_select_ws(uint32_t T, uint32_t n_head_kv, uint64_t n_blocks) {
    const uint64_t one = kv4_token_keys(n_head_kv, n_blocks);
    return (size_t)std::min(std::min(T, kSelectTokens) * one, std::max(kSelectKeys, one));
}

// Attention over listed blocks: columns of the matrix instruction a row (attn4.hpp) and splits of a token's tiles.
struct Attn4BlocksPlan {
    uint32_t C, S;
    size_t ws_bytes;
};
inline Attn4BlocksPlan attn4_blocks_plan(uint32_t T, uint32_t D, uint32_t n_head, uint32_t n_head_kv, uint32_t n_sel, uint32_t block,
                                         uint32_t n_cu) {
    Attn4BlocksPlan p{};
    const uint64_t G = n_head / n_head_kv, tiles = (uint64_t)n_sel * (block / 32u);
    p.C = G <= 4u && D >= 128u ? 4u : G <= 8u ? 2u : 1u;           // a workgroup's rows are one token's: as few columns as hold them
    const uint64_t rows = 16u / p.C, n = (uint64_t)T * n_head_kv * ((G + rows - 1u) / rows), fill = n_cu / n;
    // Splits fill the card, but a list of up to 20 tiles is not worth a join. Scores, cut and attention in us: 8 tokens of 8 heads of 256 over 4
    // over 32 tiles, S 1, 2, 4: 33.3, 30.8, 28.4; 32 such tokens S 1, 2: 38.9, 43.5; a token of 32 heads of 128 over 8 over 64
    // tiles S 1, 8, 16: 34.0, 26.6, 26.9; one of a head of 512 S 1, 8: 87, 42.8.
    const uint64_t S = tiles <= 20u ? 1u : fill;
    p.S = (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>({ S, (tiles + 3u) / 4u, 256u }));
    p.ws_bytes = p.S > 1u ? 4u * (size_t)p.S * T * n_head * (2u + D) : 0u;
    return p;
}

}  // namespace tsr
