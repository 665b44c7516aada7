// kv4.hpp -- KV caches of 4-bit blocks (q4_0, q4_1): the formats and the device layout, shared by the store, the read
// and the attention kernels.
//
// A block is 32 consecutive values of a cell's row, as ggml lays it out: q4_0 {f16 d, 16 bytes} stands for
// d (n - 8), q4_1 {f16 d, f16 m, 16 bytes} for d n + m; byte j holds n of value j (low nibble) and of value j + 16.
//
// Device layout of one plane: for every pair of blocks (64 values of a row) a run of tiles of 32 cells, 1024 bytes of
// codes and 4 (q4_1: 8) bytes of scales a cell. A tile is the operands of the matrix instruction 16x16x32 as its lanes
// hold them, so that a wave loads them with full-width loads and unpacks them with a mask alone (k_attn4.hip):
//   K codes  [2 groups of 16 cells][lane 16 g + cell][2 blocks] words: bytes 4 g .. 4 g + 3 of the block
//   V codes  [lane 16 g + j][2 blocks][2 groups of 16 cells] words: byte j of the block for cells 4 g + 0, 2, 1, 3
//   scales   [g][2 blocks][2 groups of 16 cells][2] words {d of cell 4 g + 2 x, of the next one} (q4_1: and {m, m})
// One cell owns every byte that its row is stored in, so that rows are stored without reading their neighbours'.
#pragma once

#include "kernels.hpp"

namespace tsr {

constexpr uint32_t kKv4Header = 0u;                // bytes in front of a plane's first tile
__host__ __device__ constexpr uint32_t kv4_tile_bytes(uint32_t type) { return type == kKvQ4_1 ? 1280u : 1152u; }
__host__ __device__ constexpr uint32_t kv4_block_bytes(uint32_t type) { return type == kKvQ4_1 ? 20u : 18u; }
__host__ __device__ inline uint32_t kv4_tiles(uint32_t kv_size) { return (uint32_t)(((uint64_t)kv_size + 31u) / 32u); }

// Byte offset in the plane of the tile that holds block b of cell `cell`.
__host__ __device__ inline size_t kv4_tile(uint32_t type, uint32_t n_tiles, uint32_t cell, uint32_t b) {
    return kKv4Header + ((size_t)(b >> 1) * n_tiles + (cell >> 5)) * kv4_tile_bytes(type);
}
// Byte offsets in that tile: of code byte j (0 .. 15) of the block, and of its d (q4_1: m is 4 bytes on).
__host__ __device__ inline uint32_t kv4_code(uint32_t which, uint32_t cell, uint32_t b, uint32_t j) {
    const uint32_t s = (cell >> 4) & 1u, c = cell & 15u;
    if (which == 0u) return 512u * s + 8u * (16u * (j >> 2) + c) + 4u * (b & 1u) + (j & 3u);
    const uint32_t i = c & 3u;
    return 16u * (16u * (c >> 2) + j) + 8u * (b & 1u) + 4u * s + ((i & 1u) << 1 | i >> 1);
}
__host__ __device__ inline uint32_t kv4_scale(uint32_t type, uint32_t cell, uint32_t b) {
    const uint32_t word = 8u * ((cell >> 2) & 3u) + 4u * (b & 1u) + 2u * ((cell >> 4) & 1u) + ((cell >> 1) & 1u);
    return 1024u + (type == kKvQ4_1 ? 8u : 4u) * word + 2u * (cell & 1u);
}

}  // namespace tsr
