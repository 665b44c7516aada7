// The layout of 4-bit KV planes (csrc/kv4.hpp) and the cuts of an attention call over them (csrc/attn4_plan.hpp): every
// byte of a cell's image has a place of its own inside the plane, and every call gets a launch that the kernels offer.
#include <hip/hip_runtime.h>

#include "attn4_plan.hpp"
#include "kv4.hpp"

#include <cstdio>
#include <vector>

static int bad(const char * what, unsigned a, unsigned b, unsigned c, unsigned d) {
    printf("%s: %u %u %u %u\n", what, a, b, c, d);
    return 1;
}

static int layout(uint32_t type, uint32_t which, uint32_t E, uint32_t cells) {
    using namespace tsr;
    const uint32_t n_tiles = kv4_tiles(cells), head = kv4_block_bytes(type) - 16u;
    const size_t bytes = kKv4Header + (size_t)(E / 64u) * n_tiles * kv4_tile_bytes(type);
    std::vector<uint8_t> seen(bytes, 0);
    for (uint32_t cell = 0; cell < 32u * n_tiles; ++cell)         // (the cells that fill up the last tile, too)
        for (uint32_t b = 0; b < E / 32u; ++b)
            for (uint32_t j = 0; j < head + 16u; ++j) {
                const size_t at = kv4_tile(type, n_tiles, cell, b) +
                                  (j < head ? kv4_scale(type, cell, b) + (j & 1u) + 4u * (j >> 1) : kv4_code(which, cell, b, j - head));
                if (at < kKv4Header || at >= bytes || seen[at]++) return bad("a byte outside, or used twice", type, cell, b, j);
                if (j >= head && (kv4_code(which, cell, b, 0u) & 3u) != 0u && which == 0u) return bad("a word across words", type, cell, b, j);
            }
    for (size_t i = kKv4Header; i < bytes; ++i)
        if (!seen[i]) return bad("a byte of no cell", type, which, E, (unsigned)i);
    return 0;
}

static int plans(uint32_t & n) {
    const uint32_t Ts[] = { 1, 2, 3, 4, 5, 8, 16, 17, 33, 64, 100, 300, 512, 1000, 2048, 8192, 16000, 16001, 65535 };
    const uint32_t kvs[] = { 0, 1, 31, 32, 33, 200, 640, 641, 1000, 4096, 8192, 131071, 131072, 1u << 20, 0x7FFFFFFFu };
    for (uint32_t D : { 64u, 128u, 256u, 512u })
        for (uint32_t hkv : { 1u, 2u, 3u, 8u, 32u, 512u })
            for (uint32_t G : { 1u, 2u, 3u, 4u, 7u, 8u, 9u, 16u, 64u }) {
                if ((uint64_t)hkv * G * D > 32768u) continue;
                for (uint32_t T : Ts)
                    for (uint32_t kv : kvs) {
                        const tsr::Attn4Plan p = tsr::attn4_plan(T, D, hkv * G, hkv, kv, 256u);
                        const uint64_t tiles = kv / 32u + 1u, rows = 16u / p.C * p.NT, rounds = ((uint64_t)std::min(T, 16000u) * G + rows - 1u) / rows;
                        if (!(p.C == 1u || p.C == 2u || (p.C == 4u && D >= 128u))) return bad("columns", T, D, G, kv);
                        if (!(p.NT == 1u || (p.NT == 2u && p.C == 1u && D <= 128u))) return bad("row groups", T, D, G, kv);
                        if (rounds > 65535u) return bad("a grid too long", T, D, G, kv);
                        if (p.S == 0u || p.S > tsr::kSplitsMax || p.S > tiles || (p.S > 1u && T > 16000u)) return bad("splits", T, D, G, kv);
                        if (p.ws_bytes != (p.S > 1u ? 4u * (size_t)p.S * T * hkv * G * (2u + D) : 0u)) return bad("workspace", T, D, G, kv);
                        ++n;
                    }
            }
    return 0;
}

// r / G by a product, as the kernel has it: every row of a launch.
static int tokens() {
    for (uint32_t G = 2; G <= 64u; ++G) {
        const uint32_t inv = (uint32_t)((1ull << 32) / G) + 1u;
        for (uint32_t r = 0; r < 16000u * G; ++r)
            if (__umulhi(r, inv) != r / G) return bad("a token", r, G, 0, 0);
    }
    return 0;
}

int main() {
    for (uint32_t type : { tsr::kKvQ4_0, tsr::kKvQ4_1 })
        for (uint32_t which : { 0u, 1u })
            for (uint32_t E : { 64u, 192u })
                for (uint32_t cells : { 1u, 32u, 33u, 100u })
                    if (layout(type, which, E, cells)) return 1;
    uint32_t n = 0;
    if (plans(n) || tokens()) return 1;
    printf("%u calls cut\n", n);
    return 0;
}
