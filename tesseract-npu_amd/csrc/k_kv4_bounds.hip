// k_kv4_bounds.hip -- for every block of cells of a 4-bit K cache the smallest and largest value of each channel, as bf16
// rounded outwards: for any q, sum over channels of max(q lo, q hi) is at least the score of each of the block's cells.
//
// A quarter of a wave's lanes takes a block's cells of 64 channels (a pair of the format's blocks): a lane the cells 4 x .. 4 x + 3
// of every 16 and the 16 channels of a quarter, so that a tile is whole lines, four 16-byte loads of codes and two (q4_1:
// four) of scales a lane. Codes become f16 pairs by an AND with an OR (q4_1: and a packed operation), values by one exact
// product sum, two cells at a time go into a minimum and a maximum of three. The four lanes that share channels then hand each
// other half of what is left, twice, and every lane ends with four channels and stores them: x is the lane's bits 4 and 5, where
// a step is one swap of registers between rows and one comparison a pair.
//
// Bound: 131071 cells of 1024 values in blocks of 64 (84 MB) take 20.0 us, 4.2 TB/s (a large copy runs at 4.65): vector
// instructions, 425 a tile of four units, hide most of what memory leaves. With eight lanes a unit and the exchange by selects it was
// 25.8 us (770 instructions a tile for as much), with swaps 22.7. Few blocks are a launch.
//
// Scales that are not finite count as the largest of their type, so that bounds are finite and such a block is looked at.
#include <algorithm>

#include "kernels.hpp"
#include "kv4.hpp"
#include "tsr_dev.hpp"

namespace tsr {

// bf16 bits of the nearest value not above (below) x.
__device__ __forceinline__ uint32_t bf16_below(float x) {
    const uint32_t u = fb(x), cut = u >> 16;
    return cut + ((u & 0xFFFFu) != 0u && (u >> 31) != 0u ? 1u : 0u);
}
__device__ __forceinline__ uint32_t bf16_above(float x) {
    const uint32_t u = fb(x), cut = u >> 16;
    return cut + ((u & 0xFFFFu) != 0u && (u >> 31) == 0u ? 1u : 0u);
}
__device__ __forceinline__ float finite_scale(uint32_t w, int i) {
    return __builtin_amdgcn_fmed3f((float)__builtin_bit_cast(_Float16, (uint16_t)(w >> (16 * i))), -65504.0f, 65504.0f);
}
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
// The nibbles at bits 0 and 16 (high: 4 and 20) of a word: q4_0 the f16 numbers 1024 + n (1024 + 16 n), q4_1 n.
template <uint32_t TYPE>
__device__ __forceinline__ h2 codes(uint32_t w, bool high, uint32_t magic) {
    uint32_t r;                                 // one operation: of its two constants only one may be a scalar register
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(high ? 0x00F000F0u : 0x000F000Fu), "v"(magic));
    const h2 x = __builtin_bit_cast(h2, r);
    if constexpr (TYPE == kKvQ4_0) return x;
    const _Float16 f = (_Float16)0.0625f, z = (_Float16)-64.0f, o = (_Float16)-1024.0f;
    return high ? __builtin_elementwise_fma(x, h2{ f, f }, h2{ z, z }) : x + h2{ o, o };
}

struct Least { float lo[16], hi[16]; };         // channel 32 (k / 8) + 16 (k / 4 % 2) + 4 g + k % 4

// A tile of 64 channels as a lane holds it: the codes of its cells 4 x + 2 i, 4 x + 2 i + 1 of group u in c[u][i] ({block 0,
// block 1} each), and the scales of its eight cells in both blocks.
template <uint32_t TYPE>
struct BoundsTile {
    uint4 c[2][2], s[2][TYPE == kKvQ4_1 ? 2 : 1];
    __device__ __forceinline__ void load(const uint8_t * t, uint32_t g, uint32_t x) {
#pragma unroll
        for (uint32_t u = 0; u < 2u; ++u)
#pragma unroll
            for (uint32_t i = 0; i < 2u; ++i) c[u][i] = *(const uint4 *)(t + 512u * u + 128u * g + 32u * x + 16u * i);
#pragma unroll
        for (uint32_t bb = 0; bb < 2u; ++bb)
#pragma unroll
            for (uint32_t i = 0; i < (TYPE == kKvQ4_1 ? 2u : 1u); ++i)
                s[bb][i] = *(const uint4 *)(t + 1024u + (TYPE == kKvQ4_1 ? 8u : 4u) * (8u * x + 4u * bb) + 16u * i);
    }
    // {d, d of the next cell} of cells 4 x + 2 i, .. of group u, and {m, m}
    __device__ __forceinline__ uint32_t d(int bb, int u, int i) const {
        const uint4 & w = s[bb][TYPE == kKvQ4_1 ? u : 0];
        if constexpr (TYPE == kKvQ4_1) return i ? w.z : w.x;
        return u ? (i ? w.w : w.z) : (i ? w.y : w.x);
    }
    __device__ __forceinline__ uint32_t m(int bb, int u, int i) const {
        const uint4 & w = s[bb][TYPE == kKvQ4_1 ? u : 0];
        return i ? w.w : w.y;
    }
};

template <uint32_t TYPE, bool WHOLE>
__device__ __forceinline__ void bounds_of_tile(Least & b, const BoundsTile<TYPE> & t, uint32_t x, uint32_t cells, uint32_t magic) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 & c = t.c[u][i];
            const uint32_t cell = 16u * u + 4u * x + 2u * i;
            const bool in0 = WHOLE || cell < cells, in1 = WHOLE || cell + 1u < cells;
#pragma unroll
            for (int bb = 0; bb < 2; ++bb) {
                const uint32_t w0 = bb ? c.y : c.x, w1 = bb ? c.w : c.z;
                const float d0 = finite_scale(t.d(bb, u, i), 0), d1 = finite_scale(t.d(bb, u, i), 1);
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    // q4_0: d (1024 + n) - 1032 d and d / 16 (1024 + 16 n) - 72 d, all exact
                    const float e0 = TYPE == kKvQ4_0 && hh ? 0.0625f * d0 : d0, e1 = TYPE == kKvQ4_0 && hh ? 0.0625f * d1 : d1;
                    const float m0 = TYPE == kKvQ4_1 ? finite_scale(t.m(bb, u, i), 0) : (hh ? -72.0f : -1032.0f) * d0;
                    const float m1 = TYPE == kKvQ4_1 ? finite_scale(t.m(bb, u, i), 1) : (hh ? -72.0f : -1032.0f) * d1;
                    const h2 n0[2] = { codes<TYPE>(w0, hh, magic), codes<TYPE>(w0 >> 8, hh, magic) };
                    const h2 n1[2] = { codes<TYPE>(w1, hh, magic), codes<TYPE>(w1 >> 8, hh, magic) };
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int k = 8 * bb + 4 * hh + j;
                        const float v0 = __builtin_fmaf(e0, (float)n0[j & 1][j >> 1], m0), v1 = __builtin_fmaf(e1, (float)n1[j & 1][j >> 1], m1);
                        b.lo[k] = fminf(fminf(b.lo[k], in0 ? v0 : __builtin_inff()), in1 ? v1 : __builtin_inff());
                        b.hi[k] = fmaxf(fmaxf(b.hi[k], in0 ? v0 : -__builtin_inff()), in1 ? v1 : -__builtin_inff());
                    }
                }
            }
        }
}

// One step of the exchange, between lanes that differ in bit 4 (5): those that have it keep the second half of N values.
template <int BIT, int N>
__device__ __forceinline__ void hand_over(Least & b) {
    auto swap = [](float x, float y) {
        auto r = BIT == 4 ? __builtin_amdgcn_permlane16_swap(fb(x), fb(y), false, false) : __builtin_amdgcn_permlane32_swap(fb(x), fb(y), false, false);
        return make_float2(bf(r[0]), bf(r[1]));
    };
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
        const float2 lo = swap(b.lo[k], b.lo[k + N / 2]), hi = swap(b.hi[k], b.hi[k + N / 2]);
        b.lo[k] = __builtin_amdgcn_fmed3f(lo.x, lo.y, -__builtin_inff());   // the smaller (fminf quiets its operands first)
        b.hi[k] = __builtin_amdgcn_fmed3f(hi.x, hi.y, __builtin_inff());
    }
}

template <uint32_t TYPE>
__global__ __launch_bounds__(256, 3) void k_kv4_bounds(Kv4BoundsArgs a) {
    const uint32_t lane = threadIdx.x & 63u, x = lane >> 4, g = lane & 3u;
    const uint32_t planes = a.E / 64u, step = 16u * gridDim.x;
    uint32_t first = 0u, end = a.n_kv;
    if (a.cells != nullptr) {
        end = min(end, a.cells[1]);
        if (a.cells[0] >= end) return;
        first = a.cells[0] / a.block;
    }
    const uint32_t units = min(a.n_blocks, (end + a.block - 1u) / a.block - first) * planes;
    uint32_t unit = blockIdx.x * 16u + 4u * (threadIdx.x / 64u) + ((lane >> 2) & 3u);
    if (unit >= units) return;                                     // (all the lanes that a swap joins)
    uint32_t b, plane, magic;
    auto place = [&](uint32_t u) {                                 // the unit's first tile
        const uint32_t i = u / planes;
        b = first + i;
        plane = u - i * planes;
        return a.k + kKv4Header + ((size_t)plane * a.n_tiles + b * (a.block / 32u)) * kv4_tile_bytes(TYPE);
    };
    asm("v_mov_b32 %0, 0x64006400" : "=v"(magic));                 // f16 1024, twice, in a vector register
    const uint8_t * t = place(unit);
    BoundsTile<TYPE> cur, next;
    cur.load(t, g, x);
    for (;;) {
        const uint32_t n = min(end - b * a.block, a.block), per = a.D / 64u, h = plane / per;
        uint32_t * out = a.bounds + ((size_t)h * a.stride + b) * a.D + 64u * (plane - h * per);
        const bool last = units - unit <= step;
        Least w;
#pragma unroll
        for (int k = 0; k < 16; ++k) { w.lo[k] = __builtin_inff(); w.hi[k] = -__builtin_inff(); }
        for (uint32_t at = 0u;; at += 32u) {                       // each tile behind the loads of the next one
            const bool more = at + 32u < n;
            if (more) t += kv4_tile_bytes(TYPE);
            else if (!last) t = place(unit + step);
            if (more || !last) next.load(t, g, x);
            if (at + 32u <= n) bounds_of_tile<TYPE, true>(w, cur, x, 32u, magic);
            else bounds_of_tile<TYPE, false>(w, cur, x, n - at, magic);
            cur = next;
            if (!more) break;
        }
        hand_over<5, 16>(w);
        hand_over<4, 8>(w);
        auto word = [&](int k) { return bf16_below(w.lo[k]) | bf16_above(w.hi[k]) << 16; };
        *(uint4 *)(out + 32u * (x >> 1) + 16u * (x & 1u) + 4u * g) = make_uint4(word(0), word(1), word(2), word(3));
        if (last) return;
        unit += step;
    }
}

}  // namespace tsr

int tsr_launch_kv4_bounds(const tsr::Kv4BoundsArgs & a, hipStream_t s) {
    const uint64_t units = (uint64_t)a.n_blocks * (a.E / 64u);
    const dim3 grid((uint32_t)std::min<uint64_t>((units + 15u) / 16u, 768u));
    if (a.type == tsr::kKvQ4_0) hipLaunchKernelGGL(tsr::k_kv4_bounds<tsr::kKvQ4_0>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(tsr::k_kv4_bounds<tsr::kKvQ4_1>, grid, dim3(256), 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
