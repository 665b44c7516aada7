// k_kv4_bounds.hip -- for every block of cells of a 4-bit K cache the smallest and largest value of each channel, as bf16
// rounded outwards: for any q, sum over channels of max(q lo, q hi) is at least the score of each of the block's cells.
//
// Half a wave takes a block's cells of 64 channels (a pair of the format's blocks): a lane the cells 2 x and 2 x + 1 of
// every 16 and the 16 channels of a quarter, so that a tile is whole lines, two 16-byte loads of codes and two (q4_1: four) of
// scales a lane. Codes become f32 by a byte conversion, values by one exact product sum, two cells at a time go into a minimum
// and a maximum of three. The eight lanes that share channels then hand each other half of what is left, three times: every
// lane ends with two channels and stores them.
//
// Scales that are not finite count as the largest of their type, so that bounds are finite and such a block is looked at.
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
__device__ __forceinline__ float byte_f32(uint32_t w, int i) { return (float)((w >> (8 * i)) & 255u); }   // v_cvt_f32_ubyte

struct Least { float lo[16], hi[16]; };         // channel 32 (k / 8) + 16 (k / 4 % 2) + 4 g + k % 4

template <uint32_t TYPE, bool WHOLE>
__device__ __forceinline__ void bounds_of_tile(Least & b, const uint8_t * t, uint32_t l, uint32_t cells) {
    const uint32_t x = l & 7u;                                      // pair of cells of 16
    const uint4 c0 = *(const uint4 *)(t + 16u * l), c1 = *(const uint4 *)(t + 512u + 16u * l);
    uint32_t d[2][2], m[2][2];                                     // [block][group of 16 cells]
#pragma unroll
    for (int bb = 0; bb < 2; ++bb) {
        const uint8_t * s = t + 1024u + (TYPE == kKvQ4_1 ? 8u : 4u) * (8u * (x >> 1) + 4u * bb);
        const uint4 u = *(const uint4 *)s;
        if constexpr (TYPE == kKvQ4_1) {
            const uint4 v = *(const uint4 *)(s + 16u);
            d[bb][0] = x & 1u ? u.z : u.x;
            m[bb][0] = x & 1u ? u.w : u.y;
            d[bb][1] = x & 1u ? v.z : v.x;
            m[bb][1] = x & 1u ? v.w : v.y;
        } else {
            d[bb][0] = x & 1u ? u.y : u.x;
            d[bb][1] = x & 1u ? u.w : u.z;
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const uint4 & c = u ? c1 : c0;
        const bool in0 = WHOLE || 16u * u + 2u * x < cells, in1 = WHOLE || 16u * u + 2u * x + 1u < cells;
#pragma unroll
        for (int bb = 0; bb < 2; ++bb) {
            const uint32_t w0 = bb ? c.y : c.x, w1 = bb ? c.w : c.z;
            const float d0 = finite_scale(d[bb][u], 0), d1 = finite_scale(d[bb][u], 1);
            const float m0 = TYPE == kKvQ4_1 ? finite_scale(m[bb][u], 0) : -8.0f * d0;
            const float m1 = TYPE == kKvQ4_1 ? finite_scale(m[bb][u], 1) : -8.0f * d1;
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const uint32_t n0 = (w0 >> (4 * hh)) & 0x0F0F0F0Fu, n1 = (w1 >> (4 * hh)) & 0x0F0F0F0Fu;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k = 8 * bb + 4 * hh + j;
                    const float v0 = __builtin_fmaf(d0, byte_f32(n0, j), m0), v1 = __builtin_fmaf(d1, byte_f32(n1, j), m1);
                    b.lo[k] = fminf(fminf(b.lo[k], in0 ? v0 : __builtin_inff()), in1 ? v1 : __builtin_inff());
                    b.hi[k] = fmaxf(fmaxf(b.hi[k], in0 ? v0 : -__builtin_inff()), in1 ? v1 : -__builtin_inff());
                }
            }
        }
    }
}

// One step of the exchange: a lane whose `up` is set keeps the second half of its N values, its partner the first.
template <int CTRL, int N>
__device__ __forceinline__ void hand_over(Least & b, bool up) {
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
        const float lo = up ? b.lo[k + N / 2] : b.lo[k], lo_out = up ? b.lo[k] : b.lo[k + N / 2];
        const float hi = up ? b.hi[k + N / 2] : b.hi[k], hi_out = up ? b.hi[k] : b.hi[k + N / 2];
        b.lo[k] = fminf(lo, dpp_f<CTRL>(lo_out));
        b.hi[k] = fmaxf(hi, dpp_f<CTRL>(hi_out));
    }
}

template <uint32_t TYPE>
__global__ __launch_bounds__(256) void k_kv4_bounds(Kv4BoundsArgs a) {
    const uint32_t planes = a.E / 64u, unit = blockIdx.x * 8u + threadIdx.x / 32u, l = threadIdx.x & 31u;
    const uint32_t i = unit / planes, plane = unit - i * planes;
    uint32_t first = 0u, end = a.n_kv;
    if (a.cells != nullptr) {
        end = min(end, a.cells[1]);
        if (a.cells[0] >= end) return;
        first = a.cells[0] / a.block;
    }
    const uint32_t b = first + i;
    if (i >= a.n_blocks || b >= (end + a.block - 1u) / a.block) return;
    const uint32_t c0 = b * a.block, n = min(end - c0, a.block);   // (c0 < end)
    const uint8_t * t = a.k + kKv4Header + ((size_t)plane * a.n_tiles + c0 / 32u) * kv4_tile_bytes(TYPE);
    Least w;
#pragma unroll
    for (int k = 0; k < 16; ++k) { w.lo[k] = __builtin_inff(); w.hi[k] = -__builtin_inff(); }
    uint32_t at = 0u;
#pragma unroll 2
    for (; at + 32u <= n; at += 32u, t += kv4_tile_bytes(TYPE)) bounds_of_tile<TYPE, true>(w, t, l, 32u);
    if (at < n) bounds_of_tile<TYPE, false>(w, t, l, n - at);
    hand_over<kDppRowHalfMirror, 16>(w, (l & 4u) != 0u);
    hand_over<kDppXor2, 8>(w, (l & 2u) != 0u);
    hand_over<kDppXor1, 4>(w, (l & 1u) != 0u);
    const uint32_t c = 32u * ((l >> 2) & 1u) + 16u * ((l >> 1) & 1u) + 4u * (l >> 3) + 2u * (l & 1u);
    const uint32_t per = a.D / 64u, h = plane / per;
    uint32_t * out = a.bounds + ((size_t)h * a.stride + b) * a.D + 64u * (plane - h * per) + c;
    *(uint2 *)out = make_uint2(bf16_below(w.lo[0]) | bf16_above(w.hi[0]) << 16, bf16_below(w.lo[1]) | bf16_above(w.hi[1]) << 16);
}

}  // namespace tsr

int tsr_launch_kv4_bounds(const tsr::Kv4BoundsArgs & a, hipStream_t s) {
    const uint64_t units = (uint64_t)a.n_blocks * (a.E / 64u);
    const dim3 grid((uint32_t)((units + 7u) / 8u));
    if (a.type == tsr::kKvQ4_0) hipLaunchKernelGGL(tsr::k_kv4_bounds<tsr::kKvQ4_0>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(tsr::k_kv4_bounds<tsr::kKvQ4_1>, grid, dim3(256), 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
