// k_kv_gather.hip -- cells of a KV cache of any type, bit for bit, as cells 0 .. n - 1 of another one or of itself.
//
// A thread makes 16 bytes of the destination's codes, from 2 cells (K) or 8 (V, where a cell owns single bytes: 16 loads of one,
// a wave's 64 in eight lines), or a word of scales. A list in ascending order has a tile's source cells close together. Bound: memory,
// and there the lines that the cells lie in, which 16 (K) or 8 (V) cells share: 16384 of 65536 cells of 1024 values (9.4 MB, of 37.7
// MB whose every line has some) take 10.2 us for K and 12.2 for V by themselves, 4.6 and 3.9 TB/s of lines.
//
// Into itself: cells may move onto one another, so that they first go to a workspace laid out like the cache's first n
// cells (with the cells that stay, where a source is none) and from there over them: K 14.6 us where another cache takes 8.4 in a
// row of calls, V 17.5 and 11.7.
#include "kernels.hpp"
#include "kv4.hpp"
#include "long_grid.hpp"
#include "tsr_dev.hpp"

namespace tsr {

// The source cell of the destination's cell i, or -1: it keeps what it has (into itself: its own cell).
__device__ __forceinline__ int64_t gather_from(const KvGatherArgs & a, uint32_t i) {
    if (i < a.n) {
        const int64_t c = a.idx[i];
        if (c >= 0 && c < (int64_t)a.src_size) return c;
        if (a.bad != nullptr && blockIdx.y == 0u) *a.bad = 1;
    }
    return i < a.stay_size ? (int64_t)i : -1;
}

constexpr uint32_t kGatherPlanes = 4u;                             // pairs of blocks a workgroup

// Workgroup (two tiles of 32 cells, pairs of blocks): where its cells come from is looked up once, then for two pairs at a time half
// of the threads makes codes, a quarter scales.
template <uint32_t TYPE, uint32_t WHICH>
__global__ __launch_bounds__(256) void k_kv4_gather(KvGatherArgs a) {
    constexpr uint32_t tb = kv4_tile_bytes(TYPE);
    __shared__ int64_t from[64];                                   // a cell's codes in its source plane; -1: none
    __shared__ uint32_t scale[64];                                 // its scales behind them (block 0)
    const uint32_t i0 = 64u * long_block(), planes = a.E / 64u, p0 = kGatherPlanes * blockIdx.y;
    if (i0 >= a.n) return;
    if (threadIdx.x < 64u) {
        const int64_t c = gather_from(a, i0 + threadIdx.x);
        const uint32_t cell = (uint32_t)c;
        const uint32_t in = WHICH == 0u ? kv4_code(0u, cell, 0u, 0u) : kv4_code(1u, cell, 0u, 0u);
        from[threadIdx.x] = c < 0 ? -1 : (int64_t)((cell >> 5) * (size_t)tb + in);
        scale[threadIdx.x] = kv4_scale(TYPE, cell, 0u) - in;
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < 192u * kGatherPlanes; e += 256u) {
        const bool codes = e < 128u * kGatherPlanes;
        const uint32_t plane = p0 + (codes ? e / 128u : (e - 128u * kGatherPlanes) / 64u), l = codes ? e & 127u : e & 63u;
        if (plane >= planes) continue;
        const uint8_t * src = a.src + kKv4Header + (size_t)plane * a.src_tiles * tb;
        uint8_t * dst = a.dst + kKv4Header + ((size_t)plane * a.dst_tiles + i0 / 32u) * tb;
        if (!codes) {                                              // a word of scales: cells c and c + 1, one block
            const uint32_t t = l >> 5, b = (l >> 2) & 1u, c = 16u * ((l >> 1) & 1u) + 4u * ((l >> 3) & 3u) + 2u * (l & 1u);
            if (i0 + 32u * t >= a.n) continue;
            const int64_t f0 = from[32u * t + c], f1 = from[32u * t + c + 1u];
            const uint32_t step = (TYPE == kKvQ4_1 ? 32u : 16u) * b;
            const uint8_t * s0 = src + f0 + (int32_t)scale[32u * t + c] + step, * s1 = src + f1 + (int32_t)scale[32u * t + c + 1u] + step;
            uint16_t * o = (uint16_t *)(dst + t * tb + kv4_scale(TYPE, c, b));
            if (f0 >= 0) {
                o[0] = *(const uint16_t *)s0;
                if constexpr (TYPE == kKvQ4_1) o[2] = *(const uint16_t *)(s0 + 4);
            }
            if (f1 >= 0) {
                o[1] = *(const uint16_t *)s1;
                if constexpr (TYPE == kKvQ4_1) o[3] = *(const uint16_t *)(s1 + 4);
            }
        } else if constexpr (WHICH == 0u) {                        // {block 0, block 1} of cells c and c + 1, quarter g of a block
            const uint32_t t = l >> 6, u = (l >> 5) & 1u, g = (l >> 3) & 3u, c = 2u * (l & 7u), i = 32u * t + 16u * u + c;
            if (i0 + 32u * t >= a.n) continue;
            const int64_t f0 = from[i], f1 = from[i + 1u];
            uint2 x = make_uint2(0u, 0u), y = make_uint2(0u, 0u);
            if (f0 >= 0) x = *(const uint2 *)(src + f0 + 128u * g);
            if (f1 >= 0) y = *(const uint2 *)(src + f1 + 128u * g);
            uint8_t * o = dst + t * tb + 512u * u + 8u * (16u * g + c);
            if (f0 >= 0 && f1 >= 0) *(uint4 *)o = make_uint4(x.x, x.y, y.x, y.y);
            else if (f0 >= 0) *(uint2 *)o = x;
            else if (f1 >= 0) *(uint2 *)(o + 8) = y;
        } else {                                                   // [block][group of 16 cells], a byte a cell: byte j of the block
            const uint32_t t = l >> 6, g = (l >> 4) & 3u, j = l & 15u;
            if (i0 + 32u * t >= a.n) continue;
            int64_t f[8];
#pragma unroll
            for (uint32_t k = 0; k < 8u; ++k) f[k] = from[32u * t + 16u * (k >> 2) + 4u * g + (k & 3u)];
            uint32_t v[2][8];
#pragma unroll
            for (uint32_t k = 0; k < 8u; ++k)
#pragma unroll
                for (uint32_t b = 0; b < 2u; ++b) v[b][k] = f[k] >= 0 ? src[f[k] + 16u * j + 8u * b] : 0u;
            int64_t none = 0;
#pragma unroll
            for (uint32_t k = 0; k < 8u; ++k) none |= f[k];
            uint8_t * o = dst + t * tb + 16u * (16u * g + j);
            if (none >= 0) {                                       // (cells lie in the order 0, 2, 1, 3)
                auto word = [&](uint32_t b, uint32_t u) { return v[b][4 * u] | v[b][4 * u + 2] << 8 | v[b][4 * u + 1] << 16 | v[b][4 * u + 3] << 24; };
                *(uint4 *)o = make_uint4(word(0, 0), word(0, 1), word(1, 0), word(1, 1));
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 8u; ++k)
                    if (f[k] >= 0)
#pragma unroll
                        for (uint32_t b = 0; b < 2u; ++b) o[8u * b + 4u * (k >> 2) + ((k & 1u) << 1 | ((k >> 1) & 1u))] = (uint8_t)v[b][k];
            }
        }
    }
}

// q8_0 (the layout of k_kv.hip): workgroup (16 cells, 256 values), a thread 16 bytes; half of them also the scales.
template <uint32_t WHICH>
__global__ __launch_bounds__(256) void k_kv_gather(KvGatherArgs a) {
    __shared__ int64_t from[16];
    const uint32_t u = long_block(), v0 = 256u * blockIdx.y, nbk = a.E / 32u, l = threadIdx.x;
    if (16ull * u >= a.n) return;
    if (l < 16u) from[l] = gather_from(a, 16u * u + l);
    __syncthreads();
    auto quants = [&](int64_t c) { return a.src + a.src_off + (size_t)(c >> 4) * 16u * a.E; };
    uint8_t * out = a.dst + a.dst_off + (size_t)u * 16u * a.E;
    if constexpr (WHICH == 0u) {                                   // 16 values of a cell
        const uint32_t i = v0 / 16u + l / 16u, k = l & 15u;
        const int64_t c = from[k];
        if (16u * i < a.E && c >= 0) *(uint4 *)(out + (i * 16u + k) * 16u) = *(const uint4 *)(quants(c) + (i * 16u + ((uint32_t)c & 15u)) * 16u);
    } else if (v0 + l < a.E) {                                     // a value of 16 cells
        const uint32_t i = v0 + l;
        uint32_t v[16];
        int64_t none = 0;
#pragma unroll
        for (uint32_t k = 0; k < 16u; ++k) {
            const int64_t c = from[k];
            none |= c;
            v[k] = c >= 0 ? quants(c)[(size_t)i * 16u + ((uint32_t)c & 15u)] : 0u;
        }
        if (none >= 0) {
            auto word = [&](uint32_t k) { return v[k] | v[k + 1] << 8 | v[k + 2] << 16 | v[k + 3] << 24; };
            *(uint4 *)(out + (size_t)i * 16u) = make_uint4(word(0), word(4), word(8), word(12));
        } else {
#pragma unroll
            for (uint32_t k = 0; k < 16u; ++k)
                if (from[k] >= 0) out[(size_t)i * 16u + k] = (uint8_t)v[k];
        }
    }
    if (l < 128u) {                                                // the scales of 8 blocks
        const uint32_t b = v0 / 32u + l / 16u, k = l & 15u;
        const int64_t c = from[k];
        if (b < nbk && c >= 0)
            ((uint16_t *)a.dst)[((size_t)u * nbk + b) * 16u + k] = ((const uint16_t *)a.src)[((size_t)(c >> 4) * nbk + b) * 16u + ((uint32_t)c & 15u)];
    }
}

// rows of `bytes` (a multiple of 16), from_step and to_step apart
__global__ __launch_bounds__(256) void k_kv_rows_copy(uint8_t * to, size_t to_step, const uint8_t * from, size_t from_step, size_t bytes) {
    const size_t i = 16u * ((size_t)long_block() * 256u + threadIdx.x);
    if (i < bytes) *(uint4 *)(to + blockIdx.y * to_step + i) = *(const uint4 *)(from + blockIdx.y * from_step + i);
}

}  // namespace tsr

int tsr_launch_kv_gather(const tsr::KvGatherArgs & a, uint32_t type, uint32_t which, hipStream_t s) {
    using namespace tsr;
    if (type == kKvQ8_0) {
        const dim3 grid = long_grid(((uint64_t)a.n + 15u) / 16u, (a.E + 255u) / 256u);
        if (which == 0u) hipLaunchKernelGGL(k_kv_gather<0>, grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL(k_kv_gather<1>, grid, dim3(256), 0, s, a);
    } else {
        const dim3 grid = long_grid(((uint64_t)a.n + 63u) / 64u, (a.E / 64u + kGatherPlanes - 1u) / kGatherPlanes);
        if (type == kKvQ4_0 && which == 0u) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_kv4_gather<kKvQ4_0, 0>), grid, dim3(256), 0, s, a);
        else if (type == kKvQ4_0) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_kv4_gather<kKvQ4_0, 1>), grid, dim3(256), 0, s, a);
        else if (which == 0u) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_kv4_gather<kKvQ4_1, 0>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_kv4_gather<kKvQ4_1, 1>), grid, dim3(256), 0, s, a);
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

int tsr_launch_kv_rows_copy(uint8_t * to, size_t to_step, const uint8_t * from, size_t from_step, size_t bytes, uint32_t rows, hipStream_t s) {
    hipLaunchKernelGGL(tsr::k_kv_rows_copy, tsr::long_grid((bytes + 4095u) / 4096u, rows), dim3(256), 0, s, to, to_step, from, from_step, bytes);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
