// k_kv4.hip -- KV caches of 4-bit blocks on the device: SET_ROWS (quantizing f32 rows as they are written), cells read
// back as f32 rows, and the byte conversion to / from llama.cpp's q4_0 / q4_1 images. kv4.hpp has the layout.
#include "kernels.hpp"
#include "kv4.hpp"
#include "tsr_dev.hpp"

namespace tsr {

constexpr uint32_t kRowsPerWg = 32u;      // rows a workgroup: eight threads a row of 64 values (a pair of blocks)

__device__ __forceinline__ float quad_max(float v) {              // over the four threads of a block
    v = fmaxf(v, dpp_f<kDppXor1>(v));
    return fmaxf(v, dpp_f<kDppXor2>(v));
}
__device__ __forceinline__ float quad_min(float v) {
    v = fminf(v, dpp_f<kDppXor1>(v));
    return fminf(v, dpp_f<kDppXor2>(v));
}
__device__ __forceinline__ uint32_t quad_min_u(uint32_t v) {
    v = min(v, (uint32_t)dpp_i<kDppXor1>((int)v));
    return min(v, (uint32_t)dpp_i<kDppXor2>((int)v));
}
__device__ __forceinline__ uint16_t f16_bits(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }

// ggml's block rule on the 32 values of four threads, thread k of a block holding values 4 k .. 4 k + 3 (x[0 .. 3]) and
// 16 + 4 k .. (x[4 .. 7]); every step is one f32 operation, so that the codes are those of the CPU's image. Returns the
// thread's code word (byte i: value 4 k + i low, value 16 + 4 k + i high). A NaN is stored as 0; an infinity, or a
// block beyond f16's range, makes the block's scale infinite.
template <uint32_t TYPE>
__device__ __forceinline__ uint32_t quantize4(float (&x)[8], uint32_t k, uint16_t & d16, uint16_t & m16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] != x[i] ? 0.0f : x[i];
    float d, sub, half;
    if constexpr (TYPE == kKvQ4_0) {
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(x[i]));
        a = quad_max(a);
        uint32_t first = 64u;                                      // the first value of that magnitude: 2 place + sign
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t at = (i < 4 ? 4u * k + i : 12u + 4u * k + i) * 2u + (fb(x[i]) >> 31);
            first = fabsf(x[i]) == a ? min(first, at) : first;
        }
        first = quad_min_u(first);
        d = ((first & 1u) ? -a : a) / -8.0f;
        m16 = 0;
        sub = 0.0f;
        half = 8.5f;
    } else {
        float lo = x[0], hi = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); }
        lo = quad_min(lo);
        hi = quad_max(hi);
        d = (hi - lo) / 15.0f;
        m16 = f16_bits(lo);
        sub = lo;
        half = 0.5f;
    }
    d16 = f16_bits(d);
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    uint32_t w = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = (TYPE == kKvQ4_0 ? x[i] : x[i] - sub) * id;
        const uint32_t n = (uint32_t)min(max(cvt_i32_sat(y + half), 0), 15);
        w |= n << (8 * (i & 3) + (i >> 2) * 4);
    }
    return w;
}

// SET_ROWS: workgroup (pair of blocks, 32 rows). Bound: the rows' bytes, 32768 rows of 1024 values in 23 us (6.6 TB/s); a
// launch for few rows.
template <uint32_t TYPE>
__global__ __launch_bounds__(256) void k_kv4_set_rows(Kv4Args a, uint32_t which, const float * src, uint64_t src_stride,
                                                      uint32_t n_rows, const int64_t * idx, int32_t * bad) {
    const uint32_t r = blockIdx.y * kRowsPerWg + threadIdx.x / 8u, q = threadIdx.x & 7u, k = q & 3u;
    const uint32_t b = 2u * blockIdx.x + (q >> 2);
    if (r < n_rows) {
        const int64_t cell64 = idx[r];
        const float * row = src + (size_t)r * src_stride + 32u * b + 4u * k;
        const float4 lo = *(const float4 *)row, hi = *(const float4 *)(row + 16);
        float x[8] = { lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w };
        uint16_t d16, m16;
        const uint32_t w = quantize4<TYPE>(x, k, d16, m16);
        if (cell64 < 0 || cell64 >= (int64_t)a.kv_size) {
            if (bad != nullptr && q == 0u && blockIdx.x == 0u) *bad = 1;
        } else {
            const uint32_t cell = (uint32_t)cell64;
            uint8_t * t = a.base + kv4_tile(TYPE, a.n_tiles, cell, b);
            if (which == 0u) {
                *(uint32_t *)(t + kv4_code(0u, cell, b, 4u * k)) = w;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) t[kv4_code(1u, cell, b, 4u * k + i)] = (uint8_t)(w >> (8u * i));
            }
            if (k == 0u) {
                uint16_t * sc = (uint16_t *)(t + kv4_scale(TYPE, cell, b));
                sc[0] = d16;
                if constexpr (TYPE == kKvQ4_1) sc[2] = m16;
            }
        }
    }
}

// Stores past the caches: rows read back are not read again by these kernels.
typedef float f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void store_row(float * p, float a, float b, float c, float d) {
    __builtin_nontemporal_store(f32x4{ a, b, c, d }, (f32x4 *)p);
}

// Cells as f32 rows: workgroup (pair of blocks, 32 rows), a thread values 4 q .. 4 q + 3 of both blocks. Bound: the
// rows' bytes. Every store covers whole lines of the rows and goes past the caches: 32768 rows of 1024 values (153 MB)
// take 24 us from K and 28 from V, 6.3 and 5.4 TB/s. With half a line a store and no hint they took 41 and 50, with the
// hint alone 38 and 46. d n - 8 d and d n are exact in f32; q4_1's sum is rounded once.
template <uint32_t TYPE>
__global__ __launch_bounds__(256) void k_kv4_get_rows(Kv4Args a, uint32_t which, const int64_t * idx, uint32_t n_rows,
                                                      float * dst, uint64_t dst_stride, int32_t * bad) {
    const uint32_t r = blockIdx.y * kRowsPerWg + threadIdx.x / 8u, q = threadIdx.x & 7u, k = q & 3u;
    const uint32_t b = 2u * blockIdx.x;
    if (r >= n_rows) return;
    const int64_t cell64 = idx[r];
    if (cell64 < 0 || cell64 >= (int64_t)a.kv_size) {
        if (bad != nullptr && q == 0u && blockIdx.x == 0u) *bad = 1;
        return;
    }
    const uint32_t cell = (uint32_t)cell64;
    const uint8_t * t = a.base + kv4_tile(TYPE, a.n_tiles, cell, b);
    uint32_t w[2] = { 0u, 0u };
    if (which == 0u) {
        const uint2 v = *(const uint2 *)(t + kv4_code(0u, cell, b, 4u * k));
        w[0] = v.x;
        w[1] = v.y;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            w[0] |= (uint32_t)t[kv4_code(1u, cell, b, 4u * k + i)] << (8u * i);
            w[1] |= (uint32_t)t[kv4_code(1u, cell, b + 1u, 4u * k + i)] << (8u * i);
        }
    }
    float * row = dst + (size_t)r * dst_stride + 32u * b + 4u * q;
#pragma unroll
    for (uint32_t p = 0; p < 2; ++p) {
        const uint16_t * sc = (const uint16_t *)(t + kv4_scale(TYPE, cell, b + p));
        const float d = h2f_fast(sc[0]);
        const float m = TYPE == kKvQ4_1 ? h2f_fast(sc[TYPE == kKvQ4_1 ? 2 : 0]) : 0.0f;
        const uint32_t v = w[p] >> (q & 4u);                       // threads 4 .. 7: the high nibbles
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float n = (float)((v >> (8 * i)) & 15u);
            y[i] = TYPE == kKvQ4_0 ? d * (n - 8.0f) : d * n + m;
        }
        store_row(row + 32u * p, y[0], y[1], y[2], y[3]);
    }
}

// q8_0 cells as f32 rows (the layout of k_kv.hip): a wave 256 values of a row. d q is exact in f32.
__global__ __launch_bounds__(64) void k_kv_get_rows(KvArgs a, uint32_t which, const int64_t * idx, float * dst,
                                                    uint64_t dst_stride, int32_t * bad) {
    const uint32_t r = blockIdx.y, i = 4u * (blockIdx.x * 64u + threadIdx.x);
    const int64_t cell64 = idx[r];
    if (cell64 < 0 || cell64 >= (int64_t)a.kv_size) {
        if (bad != nullptr && i == 0u) *bad = 1;
        return;
    }
    if (i >= a.E) return;
    const uint32_t u = (uint32_t)(cell64 >> 4), rr = (uint32_t)cell64 & 15u, nbk = a.E / 32u;
    const uint8_t * qb = a.base + a.quant_off + (size_t)u * 16u * a.E;
    const float d = h2f_fast(((const uint16_t *)a.base)[((size_t)u * nbk + i / 32u) * 16u + rr]);
    int8_t v[4];
    if (which == 0u) {
        *(uint32_t *)v = *(const uint32_t *)(qb + ((size_t)(i >> 4) * 16u + rr) * 16u + (i & 15u));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (int8_t)qb[(size_t)(i + j) * 16u + rr];
    }
    store_row(dst + (size_t)r * dst_stride + i, d * v[0], d * v[1], d * v[2], d * v[3]);
}

// One thread a byte [off, off + n) of the ggml image (row j = cell j, E / 32 blocks of {d[, m], 16 code bytes}).
__global__ __launch_bounds__(256) void k_kv4_bytes(Kv4Args a, uint32_t which, uint64_t off, uint64_t n, uint8_t * stage,
                                                   int to_dev) {
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (i >= n) return;
    const uint32_t bb = kv4_block_bytes(a.type), head = bb - 16u;
    const uint64_t rowb = (uint64_t)(a.E / 32u) * bb, pos = off + i;
    const uint32_t cell = (uint32_t)(pos / rowb), in = (uint32_t)(pos % rowb), b = in / bb, j = in % bb;
    const uint32_t at = j < head ? kv4_scale(a.type, cell, b) + (j & 1u) + 4u * (j >> 1) : kv4_code(which, cell, b, j - head);
    uint8_t * p = a.base + kv4_tile(a.type, a.n_tiles, cell, b) + at;
    if (to_dev) *p = stage[i];
    else stage[i] = *p;
}

}  // namespace tsr

static int launched() { return hipGetLastError() == hipSuccess ? 0 : -4; }

int tsr_launch_kv4_set_rows(const tsr::Kv4Args & a, uint32_t which, const float * src, uint32_t n_rows,
                            uint64_t src_stride, const int64_t * idx, int32_t * bad, hipStream_t s) {
    const dim3 grid(a.E / 64u, (n_rows + tsr::kRowsPerWg - 1u) / tsr::kRowsPerWg);
    const dim3 wg(n_rows >= 32u ? 256u : (8u * n_rows + 63u) & ~63u);
    if (a.type == tsr::kKvQ4_0)
        hipLaunchKernelGGL(tsr::k_kv4_set_rows<tsr::kKvQ4_0>, grid, wg, 0, s, a, which, src, src_stride, n_rows, idx, bad);
    else
        hipLaunchKernelGGL(tsr::k_kv4_set_rows<tsr::kKvQ4_1>, grid, wg, 0, s, a, which, src, src_stride, n_rows, idx, bad);
    return launched();
}

int tsr_launch_kv4_get_rows(const tsr::Kv4Args & a, uint32_t which, const int64_t * idx, uint32_t n_rows, float * dst,
                            uint64_t dst_stride, int32_t * bad, hipStream_t s) {
    const dim3 grid(a.E / 64u, (n_rows + tsr::kRowsPerWg - 1u) / tsr::kRowsPerWg);
    const dim3 wg(n_rows >= 32u ? 256u : (8u * n_rows + 63u) & ~63u);
    if (a.type == tsr::kKvQ4_0)
        hipLaunchKernelGGL(tsr::k_kv4_get_rows<tsr::kKvQ4_0>, grid, wg, 0, s, a, which, idx, n_rows, dst, dst_stride, bad);
    else
        hipLaunchKernelGGL(tsr::k_kv4_get_rows<tsr::kKvQ4_1>, grid, wg, 0, s, a, which, idx, n_rows, dst, dst_stride, bad);
    return launched();
}

int tsr_launch_kv_get_rows(const tsr::KvArgs & a, uint32_t which, const int64_t * idx, uint32_t n_rows, float * dst,
                           uint64_t dst_stride, int32_t * bad, hipStream_t s) {
    hipLaunchKernelGGL(tsr::k_kv_get_rows, dim3((a.E / 4u + 63u) / 64u, n_rows), dim3(64), 0, s, a, which, idx, dst,
                       dst_stride, bad);
    return launched();
}

int tsr_launch_kv4_bytes(const tsr::Kv4Args & a, uint32_t which, uint64_t off, uint64_t n, uint8_t * stage, int to_dev,
                         hipStream_t s) {
    if (n == 0u) return 0;
    hipLaunchKernelGGL(tsr::k_kv4_bytes, dim3((uint32_t)((n + 255u) / 256u)), dim3(256), 0, s, a, which, off, n, stage, to_dev);
    return launched();
}
