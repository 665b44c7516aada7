// k_kv_pick.hip -- the cells of a cache that are kept: the first, the last and, of those between, the ones with the largest
// weights (pick.hpp), in the order of their cells.
//
// One workgroup of 16 waves finds the cut and writes the list; up to 65536 weights stay in its registers. Bound: what one compute unit
// loads and counts: 16384 of 65536 cells take 31 us (its 64 weights a lane some 2000 instructions), 777 of 1500 5 us; a quarter of
// 8192, 16384 and 32768 8, 11 and 19, of 131072, which are read again at every pass, 128.
#include "kernels.hpp"
#include "pick.hpp"

namespace tsr {

// ROWS rows of 64 weights a wave in registers; 0: read whenever they are needed.
template <uint32_t ROWS>
__global__ __launch_bounds__(1024) void k_kv_pick(const float * weights, uint32_t n, uint32_t keep, uint32_t first, uint32_t last, int64_t * idx,
                                                  float * kept) {
    __shared__ __align__(16) PickRoom<16> room;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), lane = threadIdx.x & 63u;
    const uint32_t rows = (n + 1023u) / 1024u, c0 = wave * rows * 64u + lane;
    auto counts = [&](uint32_t c) { return c >= first && c < n - last; };
    uint32_t mine[ROWS == 0u ? 1u : ROWS];
    if constexpr (ROWS != 0u) {
        float x[ROWS];
#pragma unroll
        for (uint32_t j = 0; j < ROWS; ++j) x[j] = j < rows && c0 + 64u * j < n ? weights[c0 + 64u * j] : 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < ROWS; ++j) mine[j] = j < rows && counts(c0 + 64u * j) ? order_of(x[j]) : 0u;
    }
    auto store = [&](uint32_t at, uint32_t c, float w) {
        idx[at] = c;
        if (kept != nullptr) kept[at] = w;
    };
    for (uint32_t i = threadIdx.x; i < first + last; i += 1024u) {
        if (i < first) store(i, i, weights[i]);
        else store(keep - last + (i - first), n - last + (i - first), weights[n - last + (i - first)]);
    }
    if (keep == first + last) return;
    auto each = [&](auto f) {
        if constexpr (ROWS != 0u) {
#pragma unroll
            for (uint32_t j0 = 0; j0 < ROWS; j0 += 4u)
                if (j0 < rows)
#pragma unroll
                    for (uint32_t j = j0; j < j0 + 4u; ++j) f(c0 + 64u * j, mine[j]);
        } else {
            for (uint32_t j = 0; j < rows; ++j) {
                const uint32_t c = c0 + 64u * j;
                f(c, counts(c) ? order_of(weights[c]) : 0u);
            }
        }
    };
    Pick<16>{ room, wave, lane }.run<uint32_t>(keep - first - last, each, [&](uint32_t at, uint32_t c, uint32_t k) { store(first + at, c, of_order(k)); });
}

}  // namespace tsr

int tsr_launch_kv_pick(const float * weights, uint32_t n, uint32_t keep, uint32_t first, uint32_t last, int64_t * idx, float * kept,
                       hipStream_t s) {
    const dim3 grid(1), wg(1024);
    if (n <= 4096u) hipLaunchKernelGGL(tsr::k_kv_pick<4>, grid, wg, 0, s, weights, n, keep, first, last, idx, kept);
    else if (n <= 16384u) hipLaunchKernelGGL(tsr::k_kv_pick<16>, grid, wg, 0, s, weights, n, keep, first, last, idx, kept);
    else if (n <= 65536u) hipLaunchKernelGGL(tsr::k_kv_pick<64>, grid, wg, 0, s, weights, n, keep, first, last, idx, kept);
    else hipLaunchKernelGGL(tsr::k_kv_pick<0>, grid, wg, 0, s, weights, n, keep, first, last, idx, kept);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
