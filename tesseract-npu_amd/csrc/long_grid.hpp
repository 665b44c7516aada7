// long_grid.hpp -- launches over more workgroups than one axis takes: of 2^32 threads along an axis and more a launch runs what is
// left of them by 2^32, without an error.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

namespace tsr {

constexpr uint32_t kAxisGroups = 1u << 23;                         // workgroups of up to 256 threads along the first axis

// n workgroups along the first axis and, beyond kAxisGroups, the third; the kernel's number of one, which may be past the last.
inline dim3 long_grid(uint64_t n, uint32_t y = 1u) {
    return dim3((uint32_t)std::min<uint64_t>(n, kAxisGroups), y, (uint32_t)((n + kAxisGroups - 1u) / kAxisGroups));
}
__device__ __forceinline__ uint32_t long_block() { return blockIdx.x + blockIdx.z * kAxisGroups; }

}  // namespace tsr
