// sparse4_plan.hpp -- how the calls of sparse attention over a 4-bit cache are cut. Plain C++.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace tsr {

// Block selection: the tokens of a launch, so that their keys (one of 8 bytes a KV head and block) take at most 64 MiB (or are
// one token's) and its grid's second axis fits.
inline uint32_t kv4_select_tokens(uint32_t T, uint32_t n_head_kv, uint64_t n_blocks) {
    const uint64_t one = 8u * std::max<uint64_t>(1u, n_blocks) * n_head_kv;
    return (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>({ T, ((uint64_t)64 << 20) / one, 32768u }));
}
inline size_t kv4_select_ws(uint32_t T, uint32_t n_head_kv, uint64_t n_blocks) {
    return (size_t)kv4_select_tokens(T, n_head_kv, n_blocks) * n_head_kv * (size_t)std::max<uint64_t>(1u, n_blocks) * 8u;
}

}  // namespace tsr
