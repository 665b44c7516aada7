// The workspace of an attention call in splits (csrc/attn4_plan.hpp): every float of it has one use, whole rows lie on 16
// bytes and the pairs behind them on 8, whatever the number of rows and splits.
#include "attn4_plan.hpp"

#include <cstdio>
#include <vector>

int main() {
    uint32_t n = 0;
    for (uint32_t D : { 64u, 128u, 256u, 512u })
        for (uint32_t T : { 1u, 2u, 3u, 5u })
            for (uint32_t G : { 1u, 3u, 7u, 8u })
                for (uint32_t hkv : { 1u, 3u })
                    for (uint32_t kv : { 672u, 1056u, 2000u, 9000u }) {
                        const tsr::Attn4Plan p = tsr::attn4_plan(T, D, hkv * G, hkv, kv, 256u);
                        if (p.S < 2u) continue;
                        const uint64_t nr = (uint64_t)T * hkv * G;
                        std::vector<uint8_t> used(p.ws_bytes / 4u, 0);
                        auto take = [&](size_t at, uint32_t len) {
                            if (at + len > used.size()) return false;
                            for (uint32_t i = 0; i < len; ++i)
                                if (used[at + i]++) return false;
                            return true;
                        };
                        for (uint32_t s = 0; s < p.S; ++s)
                            for (uint64_t r = 0; r < nr; ++r) {
                                const size_t row = tsr::attn4_part_row(nr, D, s, r), sum = tsr::attn4_part_sum(nr, D, p.S, s, r);
                                if (row % 4u != 0u || sum % 2u != 0u || !take(row, D) || !take(sum, 2u)) {
                                    printf("D %u T %u G %u heads %u cells %u: split %u row %u\n", D, T, G, hkv, kv, s, (unsigned)r);
                                    return 1;
                                }
                            }
                        for (uint8_t u : used)
                            if (!u) { printf("D %u T %u G %u heads %u cells %u: a float of no use\n", D, T, G, hkv, kv); return 1; }
                        n += p.S * nr % 2u;
                    }
    if (n == 0u) { printf("no odd number of rows\n"); return 1; }
    printf("%u workspaces of an odd number of rows\n", n);
    return 0;
}
