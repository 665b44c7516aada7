// The cuts of calls (csrc/attn4_plan.hpp) on 256 compute units: arguments n_head n_head_kv D T n_kv, five a call; a line of
// C NT S for each.
#include "attn4_plan.hpp"

#include <cstdio>
#include <cstdlib>

int main(int argc, char ** argv) {
    for (int i = 1; i + 4 < argc; i += 5) {
        uint32_t v[5];
        for (int j = 0; j < 5; ++j) v[j] = (uint32_t)strtoul(argv[i + j], nullptr, 10);
        const tsr::Attn4Plan p = tsr::attn4_plan(v[3], v[2], v[0], v[1], v[4], 256u);
        printf("%u %u %u\n", p.C, p.NT, p.S);
    }
    return 0;
}
