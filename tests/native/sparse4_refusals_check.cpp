// The argument checks of the sparse attention over 4-bit KV caches (csrc/tsr_sparse4.hip) and its cuts (csrc/sparse4_plan.hpp),
// without a device: calls that are refused launch nothing, and what is launched are whole parts of the call.
#include <hip/hip_runtime.h>

hipError_t hipSetDevice(int);
#include "tsr_sparse4.hip"

#include <cstdio>
#include <vector>

static bool capturing;
static std::vector<tsr::Kv4BoundsArgs> bounds;
static std::vector<tsr::Kv4SelectArgs> selects;
static std::vector<tsr::Attn4BlocksArgs> attns;
static size_t reserved;
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus * s) {
    *s = capturing ? (hipStreamCaptureStatus)1 : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipMalloc(void ** p, size_t n) { *p = (void *)(uintptr_t)0x10000; reserved = n; return hipSuccess; }
hipError_t hipFree(void *) { return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t *, unsigned) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
int tsr::hip_err(hipError_t e, const char *) { return e == hipSuccess ? 0 : TSR_HIP_E_HIP; }
int tsr_launch_kv4_bounds(const tsr::Kv4BoundsArgs & a, hipStream_t) { bounds.push_back(a); return 0; }
int tsr_launch_kv4_select(const tsr::Kv4SelectArgs & a, hipStream_t) { selects.push_back(a); return 0; }
int tsr_launch_attn4_blocks(const tsr::Attn4BlocksArgs & a, uint32_t, hipStream_t) { attns.push_back(a); return 0; }

static int n_bad, n_done;
static tsr_hip_ctx ctx;
struct Call {
    uint32_t T = 2, D = 64, nh = 4, nkv = 2, block = 32, n_kv = 90, n_sel = 2, nf = 1, nl = 1, nb = 4, n_new = 0;
    float scale = 0.125f;
    uint64_t qs = 256, os = 256;
    uintptr_t q = 0x1000, out = 0x2000, runs = 0, ids = 0x3000, bd = 0x4000, cells = 0, ws = 0;
    size_t ws_bytes = 0;
    tsr_hip_kv k, v;
    Call() { k.type = v.type = TSR_HIP_KV_Q4_0; k.E = v.E = 128; k.kv_size = v.kv_size = 100; }
};
// what the three entry points return
template <class F>
static void want(int rb, int rs, int ra, const char * what, F change) {
    Call c;
    change(c);
    bounds.clear(); selects.clear(); attns.clear();
    const int b = tsr_hip_kv4_bounds(&ctx, &c.k, c.D, c.block, c.n_kv, (uint32_t *)c.bd, (const uint32_t *)c.cells, c.n_new, nullptr);
    const int s = tsr_hip_kv4_select(&ctx, (const float *)c.q, c.T, c.qs, (const uint32_t *)c.bd, c.nb, c.D, c.nh, c.nkv, c.block, c.n_kv,
                                     (const uint32_t *)c.runs, c.n_sel, c.nf, c.nl, (int32_t *)c.ids, (void *)c.ws, c.ws_bytes, nullptr);
    const int a = tsr_hip_flash_attn_kv4_blocks(&ctx, (const float *)c.q, c.T, c.qs, &c.k, &c.v, c.D, c.nh, c.nkv, c.scale, c.n_kv,
                                                (const uint32_t *)c.runs, (const int32_t *)c.ids, c.n_sel, c.block, (float *)c.out, c.os,
                                                (void *)c.ws, c.ws_bytes, nullptr);
    ++n_done;
    if (b != rb || s != rs || a != ra || (b && !bounds.empty()) || (s && !selects.empty()) || (a && !attns.empty())) {
        printf("%s: %d %d %d, not %d %d %d\n", what, b, s, a, rb, rs, ra);
        ++n_bad;
    }
}

static int plans() {
    for (uint32_t D : { 64u, 128u, 256u, 512u })
        for (uint32_t hkv : { 1u, 3u, 8u, 512u })
            for (uint32_t G : { 1u, 3u, 4u, 5u, 8u, 9u, 64u }) {
                if ((uint64_t)hkv * G * D > 32768u) continue;
                for (uint32_t T : { 1u, 2u, 33u, 600u, 16000u, 65535u })
                    for (uint32_t n_sel : { 1u, 16u, 65536u })
                        for (uint32_t block : { 32u, 64u, 1024u }) {
                            const tsr::Attn4BlocksPlan p = tsr::attn4_blocks_plan(T, D, hkv * G, hkv, n_sel, block, 256u);
                            const uint64_t rows = 16u / p.C, n_rg = (G + rows - 1u) / rows, tiles = (uint64_t)n_sel * (block / 32u);
                            if (!(p.C == 1u || p.C == 2u || (p.C == 4u && D >= 128u)) || p.S == 0u || p.S > 256u || p.S > tiles ||
                                n_rg * std::min(T, kBlockTokens) > 65535u || (p.S > 1u && T > kBlockTokens) ||
                                p.ws_bytes != (p.S > 1u ? 4u * (size_t)p.S * T * hkv * G * (2u + D) : 0u)) {
                                printf("plan: T %u D %u heads %u G %u n_sel %u block %u\n", T, D, hkv, G, n_sel, block);
                                return 1;
                            }
                        }
                for (uint32_t T : { 1u, 100u, 65535u })
                    for (uint64_t nb : { 0ull, 1ull, 4096ull, 1ull << 26 }) {
                        const uint32_t t = tsr::kv4_select_tokens(T, hkv, nb);
                        if (t == 0u || t > T || t > 32768u || tsr::kv4_select_ws(T, hkv, nb) < 8u * (uint64_t)t * hkv * nb ||
                            (t > 1u && 8u * (uint64_t)t * hkv * nb > (64ull << 20)))
                            return 1;
                    }
            }
    return 0;
}

int main() {
    ctx.n_cu = 256;
    const int arg = TSR_HIP_E_ARG, shape = TSR_HIP_E_SHAPE, fmt = TSR_HIP_E_FMT, range = TSR_HIP_E_RANGE;
    want(0, 0, 0, "the calls", [](Call &) {});
    if (bounds[0].n_blocks != 3 || bounds[0].stride != 4 || selects[0].n_blocks != 3) { printf("blocks\n"); ++n_bad; }
    want(0, 0, 0, "no cells", [](Call & c) { c.n_kv = 0; });
    if (!bounds.empty()) { printf("bounds of nothing\n"); ++n_bad; }
    want(0, arg, arg, "no queries", [](Call & c) { c.q = 0; });
    want(0, 0, arg, "no output", [](Call & c) { c.out = 0; });
    want(0, arg, arg, "no lists", [](Call & c) { c.ids = 0; });
    want(arg, arg, 0, "no bounds", [](Call & c) { c.bd = 0; });
    want(0, arg, arg, "no tokens", [](Call & c) { c.T = 0; });
    want(0, arg, arg, "too many tokens", [](Call & c) { c.T = 65536; });
    want(shape, shape, shape, "head size", [](Call & c) { c.D = 96; });
    want(0, shape, shape, "no heads", [](Call & c) { c.nh = 0; });
    want(0, shape, shape, "no KV heads", [](Call & c) { c.nkv = 0; });
    want(0, shape, shape, "heads that are not shared evenly", [](Call & c) { c.nh = 5; });
    want(0, shape, shape, "65 heads a KV head", [](Call & c) { c.nh = 65; c.nkv = 1; });
    want(shape, shape, shape, "no block", [](Call & c) { c.block = 0; });
    want(shape, shape, shape, "a block of 48", [](Call & c) { c.block = 48; });
    want(shape, shape, shape, "a block of 2048", [](Call & c) { c.block = 2048; });
    want(0, shape, shape, "no entries", [](Call & c) { c.n_sel = c.nf = c.nl = 0; });
    want(0, shape, shape, "too many entries", [](Call & c) { c.n_sel = 65537; });
    want(0, shape, 0, "more first and last blocks than entries", [](Call & c) { c.nf = 2; });
    want(0, shape, 0, "their sum past 2^32", [](Call & c) { c.nf = 1; c.nl = 0xFFFFFFFFu; });
    want(0, 0, shape, "scale 0", [](Call & c) { c.scale = 0.0f; });
    want(0, 0, shape, "scale NaN", [](Call & c) { c.scale = __builtin_nanf(""); });
    want(fmt, 0, fmt, "q8_0 caches", [](Call & c) { c.k.type = c.v.type = TSR_HIP_KV_Q8_0; });
    want(0, 0, fmt, "two types", [](Call & c) { c.v.type = TSR_HIP_KV_Q4_1; });
    want(shape, 0, shape, "another row length", [](Call & c) { c.k.E = 160; });
    want(0, 0, shape, "another cache length", [](Call & c) { c.v.kv_size = 101; });
    want(range, 0, range, "cells past the cache", [](Call & c) { c.n_kv = 101; });
    want(0, range, 0, "fewer bounds than blocks", [](Call & c) { c.nb = 2; });
    want(range, range, range, "2^31 cells", [](Call & c) { c.n_kv = 0x80000000u; });
    want(0, arg, arg, "unaligned queries", [](Call & c) { c.q += 8; });
    want(0, 0, arg, "unaligned output", [](Call & c) { c.out += 4; });
    want(0, arg, arg, "unaligned runs", [](Call & c) { c.runs = 0x5008; });
    want(arg, arg, 0, "unaligned bounds", [](Call & c) { c.bd += 8; });
    want(0, arg, arg, "unaligned lists", [](Call & c) { c.ids += 2; });
    want(arg, 0, 0, "unaligned cells", [](Call & c) { c.cells = 0x6002; c.n_new = 1; });
    want(arg, 0, 0, "new cells, none", [](Call & c) { c.cells = 0x6000; });
    want(0, 0, 0, "new cells", [](Call & c) { c.cells = 0x6000; c.n_new = 33; });
    if (bounds[0].n_blocks != 2) { printf("33 new cells: %u blocks\n", bounds[0].n_blocks); ++n_bad; }
    want(0, 0, 0, "new cells that may touch three blocks", [](Call & c) { c.cells = 0x6000; c.n_new = 34; });
    if (bounds[0].n_blocks != 3) { printf("34 new cells: %u blocks\n", bounds[0].n_blocks); ++n_bad; }
    want(0, 0, 0, "one new cell", [](Call & c) { c.cells = 0x6000; c.n_new = 1; });
    if (bounds[0].n_blocks != 1) { printf("a new cell: %u blocks\n", bounds[0].n_blocks); ++n_bad; }
    want(0, arg, arg, "query rows that overlap", [](Call & c) { c.qs = 252; });
    want(0, arg, arg, "a query stride of 258", [](Call & c) { c.qs = 258; });
    want(0, 0, arg, "output rows that overlap", [](Call & c) { c.os = 128; });
    want(0, 0, 0, "one row needs no strides", [](Call & c) { c.T = 1; c.qs = c.os = 0; });
    // workspaces
    const size_t ws = tsr_hip_kv4_select_ws(&ctx, 2, 2, 32, 90);
    if (ws != 2 * 2 * 3 * 8) { printf("workspace %zu\n", ws); ++n_bad; }
    auto big = [](Call & c) { c.T = 1; c.n_sel = 64; };
    const size_t wa = tsr_hip_flash_attn_kv4_blocks_ws(&ctx, 1, 64, 4, 2, 64, 32);
    if (wa == 0) { printf("no splits\n"); ++n_bad; }
    want(0, arg, 0, "a small workspace", [&](Call & c) { c.ws = 0x8000; c.ws_bytes = ws - 1; });
    want(0, 0, arg, "a small workspace for splits", [&](Call & c) { big(c); c.ws = 0x8000; c.ws_bytes = wa - 1; });
    want(0, arg, arg, "an unaligned workspace", [&](Call & c) { big(c); c.ws = 0x8004; c.ws_bytes = wa; });
    want(0, 0, 0, "a workspace", [&](Call & c) { big(c); c.ws = 0x8000; c.ws_bytes = wa; });
    if ((uintptr_t)attns[0].a.part != 0x8000 || (uintptr_t)selects[0].keys != 0x8000) { printf("not the caller's workspace\n"); ++n_bad; }
    capturing = true;
    want(0, arg, arg, "captured without a workspace", big);
    want(0, arg, 0, "captured, an attention that needs none", [](Call &) {});
    want(0, 0, 0, "captured with one", [&](Call & c) { big(c); c.ws = 0x8000; c.ws_bytes = wa; });
    capturing = false;
    want(0, 0, 0, "the context's scratch", big);
    if (reserved < wa || (uintptr_t)attns[0].a.part != 0x10000) { printf("scratch of %zu\n", reserved); ++n_bad; }
    // parts
    want(0, 0, 0, "65535 tokens", [](Call & c) { c.T = 65535; c.runs = 0x100000; });
    uint64_t t = 0;
    for (const auto & b : attns) {
        if ((uintptr_t)b.a.q != 0x1000 + t * 1024 || (uintptr_t)b.a.out != 0x2000 + t * 1024 || (uintptr_t)b.a.runs != 0x100000 + 16 * t ||
            (uintptr_t)b.blocks != 0x3000 + 16 * t || b.a.T == 0u || b.a.T > kBlockTokens) { printf("part at %llu\n", (unsigned long long)t); ++n_bad; }
        t += b.a.T;
    }
    if (t != 65535) ++n_bad;
    t = 0;
    for (const auto & b : selects) {
        if ((uintptr_t)b.q != 0x1000 + t * 1024 || (uintptr_t)b.runs != 0x100000 + 16 * t || (uintptr_t)b.blocks != 0x3000 + 16 * t) ++n_bad;
        t += b.T;
    }
    if (t != 65535) ++n_bad;
    if (tsr_hip_kv4_select_ws(nullptr, 1, 2, 32, 90) || tsr_hip_kv4_select_ws(&ctx, 1, 2, 48, 90) || tsr_hip_kv4_select_ws(&ctx, 0, 2, 32, 90) ||
        tsr_hip_flash_attn_kv4_blocks_ws(&ctx, 1, 64, 4, 2, 0, 32)) { printf("ws\n"); ++n_bad; }
    if (tsr_hip_kv4_bounds(nullptr, nullptr, 64, 32, 1, nullptr, nullptr, 0, nullptr) != arg) ++n_bad;
    n_bad += plans();
    printf("%d calls\n", n_done);
    return n_bad != 0;
}
