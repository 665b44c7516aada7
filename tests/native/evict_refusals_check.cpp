// The argument checks of eviction by attention weight (csrc/tsr_evict4.hip) and its cuts (csrc/weights4_plan.hpp), without a
// device.
#include <hip/hip_runtime.h>

hipError_t hipSetDevice(int);
#include "tsr_evict4.hip"

#include <cstdio>
#include <vector>

static bool capturing;
struct Weights { tsr::Attn4Args a; tsr::Weights4Plan p; const float * before; float decay; };
static std::vector<Weights> weights;
static std::vector<tsr::KvGatherArgs> gathers;
static int picks, copies;
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
int tsr_launch_attn4_weights(const tsr::Attn4Args & a, const tsr::Weights4Plan & p, const float * before, float decay, hipStream_t) {
    weights.push_back({ a, p, before, decay });
    return 0;
}
int tsr_launch_kv_pick(const float *, uint32_t, uint32_t, uint32_t, uint32_t, int64_t *, float *, hipStream_t) { ++picks; return 0; }
int tsr_launch_kv_gather(const tsr::KvGatherArgs & a, uint32_t, uint32_t, hipStream_t) { gathers.push_back(a); return 0; }
int tsr_launch_kv_rows_copy(uint8_t *, size_t, const uint8_t *, size_t, size_t, uint32_t, hipStream_t) { ++copies; return 0; }

static int n_bad, n_done;
static tsr_hip_ctx ctx;
struct Call {
    uint32_t T = 2, D = 64, nh = 4, nkv = 2, n_kv = 90;
    float scale = 0.125f, decay = 0.5f;
    uint64_t qs = 256;
    uintptr_t q = 0x1000, out = 0x2000, before = 0x3000, runs = 0, ws = 0;
    size_t ws_bytes = 0;
    tsr_hip_kv k;
    Call() { k.type = TSR_HIP_KV_Q4_0; k.E = 128; k.kv_size = 100; }
};
template <class F>
static void want(int rc, const char * what, F change) {
    Call c;
    change(c);
    weights.clear();
    const int got = tsr_hip_attn_weights_kv4(&ctx, (const float *)c.q, c.T, c.qs, &c.k, c.D, c.nh, c.nkv, c.scale, c.n_kv, (const uint32_t *)c.runs,
                                             (const float *)c.before, c.decay, (float *)c.out, (void *)c.ws, c.ws_bytes, nullptr);
    ++n_done;
    if (got != rc || (rc && !weights.empty())) { printf("%s: %d, not %d\n", what, got, rc); ++n_bad; }
}
struct Pick {
    uintptr_t w = 0x1000, idx = 0x2000, kept = 0x3000;
    uint32_t n = 10, keep = 5, first = 1, last = 2;
};
template <class F>
static void want_pick(int rc, const char * what, F change) {
    Pick c;
    change(c);
    picks = 0;
    const int got = tsr_hip_kv_pick(&ctx, (const float *)c.w, c.n, c.keep, c.first, c.last, (int64_t *)c.idx, (float *)c.kept, nullptr);
    ++n_done;
    if (got != rc || picks != (rc == 0 && c.keep != 0)) { printf("pick, %s: %d, not %d\n", what, got, rc); ++n_bad; }
}
struct Gather {
    tsr_hip_kv d, s;
    bool self = false;
    uint32_t which = 1, n = 40;
    uintptr_t idx = 0x1000, bad = 0x2000, ws = 0;
    size_t ws_bytes = 0;
    Gather() { d.type = s.type = TSR_HIP_KV_Q4_1; d.E = s.E = 128; d.kv_size = 50; s.kv_size = 1000; d.dev = (uint8_t *)0x100000; s.dev = (uint8_t *)0x200000; }
};
template <class F>
static void want_gather(int rc, const char * what, F change) {
    Gather c;
    change(c);
    gathers.clear();
    copies = 0;
    const int got = tsr_hip_kv_gather(&ctx, &c.d, c.self ? &c.d : &c.s, c.which, (const int64_t *)c.idx, c.n, (int32_t *)c.bad, (void *)c.ws, c.ws_bytes, nullptr);
    ++n_done;
    const int parts = c.d.type == TSR_HIP_KV_Q8_0 ? 2 : 1;
    if (got != rc || gathers.size() != (rc == 0 && c.n != 0) || copies != (rc == 0 && c.n != 0 && c.self ? parts : 0)) { printf("gather, %s: %d, not %d\n", what, got, rc); ++n_bad; }
}

// Pairs and sums lie apart inside the workspace; the launches' grids fit.
static int plans() {
    for (uint32_t D : { 64u, 128u, 256u, 512u })
        for (uint32_t hkv : { 1u, 3u, 8u })
            for (uint32_t G : { 1u, 4u, 7u, 64u }) {
                if ((uint64_t)hkv * G * D > 32768u) continue;
                for (uint32_t T : { 1u, 2u, 9u, 64u, 2000u, 65535u })
                    for (uint32_t kv : { 1u, 31u, 8192u, 131071u, 0x7FFFFFFFu }) {
                        const tsr::Weights4Plan p = tsr::weights4_plan(T, D, hkv * G, hkv, kv, 256u);
                        const uint64_t tiles = ((uint64_t)kv + 31u) / 32u, n = (uint64_t)hkv * p.n_rg;
                        const size_t last = tsr::weights4_pair(p, hkv, p.S - 1u, hkv - 1u, p.n_rg - 1u, 16u * p.NT - 1u);
                        if (!(p.NT == 1u || (p.NT == 2u && D <= 256u) || (p.NT == 4u && D <= 128u)) || p.S == 0u || p.S > tsr::kWeightsSplits || p.S > tiles ||
                            p.tokens == 0u || p.tokens > T || (uint64_t)p.n_rg * 16u * p.NT < (uint64_t)p.tokens * G || p.n_rg > 65535u ||
                            p.one > tiles || (p.one != 0u && (hkv * D > 1024u || p.n_rg != 1u || p.NT != 1u || p.tokens != T)) || p.n_pad != 32u * tiles || 8u * (last + 1u) != p.sums || p.ws_bytes != p.sums + 4u * n * p.n_pad || p.sums % 16u != 0u) {
                            printf("plan: T %u D %u heads %u G %u cells %u\n", T, D, hkv, G, kv);
                            return 1;
                        }
                    }
            }
    return 0;
}

int main() {
    ctx.n_cu = 256;
    const int arg = TSR_HIP_E_ARG, shape = TSR_HIP_E_SHAPE, fmt = TSR_HIP_E_FMT, range = TSR_HIP_E_RANGE;
    want(0, "the call", [](Call &) {});
    if (weights[0].before != (const float *)0x3000 || weights[0].decay != 0.5f) { printf("addend\n"); ++n_bad; }
    want(0, "no cells", [](Call & c) { c.n_kv = 0; });
    if (!weights.empty()) { printf("weights of nothing\n"); ++n_bad; }
    want(0, "no addend", [](Call & c) { c.before = 0; });
    want(0, "decay 0", [](Call & c) { c.decay = 0.0f; });
    if (weights[0].before != nullptr) { printf("decay 0 reads the addend\n"); ++n_bad; }
    want(0, "in place", [](Call & c) { c.before = c.out; });
    want(arg, "no queries", [](Call & c) { c.q = 0; });
    want(arg, "no output", [](Call & c) { c.out = 0; });
    want(arg, "no tokens", [](Call & c) { c.T = 0; });
    want(arg, "too many tokens", [](Call & c) { c.T = 65536; });
    want(shape, "head size", [](Call & c) { c.D = 96; });
    want(shape, "no heads", [](Call & c) { c.nh = 0; });
    want(shape, "no KV heads", [](Call & c) { c.nkv = 0; });
    want(shape, "heads that are not shared evenly", [](Call & c) { c.nh = 5; });
    want(shape, "scale 0", [](Call & c) { c.scale = 0.0f; });
    want(shape, "scale inf", [](Call & c) { c.scale = __builtin_inff(); });
    want(shape, "decay NaN", [](Call & c) { c.decay = __builtin_nanf(""); });
    want(fmt, "a q8_0 cache", [](Call & c) { c.k.type = TSR_HIP_KV_Q8_0; });
    want(shape, "another row length", [](Call & c) { c.k.E = 192; });
    want(range, "cells past the cache", [](Call & c) { c.n_kv = 101; });
    want(arg, "unaligned queries", [](Call & c) { c.q += 8; });
    want(arg, "unaligned runs", [](Call & c) { c.runs = 0x5008; });
    want(arg, "unaligned output", [](Call & c) { c.out += 2; });
    want(arg, "unaligned addend", [](Call & c) { c.before += 2; });
    want(arg, "query rows that overlap", [](Call & c) { c.qs = 252; });
    want(arg, "a query stride of 258", [](Call & c) { c.qs = 258; });
    want(0, "one row needs no stride", [](Call & c) { c.T = 1; c.qs = 0; });
    const size_t ws = tsr_hip_attn_weights_kv4_ws(&ctx, 2, 64, 4, 2, 90);
    want(arg, "a small workspace", [&](Call & c) { c.ws = 0x8000; c.ws_bytes = ws - 1; });
    want(arg, "an unaligned workspace", [&](Call & c) { c.ws = 0x8008; c.ws_bytes = ws; });
    want(0, "a workspace", [&](Call & c) { c.ws = 0x8000; c.ws_bytes = ws; });
    if ((uintptr_t)weights[0].a.part != 0x8000) { printf("not the caller's workspace\n"); ++n_bad; }
    capturing = true;
    want(arg, "captured without a workspace", [](Call &) {});
    want(0, "captured with one", [&](Call & c) { c.ws = 0x8000; c.ws_bytes = ws; });
    capturing = false;
    if (tsr_hip_attn_weights_kv4_ws(&ctx, 1, 96, 4, 2, 90) || tsr_hip_attn_weights_kv4_ws(nullptr, 1, 64, 4, 2, 90) || tsr_hip_attn_weights_kv4_ws(&ctx, 1, 64, 4, 2, 0)) ++n_bad;
    want(0, "long calls in parts", [](Call & c) { c.T = 65535; c.n_kv = c.k.kv_size = 100000; c.runs = 0x100000; });
    uint64_t t = 0;
    for (const Weights & w : weights) {
        if ((uintptr_t)w.a.q != 0x1000 + t * 1024 || (uintptr_t)w.a.runs != 0x100000 + 16 * t || w.a.T == 0u || w.a.T > w.p.tokens ||
            w.p.n_rg != (w.a.T * 2u + 16u * w.p.NT - 1u) / (16u * w.p.NT) || w.before != (const float *)(uintptr_t)(t ? 0x2000 : 0x3000) || w.decay != (t ? 1.0f : 0.5f)) {
            printf("part at %llu\n", (unsigned long long)t);
            ++n_bad;
        }
        t += w.a.T;
    }
    if (t != 65535 || weights.size() < 2) ++n_bad;

    want_pick(0, "the call", [](Pick &) {});
    want_pick(0, "none kept", [](Pick & c) { c.keep = c.first = c.last = 0; });
    want_pick(0, "all kept", [](Pick & c) { c.keep = 10; });
    want_pick(0, "no kept weights", [](Pick & c) { c.kept = 0; });
    want_pick(arg, "no weights", [](Pick & c) { c.w = 0; });
    want_pick(arg, "no list", [](Pick & c) { c.idx = 0; });
    want_pick(range, "more than there are", [](Pick & c) { c.keep = 11; });
    want_pick(range, "2^31 cells", [](Pick & c) { c.n = 0x80000000u; });
    want_pick(shape, "more first and last ones than kept", [](Pick & c) { c.first = 4; });
    want_pick(shape, "their sum past 2^32", [](Pick & c) { c.last = 0xFFFFFFFFu; });
    want_pick(arg, "an unaligned list", [](Pick & c) { c.idx = 0x2004; });
    want_pick(arg, "unaligned weights", [](Pick & c) { c.w = 0x1002; });
    want_pick(arg, "kept weights over the weights", [](Pick & c) { c.kept = c.w; });

    want_gather(0, "the call", [](Gather &) {});
    if (gathers[0].stay_size != 0 || gathers[0].dst != (uint8_t *)0x100000) { printf("gather\n"); ++n_bad; }
    want_gather(0, "nothing", [](Gather & c) { c.n = 0; });
    want_gather(0, "within a cache", [](Gather & c) { c.self = true; });
    if ((uintptr_t)gathers[0].dst != 0x10000 || gathers[0].stay_size != 64) { printf("gather within\n"); ++n_bad; }
    want_gather(0, "within a q8_0 cache", [](Gather & c) { c.self = true; c.d.type = TSR_HIP_KV_Q8_0; c.d.meta_row = 8; c.d.quant_off = 512; });
    if (gathers[0].stay_size != 64 || gathers[0].dst_off != 512 || gathers[0].src_off != 512) { printf("gather within q8_0\n"); ++n_bad; }
    want_gather(arg, "no list", [](Gather & c) { c.idx = 0; });
    want_gather(arg, "an unaligned list", [](Gather & c) { c.idx = 0x1004; });
    want_gather(arg, "no such plane", [](Gather & c) { c.which = 2; });
    want_gather(fmt, "two types", [](Gather & c) { c.s.type = TSR_HIP_KV_Q4_0; });
    want_gather(shape, "two row lengths", [](Gather & c) { c.s.E = 64; });
    want_gather(range, "more than the cache holds", [](Gather & c) { c.n = 51; });
    Gather g;
    const size_t gw = tsr_hip_kv_gather_ws(&ctx, &g.d, 40);
    if (gw != 2u * 2u * 1280u) { printf("gather workspace %zu\n", gw); ++n_bad; }
    want_gather(arg, "a small workspace", [&](Gather & c) { c.self = true; c.ws = 0x8000; c.ws_bytes = gw - 1; });
    want_gather(0, "a workspace", [&](Gather & c) { c.self = true; c.ws = 0x8000; c.ws_bytes = gw; });
    if ((uintptr_t)gathers[0].dst != 0x8000) { printf("not the caller's workspace\n"); ++n_bad; }
    capturing = true;
    want_gather(arg, "captured within a cache", [](Gather & c) { c.self = true; });
    want_gather(0, "captured into another", [](Gather &) {});
    capturing = false;
    if (tsr_hip_kv_gather_ws(&ctx, &g.d, 51) || tsr_hip_kv_gather_ws(&ctx, nullptr, 1)) ++n_bad;
    n_bad += plans();
    printf("%d calls\n", n_done);
    return n_bad != 0;
}
