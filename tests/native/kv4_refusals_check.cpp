// The argument checks of the attention over 4-bit KV caches (csrc/tsr_kv4.hip), without a device: calls that are refused
// launch nothing, and what is launched are whole chunks of the call.
#include <hip/hip_runtime.h>

hipError_t hipSetDevice(int);
#include "tsr_kv4.hip"

#include <cstdio>
#include <vector>

static bool capturing;
static std::vector<tsr::Attn4Args> launched;
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
int tsr_launch_attn4(const tsr::Attn4Args & a, const tsr::Attn4Plan &, hipStream_t) { launched.push_back(a); return 0; }

static int n_bad, n_done;
struct Call {
    uint32_t T = 2, D = 64, nh = 4, nkv = 2, n_kv = 40;
    float scale = 0.125f;
    uint64_t qs = 256, os = 256, ms = 40;
    uintptr_t q = 0x1000, out = 0x2000, runs = 0, mask = 0, ws = 0;
    size_t ws_bytes = 0;
    tsr_hip_kv k, v;
    Call() { k.type = v.type = TSR_HIP_KV_Q4_0; k.E = v.E = 128; k.kv_size = v.kv_size = 64; }
};
static tsr_hip_ctx ctx;
static int run(const Call & c) {
    launched.clear();
    return tsr_hip_flash_attn_kv4(&ctx, (const float *)c.q, c.T, c.qs, &c.k, &c.v, c.D, c.nh, c.nkv, c.scale, c.n_kv, (const uint32_t *)c.runs,
                                  (const uint16_t *)c.mask, c.ms, (float *)c.out, c.os, (void *)c.ws, c.ws_bytes, nullptr);
}
template <class F>
static void want(int rc, const char * what, F change) {
    Call c;
    change(c);
    const int got = run(c);
    ++n_done;
    if (got != rc || (rc != 0 && !launched.empty())) { printf("%s: %d, not %d\n", what, got, rc); ++n_bad; }
}

int main() {
    ctx.n_cu = 256;
    const int arg = TSR_HIP_E_ARG, shape = TSR_HIP_E_SHAPE, fmt = TSR_HIP_E_FMT, range = TSR_HIP_E_RANGE;
    want(0, "the call", [](Call &) {});
    want(0, "no cells", [](Call & c) { c.n_kv = 0; });
    want(arg, "no queries", [](Call & c) { c.q = 0; });
    want(arg, "no output", [](Call & c) { c.out = 0; });
    want(arg, "no tokens", [](Call & c) { c.T = 0; });
    want(arg, "too many tokens", [](Call & c) { c.T = 65536; });
    want(shape, "head size", [](Call & c) { c.D = 96; });
    want(shape, "no heads", [](Call & c) { c.nh = 0; });
    want(shape, "no KV heads", [](Call & c) { c.nkv = 0; });
    want(shape, "heads that are not shared evenly", [](Call & c) { c.nh = 5; });
    want(shape, "65 heads a KV head", [](Call & c) { c.nh = 65; c.nkv = 1; c.k.E = c.v.E = 64; });
    want(shape, "rows too long", [](Call & c) { c.nh = 1024; c.nkv = 512; c.k.E = c.v.E = 32768; });
    want(shape, "scale 0", [](Call & c) { c.scale = 0.0f; });
    want(shape, "scale NaN", [](Call & c) { c.scale = __builtin_nanf(""); });
    want(shape, "scale inf", [](Call & c) { c.scale = __builtin_inff(); });
    want(shape, "subnormal scale", [](Call & c) { c.scale = 1e-39f; });
    want(fmt, "q8_0 caches", [](Call & c) { c.k.type = c.v.type = TSR_HIP_KV_Q8_0; });
    want(fmt, "two types", [](Call & c) { c.v.type = TSR_HIP_KV_Q4_1; });
    want(shape, "another row length", [](Call & c) { c.k.E = 192; });
    want(shape, "another cache length", [](Call & c) { c.v.kv_size = 65; });
    want(range, "cells past the cache", [](Call & c) { c.n_kv = 65; });
    want(arg, "unaligned queries", [](Call & c) { c.q += 8; });
    want(arg, "unaligned output", [](Call & c) { c.out += 4; });
    want(arg, "unaligned runs", [](Call & c) { c.runs = 0x3008; });
    want(arg, "a mask at an odd byte", [](Call & c) { c.mask = 0x4001; });
    want(arg, "query rows that overlap", [](Call & c) { c.qs = 252; });
    want(arg, "a query stride of 258", [](Call & c) { c.qs = 258; });
    want(arg, "output rows that overlap", [](Call & c) { c.os = 128; });
    want(arg, "mask rows that overlap", [](Call & c) { c.mask = 0x4000; c.ms = 39; });
    want(0, "one row needs no strides", [](Call & c) { c.T = 1; c.qs = c.os = c.ms = 0; c.mask = 0x4002; });
    // calls in splits: the workspace
    auto split = [](Call & c) { c.T = 1; c.k.kv_size = c.v.kv_size = c.n_kv = 8192; };
    const size_t ws = tsr_hip_flash_attn_kv4_ws(&ctx, 1, 64, 4, 2, 8192);
    if (ws == 0) { printf("no split\n"); ++n_bad; }
    want(arg, "a small workspace", [&](Call & c) { split(c); c.ws = 0x8000; c.ws_bytes = ws - 1; });
    want(arg, "an unaligned workspace", [&](Call & c) { split(c); c.ws = 0x8004; c.ws_bytes = ws; });
    want(0, "a workspace", [&](Call & c) { split(c); c.ws = 0x8000; c.ws_bytes = ws; });
    if (launched.size() != 1 || (uintptr_t)launched[0].part != 0x8000 || reserved != 0) { printf("not the caller's workspace\n"); ++n_bad; }
    capturing = true;
    want(arg, "a captured call that needs a workspace", split);
    want(0, "a captured call that needs none", [](Call &) {});
    want(0, "a captured call with its own", [&](Call & c) { split(c); c.ws = 0x8000; c.ws_bytes = ws; });
    capturing = false;
    want(0, "the context's scratch", split);
    if (reserved < ws || (uintptr_t)launched[0].part != 0x10000) { printf("scratch of %zu\n", reserved); ++n_bad; }
    // chunks
    want(0, "65535 tokens", [](Call & c) { c.T = 65535; c.runs = 0x100000; c.mask = 0x200000; });
    uint64_t t = 0;
    for (const tsr::Attn4Args & a : launched) {
        if ((uintptr_t)a.q != 0x1000 + t * 256 * 4 || (uintptr_t)a.out != 0x2000 + t * 256 * 4 || (uintptr_t)a.runs != 0x100000 + 16 * t ||
            (uintptr_t)a.mask != 0x200000 + 2 * 40 * t || a.T == 0u || a.T > kTokens) {
            printf("chunk at %llu\n", (unsigned long long)t);
            ++n_bad;
        }
        t += a.T;
    }
    if (t != 65535) { printf("%llu tokens\n", (unsigned long long)t); ++n_bad; }
    if (tsr_hip_flash_attn_kv4_ws(nullptr, 1, 64, 4, 2, 8192) || tsr_hip_flash_attn_kv4_ws(&ctx, 1, 96, 4, 2, 8192)) { printf("ws\n"); ++n_bad; }
    printf("%d calls\n", n_done);
    return n_bad != 0;
}
