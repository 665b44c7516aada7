// The argument checks of the scaled rotary positions (csrc/tsr_rope_scaled.hip), without a device.
#include <hip/hip_runtime.h>

hipError_t hipSetDevice(int);
#include "tsr_rope_scaled.hip"

#include <cstdio>

static int launched, n_bad, n_done;
static tsr::RopeScaledArgs last;
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *) { return hipSuccess; }
int tsr::hip_err(hipError_t e, const char *) { return e == hipSuccess ? 0 : TSR_HIP_E_HIP; }
int tsr_launch_rope_scaled(tsr::RopeScaledArgs a, uint32_t, hipStream_t) { ++launched; last = a; return 0; }
int tsr_launch_rope_scaled_table(const tsr::RopeScaledArgs & a, float *, hipStream_t) { ++launched; last = a; return 0; }

struct Call {
    uint32_t T = 2, hd = 64, heads = 4, n = 64;
    uint64_t xs = 256, ys = 256;
    int mode = TSR_HIP_ROPE_NORMAL;
    uintptr_t x = 0x1000, y = 0x2000, pos = 0x3000, ff = 0, tab = 0x4000;
    tsr_hip_rope_scaling r = { 10000.0f, 0.25f, 1.0f, 1.0f, 32.0f, 1.0f, 4096u };
    bool none = false;
};
static tsr_hip_ctx ctx;
template <class F>
static void want(int rc, int rc_table, const char * what, F change) {
    Call c;
    change(c);
    launched = 0;
    const int got = tsr_hip_rope_scaled(&ctx, (const float *)c.x, c.T, c.xs, c.hd, c.heads, c.n, c.mode, (const int32_t *)c.pos,
                                        c.none ? nullptr : &c.r, (const float *)c.ff, (float *)c.y, c.ys, nullptr);
    const int n = launched;
    const int tab = tsr_hip_rope_scaled_table(&ctx, (const int32_t *)c.pos, c.n, c.none ? nullptr : &c.r, (const float *)c.ff,
                                              (float *)c.tab, nullptr);
    ++n_done;
    if (got != rc || n != (rc == 0) || tab != rc_table || launched != n + (rc_table == 0)) {
        printf("%s: %d and %d\n", what, got, tab);
        ++n_bad;
    }
}

int main() {
    const int arg = TSR_HIP_E_ARG, shape = TSR_HIP_E_SHAPE;
    want(0, 0, "the call", [](Call &) {});
    if (!(last.ramp_lo == 10.0 && last.ramp_len == 13.0)) { printf("ramp %f %f\n", last.ramp_lo, last.ramp_len); ++n_bad; }
    want(arg, 0, "no values", [](Call & c) { c.x = 0; });
    want(arg, 0, "no result", [](Call & c) { c.y = 0; });
    want(arg, arg, "no positions", [](Call & c) { c.pos = 0; });
    want(arg, arg, "no scaling", [](Call & c) { c.none = true; });
    want(arg, 0, "no tokens", [](Call & c) { c.T = 0; });
    want(arg, 0, "no heads", [](Call & c) { c.heads = 0; });
    want(0, arg, "no table", [](Call & c) { c.tab = 0; });
    want(0, arg, "a table at an odd word", [](Call & c) { c.tab = 0x4004; });
    want(shape, 0, "a mode that there is not", [](Call & c) { c.mode = 1; });
    want(0, 0, "the other mode of halves", [](Call & c) { c.mode = TSR_HIP_ROPE_IMROPE; });
    want(shape, shape, "an odd part", [](Call & c) { c.n = 63; });
    want(shape, shape, "no part", [](Call & c) { c.n = 0; });
    want(shape, 0, "a part beyond the head", [](Call & c) { c.n = 66; });
    want(0, shape, "a table of more than 128", [](Call & c) { c.n = 256; c.hd = 256; c.xs = c.ys = 1024; });
    want(shape, shape, "more than 1024", [](Call & c) { c.n = c.hd = 1026; c.xs = c.ys = 5000; });
    want(shape, 0, "rows too long", [](Call & c) { c.heads = 5000; c.xs = c.ys = 1000000; });
    want(arg, 0, "rows that overlap", [](Call & c) { c.xs = 255; });
    want(arg, 0, "results that overlap", [](Call & c) { c.ys = 255; });
    want(0, 0, "one row needs no strides", [](Call & c) { c.T = 1; c.xs = c.ys = 0; });
    want(0, 0, "in place", [](Call & c) { c.y = c.x; });
    want(arg, 0, "in place with another stride", [](Call & c) { c.y = c.x; c.ys = 260; });
    want(0, 0, "one row in place, whatever the strides", [](Call & c) { c.T = 1; c.y = c.x; c.ys = 260; });
    want(0, 0, "as many tokens as a launch holds", [](Call & c) { c.T = (1u << 24) - 1u; });
    want(shape, 0, "more", [](Call & c) { c.T = 1u << 24; });
    want(arg, 0, "a misaligned row", [](Call & c) { c.x = 0x1002; });
    want(arg, arg, "base 1", [](Call & c) { c.r.freq_base = 1.0f; });
    want(arg, arg, "base NaN", [](Call & c) { c.r.freq_base = __builtin_nanf(""); });
    want(arg, arg, "scale 0", [](Call & c) { c.r.freq_scale = 0.0f; });
    want(arg, arg, "scale inf", [](Call & c) { c.r.freq_scale = __builtin_inff(); });
    want(arg, arg, "attention factor NaN", [](Call & c) { c.r.attn_factor = __builtin_nanf(""); });
    want(arg, arg, "ext below 0", [](Call & c) { c.r.ext_factor = -0.5f; });
    want(arg, arg, "ext above 1", [](Call & c) { c.r.ext_factor = 1.5f; });
    want(arg, arg, "no trained length", [](Call & c) { c.r.n_ctx_orig = 0; });
    want(arg, arg, "beta 0", [](Call & c) { c.r.beta_slow = 0.0f; });
    want(0, 0, "no ramp needs no length", [](Call & c) { c.r.ext_factor = 0.0f; c.r.n_ctx_orig = 0; c.r.beta_fast = 0.0f; });
    if (tsr_hip_rope_scaled(nullptr, nullptr, 1, 0, 2, 1, 2, 0, nullptr, nullptr, nullptr, nullptr, 0, nullptr) != arg) ++n_bad;
    printf("%d calls\n", n_done);
    return n_bad != 0;
}
