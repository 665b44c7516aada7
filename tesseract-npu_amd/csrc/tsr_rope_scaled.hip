// tsr_rope_scaled.hip -- host side of the rotary positions scaled for long contexts.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "kernels.hpp"
#include "runtime.hpp"
#include "tsr_hip.h"

// The scaling's part of the kernels' arguments; false: a scaling that is refused.
static bool scaling_args(const tsr_hip_rope_scaling & r, uint32_t n_dims, tsr::RopeScaledArgs & a) {
    if (!(r.freq_base > 1.0f) || !std::isfinite(r.freq_base)) return false;
    if (!(r.freq_scale > 0.0f) || !std::isfinite(r.freq_scale) || !std::isfinite(r.attn_factor)) return false;
    if (!(r.ext_factor >= 0.0f && r.ext_factor <= 1.0f)) return false;
    const double base = r.freq_base;
    a.log2_step = -2.0 * std::log2(base) / n_dims;
    a.freq_scale = r.freq_scale;
    a.ext = r.ext_factor;
    a.m = r.attn_factor;
    a.ramp_len = 1.0;
    if (r.ext_factor != 0.0f) {
        if (r.n_ctx_orig == 0u || !(r.beta_fast > 0.0f) || !(r.beta_slow > 0.0f) || !std::isfinite(r.beta_fast) ||
            !std::isfinite(r.beta_slow))
            return false;
        // the pair that turns beta times within the trained length
        auto pair_of = [&](double beta) {
            return n_dims * std::log(r.n_ctx_orig / (beta * 2.0 * 3.14159265358979323846)) / (2.0 * std::log(base));
        };
        const double lo = std::max(0.0, std::floor(pair_of(r.beta_fast)));
        const double hi = std::min(n_dims - 1.0, std::ceil(pair_of(r.beta_slow)));
        a.ramp_lo = lo;
        a.ramp_len = std::max(0.001, hi - lo);
        a.m *= 1.0 + 0.1 * std::log(1.0 / a.freq_scale);
    }
    return true;
}

int tsr_hip_rope_scaled(tsr_hip_ctx * ctx, const float * x_dev, uint32_t T, uint64_t x_stride, uint32_t head_dim,
                        uint32_t n_heads, uint32_t n_dims, int mode, const int32_t * pos_dev,
                        const tsr_hip_rope_scaling * scaling, const float * freq_factors_dev, float * y_dev, uint64_t y_stride,
                        void * stream) {
    if (ctx == nullptr || x_dev == nullptr || y_dev == nullptr || pos_dev == nullptr || scaling == nullptr || T == 0u ||
        n_heads == 0u)
        return TSR_HIP_E_ARG;
    if (mode != TSR_HIP_ROPE_NORMAL && mode != TSR_HIP_ROPE_NEOX && mode != TSR_HIP_ROPE_IMROPE) return TSR_HIP_E_SHAPE;
    if (n_dims < 2u || n_dims % 2u != 0u || n_dims > head_dim || n_dims > 1024u || head_dim > 16384u) return TSR_HIP_E_SHAPE;
    const uint64_t width = (uint64_t)head_dim * n_heads;
    if (T >= 1u << 24 || width > (1u << 18)) return TSR_HIP_E_SHAPE;   // (a launch's threads and units below 2^32)
    if (T > 1u && (x_stride < width || y_stride < width || (x_dev == y_dev && x_stride != y_stride))) return TSR_HIP_E_ARG;
    if ((((uintptr_t)x_dev | (uintptr_t)y_dev | (uintptr_t)pos_dev | (uintptr_t)freq_factors_dev) & 3u) != 0u) return TSR_HIP_E_ARG;
    tsr::RopeScaledArgs a{};
    if (!scaling_args(*scaling, n_dims, a)) return TSR_HIP_E_ARG;
    a.x = x_dev;
    a.x_stride = x_stride;
    a.y = y_dev;
    a.y_stride = y_stride;
    a.pos = pos_dev;
    a.ff = freq_factors_dev;
    a.head_dim = head_dim;
    a.n_heads = n_heads;
    a.n_dims = n_dims;
    a.halves = mode != TSR_HIP_ROPE_NORMAL ? 1u : 0u;
    std::lock_guard<std::mutex> lk(ctx->mtx);
    (void)hipSetDevice(ctx->device);
    return tsr_launch_rope_scaled(a, T, ctx->pick(stream)) ? TSR_HIP_E_HIP : TSR_HIP_OK;
}

int tsr_hip_rope_scaled_table(tsr_hip_ctx * ctx, const int32_t * pos_dev, uint32_t n_dims, const tsr_hip_rope_scaling * scaling,
                              const float * freq_factors_dev, float * tab_dev, void * stream) {
    if (ctx == nullptr || pos_dev == nullptr || scaling == nullptr || tab_dev == nullptr || ((uintptr_t)tab_dev & 7u) != 0u)
        return TSR_HIP_E_ARG;
    if (n_dims < 2u || n_dims % 2u != 0u || n_dims > 128u) return TSR_HIP_E_SHAPE;
    tsr::RopeScaledArgs a{};
    if (!scaling_args(*scaling, n_dims, a)) return TSR_HIP_E_ARG;
    a.pos = pos_dev;
    a.ff = freq_factors_dev;
    a.n_dims = n_dims;
    std::lock_guard<std::mutex> lk(ctx->mtx);
    (void)hipSetDevice(ctx->device);
    return tsr_launch_rope_scaled_table(a, tab_dev, ctx->pick(stream)) ? TSR_HIP_E_HIP : TSR_HIP_OK;
}
