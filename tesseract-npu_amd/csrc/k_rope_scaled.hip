// k_rope_scaled.hip -- rotary positions scaled for contexts beyond the trained one.
//
// Pair i of a head turns by pos f_i, f_i = base^(-2 i / n) / ff_i (s (1 - w_i) + w_i): s is the interpolation of positions
// (trained / new length), w_i the share of the pair's own frequency, which YaRN keeps for pairs that turn often within the
// trained length and gives up over a ramp of i. An angle is many turns at far positions (131071 rad for pair 0), of which
// only the fraction counts: f_i, the angle, its reduction to an eighth of a turn and the sine and cosine (Taylor sums, 1.2e-10
// from the truth there) are f64, rounded to f32 once; on f32 they would be off by 0.008 rad. f64 operations run here at the rate of f32's.
//
// A workgroup rotates one token's heads: its first threads make the token's n / 2 pairs of cosine and sine, while the
// values of its units are on their way. A unit is four values (interleaved pairs) or two times four (halves), and where rows
// are not of whole aligned quads a pair, or a single value to copy; one thread reads and writes all of it, so that y may be x.
//
// Bound: the rows' bytes, once in and once out. 2047 tokens of 40 heads of 128 (84 MB) take 18.6 us, 4.5 TB/s where a large
// copy reaches 4.65; the f64 angles hide behind them. One token is a launch (5.0 us a call).
#include "kernels.hpp"
#include "tsr_dev.hpp"

namespace tsr {

constexpr uint32_t kRsThreads = 256u, kRsUnits = 4u;               // units a thread has in flight

// m cos and m sin of the angle of pair i at position pos.
__device__ __forceinline__ float2 rope_scaled_cs(const RopeScaledArgs & a, int32_t pos, uint32_t i) {
    double f = exp2(a.log2_step * (double)i);
    if (a.ff != nullptr) f /= (double)a.ff[i];
    const double w = a.ext * (1.0 - fmin(fmax(((double)i - a.ramp_lo) / a.ramp_len, 0.0), 1.0));
    f *= a.freq_scale * (1.0 - w) + w;
    const double turns = (double)pos * f * 0.63661977236758134308;  // quarters of a turn: angle 2 / pi
    const double k = __builtin_rint(turns);
    const double x = (turns - k) * 1.57079632679489661923, z = x * x;
    // sin x and cos x for |x| <= pi / 4: Taylor's sums to x^11 and x^10
    const double s = x + x * z * (-1.0 / 6 + z * (1.0 / 120 + z * (-1.0 / 5040 + z * (1.0 / 362880 - z * (1.0 / 39916800)))));
    const double c = 1.0 + z * (-0.5 + z * (1.0 / 24 + z * (-1.0 / 720 + z * (1.0 / 40320 - z * (1.0 / 3628800)))));
    const uint32_t q = (uint32_t)(k - 4.0 * __builtin_floor(k * 0.25));   // quarter 0 .. 3
    const double u = q & 1u ? s : c, v = q & 1u ? c : s;
    return make_float2((float)(a.m * (q == 1u || q == 2u ? -u : u)), (float)(a.m * (q >= 2u ? -v : v)));
}

template <int V>
struct RsVec {
    float v[V];
};
template <int V>
__device__ __forceinline__ RsVec<V> rs_load(const float * p) {
    RsVec<V> r;
    if constexpr (V == 4) {
        const float4 x = *(const float4 *)p;
        r.v[0] = x.x; r.v[1] = x.y; r.v[2] = x.z; r.v[3] = x.w;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = p[i];
    }
    return r;
}
template <int V>
__device__ __forceinline__ void rs_store(float * p, const RsVec<V> & r) {
    if constexpr (V == 4) {
        *(float4 *)p = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = r.v[i];
    }
}

// Pairs turned by ROPE's operations (k_glue.hip: subnormals are 0, a NaN is the canonical one), so that the fused attention calls,
// which take the angles as a table, give the same bits. Plain products and sums are these but for values that a class test finds,
// and then all of a unit's are made again by the rules (2047 tokens of 40 heads: 22.4 us by the rules alone).
__device__ __forceinline__ bool rs_odd(float x) { return __builtin_amdgcn_classf(x, 0x93); }   // subnormal or a NaN
template <int N>
__device__ __forceinline__ void rs_turn(float (&p)[N], float (&q)[N], const float2 (&cs)[N]) {
    float x[N], y[N];
    bool odd = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float pc = p[i] * cs[i].x, qs = q[i] * cs[i].y, ps = p[i] * cs[i].y, qc = q[i] * cs[i].x;
        x[i] = pc - qs;
        y[i] = ps + qc;
        odd |= rs_odd(p[i]) | rs_odd(q[i]) | rs_odd(pc) | rs_odd(qs) | rs_odd(ps) | rs_odd(qc) | rs_odd(x[i]) | rs_odd(y[i]);
    }
    if (__builtin_expect(odd, 0)) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = ssub(smul(p[i], cs[i].x), smul(q[i], cs[i].y));
            y[i] = sadd(smul(p[i], cs[i].y), smul(q[i], cs[i].x));
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = x[i], q[i] = y[i];
}

// Units of a head: first those that turn (n_dims / V interleaved; n_dims / (2 V) halves), then those that are copied, of V
// values where V is 4, else of one.
template <int V, bool HALVES>
__global__ __launch_bounds__(kRsThreads) void k_rope_scaled(RopeScaledArgs a) {
    __shared__ float2 cs[512];
    constexpr uint32_t CW = V == 4 ? 4u : 1u;                      // of a copy
    const uint32_t t = blockIdx.x, half = a.n_dims / 2u, turn = HALVES ? half / V : a.n_dims / V;
    const uint32_t total = a.n_heads * a.units;
    const float * x = a.x + (size_t)t * a.x_stride;
    float * y = a.y + (size_t)t * a.y_stride;
    struct Unit {
        uint32_t at, j;                                            // where it lies in the row, its place in the head
        RsVec<V> p, q;
    };
    Unit u[kRsUnits];
    const uint32_t first = blockIdx.y * kRsThreads * kRsUnits + threadIdx.x;
#pragma unroll
    for (uint32_t k = 0; k < kRsUnits; ++k) {
        const uint32_t i = first + k * kRsThreads;
        if (i < total) {
            const uint32_t h = a.units == 1u ? i : __umulhi(i, a.inv_units), w = i - h * a.units;
            const float * px = x + (size_t)h * a.head_dim;
            u[k].j = w;
            u[k].at = h * a.head_dim;
            if (w >= turn) {
                u[k].at += a.n_dims + (w - turn) * CW;
                if constexpr (V == CW) u[k].p = rs_load<V>(x + u[k].at);
                else u[k].p.v[0] = x[u[k].at];
            } else {
                u[k].at += w * V;
                u[k].p = rs_load<V>(px + w * V);
                if constexpr (HALVES) u[k].q = rs_load<V>(px + w * V + half);
            }
        }
    }
    const int32_t pos = a.pos[t];
    for (uint32_t i = threadIdx.x; i < half; i += kRsThreads) {
        const float2 c = rope_scaled_cs(a, pos, i);
        cs[i] = make_float2(daz(c.x), daz(c.y));
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kRsUnits; ++k) {
        if (first + k * kRsThreads >= total) continue;
        Unit & w = u[k];
        if (w.j >= turn) {
            if constexpr (V == CW) rs_store<V>(y + w.at, w.p);
            else y[w.at] = w.p.v[0];
        } else {
            constexpr int N = HALVES ? V : V / 2;
            float p[N], q[N];
            float2 c[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                p[i] = w.p.v[HALVES ? i : 2 * i];
                q[i] = HALVES ? w.q.v[i] : w.p.v[2 * i + 1];
                c[i] = cs[HALVES ? w.j * V + i : w.j * V / 2u + i];
            }
            rs_turn(p, q, c);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                w.p.v[HALVES ? i : 2 * i] = p[i];
                if constexpr (HALVES) w.q.v[i] = q[i];
                else w.p.v[2 * i + 1] = q[i];
            }
            rs_store<V>(y + w.at, w.p);
            if constexpr (HALVES) rs_store<V>(y + w.at + half, w.q);
        }
    }
}

__global__ __launch_bounds__(64) void k_rope_scaled_table(RopeScaledArgs a, float * tab) {
    const uint32_t i = threadIdx.x;
    if (i < a.n_dims / 2u) *(float2 *)(tab + 2u * i) = rope_scaled_cs(a, a.pos[0], i);
}

}  // namespace tsr

int tsr_launch_rope_scaled(tsr::RopeScaledArgs a, uint32_t T, hipStream_t s) {
    // whole aligned quads: every unit is one load or store of 16 bytes
    const bool quads = a.head_dim % 4u == 0u && a.n_dims % (a.halves ? 8u : 4u) == 0u && (a.x_stride | a.y_stride) % 4u == 0u &&
                       (((uintptr_t)a.x | (uintptr_t)a.y) & 15u) == 0u;
    const uint32_t V = quads ? 4u : a.halves ? 1u : 2u;
    a.units = (a.halves ? a.n_dims / 2u : a.n_dims) / V + (a.head_dim - a.n_dims) / (quads ? 4u : 1u);
    a.inv_units = a.units == 1u ? 0u : (uint32_t)((1ull << 32) / a.units) + 1u;
    const uint32_t total = a.n_heads * a.units, per = tsr::kRsThreads * tsr::kRsUnits;
    const dim3 grid(T, (total + per - 1u) / per), wg(tsr::kRsThreads);
    if (quads && a.halves) hipLaunchKernelGGL(HIP_KERNEL_NAME(tsr::k_rope_scaled<4, true>), grid, wg, 0, s, a);
    else if (quads) hipLaunchKernelGGL(HIP_KERNEL_NAME(tsr::k_rope_scaled<4, false>), grid, wg, 0, s, a);
    else if (a.halves) hipLaunchKernelGGL(HIP_KERNEL_NAME(tsr::k_rope_scaled<1, true>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(tsr::k_rope_scaled<2, false>), grid, wg, 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

int tsr_launch_rope_scaled_table(const tsr::RopeScaledArgs & a, float * tab, hipStream_t s) {
    hipLaunchKernelGGL(tsr::k_rope_scaled_table, dim3(1), dim3(64), 0, s, a, tab);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
