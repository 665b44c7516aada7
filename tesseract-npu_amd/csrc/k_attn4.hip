// k_attn4.hip -- attention of f32 query rows over a 4-bit KV cache (kv4.hpp): o = softmax(scale q K^T + mask) V.
//
// A wave takes 16 NT query rows of one KV head (row r of a KV head is token r / G, query head r % G of the head's G) and
// tiles of 32 cells, one pass with a running maximum and sum; everything stays in registers.
//   scores   S^T[cell][row] = sum over blocks of d[cell] (sum of n q): the matrix instruction f32 <- f16 16x16x32, one a
//            block and piece of q. The operand n is not converted: four bits in the low mantissa bits of an f16 are the
//            subnormal n 2^-24 (2^-20 in the next four), which the instruction multiplies exactly, so that a word of eight
//            codes is unpacked by four ANDs and one shift. q is scaled to [2^13, 2^14) by a power of two a row and split
//            into two f16 pieces (22 bits). The zero point of q4_0 (n - 8) is the instruction's starting value
//            -8 sum(q), that of q4_1 (d n + m) one product m sum(q) a block.
//   softmax  in base 2, f32: a lane holds the scores of one row for four cells of every 16, which is, cells
//            permuted, the second operand of the next product: P stays where it is.
//   P V      O^T[value][row]: the first operand are codes as they are again, the second p d[cell] of a block in two f16
//            pieces (one instruction makes each: f16(p d), f16(p d - hi)). p carries 2^k with 2^k max|d| in [2^14, 2^15)
//            from the plane's header, so that no piece overflows and the pieces keep 2^-39 of the largest. The zero
//            point -8 sum(p d) (q4_1: + sum(p m)) is summed aside in f32.
// The scales meet the f32 sums only, where a cell that its row does not see is replaced by nothing: an infinity or a
// NaN in a masked cell reaches no result. Sums, maxima and results are f32; both splits keep 22 bits of f32's 24.
#include "kernels.hpp"
#include "kv4.hpp"
#include "tsr_dev.hpp"

namespace tsr {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float half_of(uint32_t w, int i) {     // f16 half i of a word, as f32
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> (16 * i)));
}
__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// The eight codes of two words whose nibbles sit at bits 0 and 16 (times 16: at bits 4 and 20) of the word and of the
// word shifted by 8.
__device__ __forceinline__ h8 codes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(h8, make_uint4(a, b, c, d));
}
// max / sum over the four lanes that hold one row (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float rows_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(fb(x), fb(x), false, false);
    x = fmaxf(bf(a[0]), bf(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(fb(x), fb(x), false, false);
    return fmaxf(bf(b[0]), bf(b[1]));
}
__device__ __forceinline__ float rows_sum(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(fb(x), fb(x), false, false);
    x = bf(a[0]) + bf(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(fb(x), fb(x), false, false);
    return bf(b[0]) + bf(b[1]);
}

constexpr uint32_t kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;

// One tile's operands of a plane as a lane holds them.
template <int D, uint32_t TYPE>
struct KTile {
    uint2 w[D / 64][2];                         // codes of 16 cells x 64 values
    uint4 sc[D / 64][2][TYPE == kKvQ4_1 ? 2 : 1];
};
template <int D, uint32_t TYPE>
struct VTile {
    uint4 w[D / 64];
    uint4 sc[D / 64][2][TYPE == kKvQ4_1 ? 2 : 1];
};

// The word {d of block 0, d of block 1} of cell i (of the lane's four) and, q4_1, {m, m}.
template <uint32_t TYPE, class T>
__device__ __forceinline__ uint32_t scale_d(const T & sc, int i) {
    if constexpr (TYPE == kKvQ4_1) return i == 0 ? sc[0].x : i == 1 ? sc[0].z : i == 2 ? sc[1].x : sc[1].z;
    else return i == 0 ? sc[0].x : i == 1 ? sc[0].y : i == 2 ? sc[0].z : sc[0].w;
}
template <class T>
__device__ __forceinline__ uint32_t scale_m(const T & sc, int i) {
    return i == 0 ? sc[0].y : i == 1 ? sc[0].w : i == 2 ? sc[1].y : sc[1].w;
}

template <int D, uint32_t TYPE>
__device__ __forceinline__ void load_scales(uint4 (&sc)[2][TYPE == kKvQ4_1 ? 2 : 1], const uint8_t * t, uint32_t g) {
    constexpr uint32_t n = TYPE == kKvQ4_1 ? 2u : 1u;
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s)
#pragma unroll
        for (uint32_t j = 0; j < n; ++j) sc[s][j] = *(const uint4 *)(t + 1024u + 4u * n * (16u * s + 4u * g) + 16u * j);
}

// SPLIT: the four waves of a workgroup have the same rows and take different tiles; else each has rows of its own.
template <int D, int NT, uint32_t TYPE, bool SPLIT>
struct Attn4 {
    static constexpr int NB = D / 32, NP = D / 64;
    struct Row {                                // of the lane's query row in each group of 16
        uint32_t lo0, hi0, lo1, hi1, t;
    };
    Row row[NT];
    h8 qh[NT][NB], ql[NT][NB];
    float qs[NT][NB];                           // sum of the block's q, times 2^-24
    float csc[NT];                              // scores' unit, base 2
    f4 o[NT][2 * NB];
    float bias[NT][NB];
    float m[NT], l[NT];

    __device__ __forceinline__ bool sees(int n, uint32_t c) const {
        return (c >= row[n].lo0 && c < row[n].hi0) || (c >= row[n].lo1 && c < row[n].hi1);
    }

    __device__ __forceinline__ void load_rows(const Attn4Args & a, uint32_t h, uint32_t r0, uint32_t lane) {
        const uint32_t g = lane >> 4;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t r = r0 + 16u * n + (lane & 15u);
            const uint32_t ru = min(r, a.T * a.G - 1u), t = ru / a.G, hq = h * a.G + ru % a.G;   // (past the last: its copies)
            Row & w = row[n];
            w.t = t;
            if (a.runs != nullptr) {
                const uint4 u = *(const uint4 *)(a.runs + 4u * (size_t)t);
                w.lo0 = u.x;
                w.hi0 = min(u.y, a.n_kv);
                w.lo1 = u.z;
                w.hi1 = min(u.w, a.n_kv);
            } else {
                w.lo0 = w.lo1 = w.hi1 = 0u;
                w.hi0 = a.n_kv;
            }
            const float * q = a.q + (size_t)t * a.q_stride + (size_t)hq * D + 4u * g;
            float x[NB][8], top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float4 u = *(const float4 *)(q + 32 * b), v = *(const float4 *)(q + 32 * b + 16);
                x[b][0] = u.x; x[b][1] = u.y; x[b][2] = u.z; x[b][3] = u.w;
                x[b][4] = v.x; x[b][5] = v.y; x[b][6] = v.z; x[b][7] = v.w;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[b][i]));
            }
            top = rows_max(top);
            const int e = 140 - (int)(fb(top) >> 23);              // 2^e top in [2^13, 2^14)
            csc[n] = __builtin_ldexpf(a.scale * kLog2e, 24 - e);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float sum = 0.0f;
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    y[i] = __builtin_ldexpf(x[b][i], e);
                    sum += y[i];
                    if (i >= 4) y[i] *= 0.0625f;                   // these meet codes times 16
                }
                qs[n][b] = rows_sum(sum) * 0x1p-24f;
                const float z[8] = { y[0], y[2], y[4], y[6], y[1], y[3], y[5], y[7] };
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const _Float16 hi = (_Float16)z[i];
                    qh[n][b][i] = hi;
                    ql[n][b][i] = (_Float16)(z[i] - (float)hi);
                }
                bias[n][b] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 2 * NB; ++j) o[n][j] = f4{ 0.0f, 0.0f, 0.0f, 0.0f };
            m[n] = -__builtin_inff();
            l[n] = 0.0f;
        }
    }

    __device__ __forceinline__ void load_k(KTile<D, TYPE> & k, const uint8_t * p, size_t pair, uint32_t lane) const {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const uint8_t * t = p + j * pair;
#pragma unroll
            for (int s = 0; s < 2; ++s) k.w[j][s] = *(const uint2 *)(t + 512u * s + 8u * lane);
            load_scales<D, TYPE>(k.sc[j], t, lane >> 4);
        }
    }
    __device__ __forceinline__ void load_v(VTile<D, TYPE> & v, const uint8_t * p, size_t pair, uint32_t lane) const {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const uint8_t * t = p + j * pair;
            v.w[j] = *(const uint4 *)(t + 16u * lane);
            load_scales<D, TYPE>(v.sc[j], t, lane >> 4);
        }
    }

    __device__ __forceinline__ void scores(const KTile<D, TYPE> & k, f4 (&s)[NT][2]) const {
        constexpr uint32_t L = 0x000F000Fu, H = 0x00F000F0u;
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = f4{ 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int bb = 0; bb < 2; ++bb) {
                    const int b = 2 * j + bb;
                    const uint32_t w = bb ? k.w[j][u].y : k.w[j][u].x, w8 = w >> 8;
                    const h8 c = codes(w & L, w & H, w8 & L, w8 & H);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float z = TYPE == kKvQ4_0 ? -8.0f * qs[n][b] : 0.0f;
                        f4 x = mfma(c, qh[n][b], f4{ z, z, z, z });
                        x = mfma(c, ql[n][b], x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s[n][u][i] = __builtin_fmaf(half_of(scale_d<TYPE>(k.sc[j][u], i), bb), x[i], s[n][u][i]);
                            if constexpr (TYPE == kKvQ4_1)
                                s[n][u][i] = __builtin_fmaf(half_of(scale_m(k.sc[j][u], i), bb), qs[n][b], s[n][u][i]);
                        }
                    }
                }
    }

    // One tile: MASKED when some row does not see all of it (or a mask is given); c0 its first cell.
    template <bool MASKED>
    __device__ __forceinline__ void tile(const Attn4Args & a, f4 (&s)[NT][2], const VTile<D, TYPE> & v, uint32_t c0,
                                         uint32_t lane, float kexp) {
        constexpr uint32_t L = 0x000F000Fu, H = 0x00F000F0u;
        const uint32_t g = lane >> 4;
        uint32_t vis[NT];                                          // bit 4 u + i: the lane's cell i of group u
        bool grow = false;
        float top[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            vis[n] = 0xFFu;
            if constexpr (MASKED) {
                vis[n] = 0u;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t c = c0 + 16u * u + 4u * g + i;
                        bool in = sees(n, c);
                        float x = s[n][u][i] * csc[n];
                        if (a.mask != nullptr && in) {
                            const float w = h2f_fast(a.mask[(size_t)row[n].t * a.mask_stride + c]);
                            in = w != -__builtin_inff();
                            x = __builtin_fmaf(w, kLog2e, x);
                        }
                        vis[n] |= in ? 1u << (4 * u + i) : 0u;
                        s[n][u][i] = in ? x : -__builtin_inff();
                    }
            } else {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][u][i] *= csc[n];
            }
            float x = fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3]));
            x = fmaxf(x, fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
            top[n] = rows_max(x);
            grow |= top[n] > m[n];
        }
        if (__ballot(grow)) {                                      // a new maximum: what is summed so far shrinks
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float mn = fmaxf(m[n], top[n]);
                const float f = mn == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - mn);
                m[n] = mn;
                l[n] *= f;
#pragma unroll
                for (int b = 0; b < NB; ++b) bias[n][b] *= f;
#pragma unroll
                for (int j = 0; j < 2 * NB; ++j) o[n][j] *= f;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float sub = (m[n] == -__builtin_inff() ? 0.0f : m[n]) - kexp;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[n][u][i] = __builtin_amdgcn_exp2f(s[n][u][i] - sub);
                    l[n] += s[n][u][i];
                }
        }
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int bb = 0; bb < 2; ++bb) {
                const int b = 2 * j + bb;
                const uint32_t w0 = bb ? v.w[j].z : v.w[j].x, w1 = bb ? v.w[j].w : v.w[j].y, x0 = w0 >> 8, x1 = w1 >> 8;
                const h8 clo = codes(w0 & L, x0 & L, w1 & L, x1 & L), chi = codes(w0 & H, x0 & H, w1 & H, x1 & H);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    h8 ph, pl;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool in = !MASKED || ((vis[n] >> (4 * u + i)) & 1u);
                            const float d = half_of(in ? scale_d<TYPE>(v.sc[j][u], i) : 0u, bb);
                            const float p = s[n][u][i];
                            const _Float16 hi = (_Float16)__builtin_fmaf(p, d, -0.0f);
                            ph[4 * u + i] = hi;
                            pl[4 * u + i] = (_Float16)__builtin_fmaf(p, d, -(float)hi);
                            if constexpr (TYPE == kKvQ4_0) bias[n][b] = __builtin_fmaf(p, d, bias[n][b]);
                            else bias[n][b] = __builtin_fmaf(p, half_of(in ? scale_m(v.sc[j][u], i) : 0u, bb), bias[n][b]);
                        }
                    o[n][2 * b] = mfma(clo, ph, o[n][2 * b]);
                    o[n][2 * b] = mfma(clo, pl, o[n][2 * b]);
                    o[n][2 * b + 1] = mfma(chi, ph, o[n][2 * b + 1]);
                    o[n][2 * b + 1] = mfma(chi, pl, o[n][2 * b + 1]);
                }
            }
    }

    // The next tile at or after i (in steps) that a row of the wave sees; t1 when there is none.
    __device__ __forceinline__ uint32_t next(uint32_t i, uint32_t t1, uint32_t step) const {
        for (; i < t1; i += step) {
            bool any = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
                any |= (row[n].lo0 < row[n].hi0 && row[n].lo0 < 32u * i + 32u && row[n].hi0 > 32u * i) ||
                       (row[n].lo1 < row[n].hi1 && row[n].lo1 < 32u * i + 32u && row[n].hi1 > 32u * i);
            if (__ballot(any)) break;
        }
        return min(i, t1);
    }
    __device__ __forceinline__ bool whole(const Attn4Args & a, uint32_t i) const {
        bool all = a.mask == nullptr;
#pragma unroll
        for (int n = 0; n < NT; ++n)
            all = all && ((row[n].lo0 <= 32u * i && row[n].hi0 >= 32u * i + 32u) ||
                          (row[n].lo1 <= 32u * i && row[n].hi1 >= 32u * i + 32u));
        return __ballot(!all) == 0ull;
    }
    // The tiles that the rows can see: [lo, hi)
    __device__ __forceinline__ void hull(uint32_t & t0, uint32_t & t1) const {
        uint32_t lo = 0xFFFFFFFFu, hi = 0u;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (row[n].lo0 < row[n].hi0) { lo = min(lo, row[n].lo0); hi = max(hi, row[n].hi0); }
            if (row[n].lo1 < row[n].hi1) { lo = min(lo, row[n].lo1); hi = max(hi, row[n].hi1); }
        }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            lo = min(lo, (uint32_t)__shfl_xor((int)lo, d));
            hi = max(hi, (uint32_t)__shfl_xor((int)hi, d));
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
        t0 = min(lo, hi) / 32u;
        t1 = (uint32_t)(((uint64_t)hi + 31u) / 32u);
    }

    __device__ __forceinline__ void run(const Attn4Args & a, uint32_t h, uint32_t part, uint32_t parts, uint32_t lane) {
        const size_t tb = kv4_tile_bytes(TYPE), pair = (size_t)a.n_tiles * tb;
        const uint8_t * kp = a.k + kKv4Header + (size_t)h * NP * pair, * vp = a.v + kKv4Header + (size_t)h * NP * pair;
        // 2^k: the largest |d| of the V plane times 2^k in [2^14, 2^15) (an infinite one counts as the largest finite)
        const uint32_t dm = *(const uint32_t *)a.v;
        const float top = (float)__builtin_bit_cast(_Float16, (uint16_t)min(dm, 0x7BFFu));
        const float kexp = top == 0.0f ? 0.0f : (float)(14 - ((int)(fb(top) >> 23) - 127));
        uint32_t t0, t1;
        hull(t0, t1);
        uint32_t i = next(t0 + part, t1, parts);
        if (i >= t1) return;
        KTile<D, TYPE> k;
        VTile<D, TYPE> v;
        load_k(k, kp + i * tb, pair, lane);
        load_v(v, vp + i * tb, pair, lane);
        for (;;) {
            const uint32_t nx = next(i + parts, t1, parts), ld = nx < t1 ? nx : i;
            f4 s[NT][2];
            scores(k, s);
            load_k(k, kp + ld * tb, pair, lane);
            if (whole(a, i)) tile<false>(a, s, v, 32u * i, lane, kexp);
            else tile<true>(a, s, v, 32u * i, lane, kexp);
            if (nx >= t1) break;
            load_v(v, vp + ld * tb, pair, lane);
            i = nx;
        }
    }

    // Rows summed over their lanes; o becomes sum p v (2^k times), value 32 b + 16 c + 4 g + i in o[2 b + c][i].
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            l[n] = rows_sum(l[n]);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float z = rows_sum(bias[n][b]) * (TYPE == kKvQ4_0 ? -8.0f : 1.0f);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[n][2 * b][i] = __builtin_fmaf(o[n][2 * b][i], 0x1p24f, z);
                    o[n][2 * b + 1][i] = __builtin_fmaf(o[n][2 * b + 1][i], 0x1p20f, z);
                }
            }
        }
    }
};

// Workgroup (KV head, split, group of rows), KV heads fastest: with eight of them every XCD's L2 holds one head.
template <int D, int NT, uint32_t TYPE, bool SPLIT>
__global__ __launch_bounds__(256, D >= 256 || NT > 1 ? 1 : 2) void k_attn4(Attn4Args a) {
    using A = Attn4<D, NT, TYPE, SPLIT>;
    constexpr uint32_t kRows = 16u * NT * (SPLIT ? 1u : kWaves);
    const uint32_t h = blockIdx.x % a.n_head_kv, rest = blockIdx.x / a.n_head_kv, split = rest % a.S;
    const uint32_t n_rg = gridDim.x / a.n_head_kv / a.S, rg = n_rg - 1u - rest / a.S;   // causal: the long rows first
    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x & 63u, g = lane >> 4;
    const uint32_t r0 = rg * kRows + (SPLIT ? 0u : 16u * NT * wave), R = a.T * a.G;
    A w;
    w.load_rows(a, h, r0, lane);
    if constexpr (SPLIT) w.run(a, h, split * kWaves + wave, a.S * kWaves, lane);
    else w.run(a, h, split, a.S, lane);
    w.finish();
    if constexpr (SPLIT) {                                         // the waves' sums joined
        constexpr uint32_t DC = D < 128 ? D : 128;                  // values joined at a time
        __shared__ float lm[kWaves * 16 * NT], ll[kWaves * 16 * NT];
        __shared__ __align__(16) float lo[kWaves * 16 * NT * DC];
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if (g == 0u) {
                lm[wave * 16 * NT + 16 * n + lane] = w.m[n];
                ll[wave * 16 * NT + 16 * n + lane] = w.l[n];
            }
        __syncthreads();
        float f[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t r = 16u * n + (lane & 15u);
            float M = lm[r];
#pragma unroll
            for (uint32_t x = 1; x < kWaves; ++x) M = fmaxf(M, lm[x * 16 * NT + r]);
            f[n] = M == w.m[n] ? 1.0f : __builtin_amdgcn_exp2f(w.m[n] - M);
        }
#pragma unroll
        for (uint32_t c = 0; c < D / DC; ++c) {
            if (c != 0u) __syncthreads();
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (uint32_t j = 0; j < DC / 16; ++j) {
                    const f4 x = w.o[n][c * (DC / 16) + j] * f[n];
                    *(float4 *)(lo + (wave * 16 * NT + 16 * n + (lane & 15u)) * DC + 16 * j + 4 * g) =
                        make_float4(x[0], x[1], x[2], x[3]);
                }
            __syncthreads();
            for (uint32_t e = threadIdx.x; e < 16u * NT * (DC / 4); e += 256u) {
                const uint32_t r = e / (DC / 4), d = 4u * (e % (DC / 4));
                if (r0 + r >= R) continue;
                float M = lm[r], L = 0.0f;
#pragma unroll
                for (uint32_t x = 1; x < kWaves; ++x) M = fmaxf(M, lm[x * 16 * NT + r]);
                float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (uint32_t x = 0; x < kWaves; ++x) {
                    const float mx = lm[x * 16 * NT + r];
                    L += ll[x * 16 * NT + r] * (mx == M ? 1.0f : __builtin_amdgcn_exp2f(mx - M));
                    const float4 z = *(const float4 *)(lo + (x * 16 * NT + r) * DC + d);
                    y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
                }
                const uint32_t t = (r0 + r) / a.G, hq = h * a.G + (r0 + r) % a.G, nh = a.G * a.n_head_kv;
                const size_t nr = (size_t)a.T * nh, ro = (size_t)t * nh + hq;
                if (a.S == 1u) {
                    const float il = L == 0.0f ? 0.0f : 1.0f / L;
                    *(float4 *)(a.out + (size_t)t * a.out_stride + (size_t)hq * D + c * DC + d) =
                        make_float4(y.x * il, y.y * il, y.z * il, y.w * il);
                } else {
                    *(float4 *)(a.part + 2u * a.S * nr + (split * nr + ro) * D + c * DC + d) = y;
                    if (c == 0u && d == 0u) *(float2 *)(a.part + 2u * (split * nr + ro)) = make_float2(M, L);
                }
            }
        }
    } else {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t r = r0 + 16u * n + (lane & 15u);
            if (r >= R) continue;
            const uint32_t t = r / a.G, hq = h * a.G + r % a.G, nh = a.G * a.n_head_kv;
            const size_t nr = (size_t)a.T * nh, ro = (size_t)t * nh + hq;
            const float f = a.S > 1u ? 1.0f : w.l[n] == 0.0f ? 0.0f : 1.0f / w.l[n];
            float * y = a.S > 1u ? a.part + 2u * a.S * nr + (split * nr + ro) * D
                                 : a.out + (size_t)t * a.out_stride + (size_t)hq * D;
#pragma unroll
            for (int j = 0; j < 2 * A::NB; ++j) {
                const f4 x = w.o[n][j] * f;
                *(float4 *)(y + 16 * j + 4 * g) = make_float4(x[0], x[1], x[2], x[3]);
            }
            if (a.S > 1u && g == 0u) *(float2 *)(a.part + 2u * (split * nr + ro)) = make_float2(w.m[n], w.l[n]);
        }
    }
}

// The splits of a row joined, in order: a thread a value.
template <int D>
__global__ __launch_bounds__(D) void k_attn4_join(Attn4Args a) {
    const uint32_t ro = blockIdx.x, nh = a.G * a.n_head_kv, d = threadIdx.x;
    const size_t nr = (size_t)a.T * nh;
    const float2 * ml = (const float2 *)a.part;
    const float * po = a.part + 2u * a.S * nr + (size_t)ro * D + d;
    float M = -__builtin_inff();
    for (uint32_t s = 0; s < a.S; ++s) M = fmaxf(M, ml[s * nr + ro].x);
    float y = 0.0f, L = 0.0f;
    for (uint32_t s = 0; s < a.S; ++s) {
        const float2 e = ml[s * nr + ro];
        const float f = e.x == M ? 1.0f : __builtin_amdgcn_exp2f(e.x - M);
        L += e.y * f;
        y += po[s * nr * D] * f;
    }
    a.out[(size_t)(ro / nh) * a.out_stride + (size_t)(ro % nh) * D + d] = L == 0.0f ? 0.0f : y / L;
}

template <int D, int NT, uint32_t TYPE, bool SPLIT>
static int launch(const Attn4Args & a, hipStream_t s) {
    const uint32_t rows = 16u * NT * (SPLIT ? 1u : kWaves), n_rg = (a.T * a.G + rows - 1u) / rows;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_attn4<D, NT, TYPE, SPLIT>), dim3(n_rg * a.S * a.n_head_kv), dim3(256), 0, s, a);
    if (a.S > 1u) hipLaunchKernelGGL(k_attn4_join<D>, dim3(a.T * a.G * a.n_head_kv), dim3(D), 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

template <int D>
static int launch_d(const Attn4Args & a, bool split, hipStream_t s) {
    if (a.type == kKvQ4_0) return split ? launch<D, 1, kKvQ4_0, true>(a, s) : launch<D, 1, kKvQ4_0, false>(a, s);
    return split ? launch<D, 1, kKvQ4_1, true>(a, s) : launch<D, 1, kKvQ4_1, false>(a, s);
}

}  // namespace tsr

int tsr_launch_attn4(const tsr::Attn4Args & a, bool split_waves, hipStream_t s) {
    switch (a.D) {
        case 64: return tsr::launch_d<64>(a, split_waves, s);
        case 128: return tsr::launch_d<128>(a, split_waves, s);
        case 256: return tsr::launch_d<256>(a, split_waves, s);
        case 512: return tsr::launch_d<512>(a, split_waves, s);
        default: return -2;
    }
}
