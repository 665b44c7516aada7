// k_attn4.hip -- attention of f32 query rows over a 4-bit KV cache (kv4.hpp): o = softmax(scale q K^T + mask) V.
//
// A wave takes 16 NT query rows of one KV head (row r of a KV head is token r / G, query head r % G of the head's G) and
// tiles of 32 cells, one pass with a running maximum and sum; everything stays in registers.
//   scores   S^T[cell][row] = sum over blocks of d[cell] (sum of n q): the matrix instruction f32 <- f16 16x16x32, one a
//            block and piece of q. The first operand are n - 8 (q4_1: n), made of a word of eight codes by an AND with an OR
//            and one packed f16 operation a pair. q is scaled to [2^13, 2^14) by a power of two a row and split into two f16
//            pieces (22 bits). q4_1 (d n + m) adds m sum(q) a block.
//   softmax  in base 2, f32: a lane holds the scores of one row for four cells of every 16, which is, cells
//            permuted, the second operand of the next product: P stays where it is.
//   P V      O^T[value][row]: the first operand are n - 8 again, the second p d[cell] of a block in two f16 pieces (one instruction makes each: f16(p d),
//            f16(p d - hi)). Sums of raw codes would be large and nearly cancel: an error that grows with the root of the
//            cells. p carries 2^k with 2^k max|d| in [2^8, 2^9) from the plane's header and is at most 2^6 (the maximum
//            follows when it is passed by that), so that no piece overflows and the pieces keep 2^-33 of the largest.
//            q4_1: sum p (m + 8 d) is summed aside in f32.
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
// n - zero of the nibbles at bits 0 and 16 of a word ((1024 + n) - (1024 + zero)) and at bits 4 and 20 ((1024 + 16 n) / 16 -
// (64 + zero)), exact. (The bits alone, as subnormals n 2^-24, would save the packed operation; but the instruction aligns
// subnormal operands by their nominal exponent and loses four bits of every product.)
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t magic) {
    uint32_t r;                                 // one operation: of its two constants only one may be a scalar register
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(magic));
    return r;
}
__device__ __forceinline__ h2 codes_lo(uint32_t w, uint32_t magic, float zero) {
    const _Float16 z = (_Float16)(-1024.0f - zero);
    return __builtin_bit_cast(h2, and_or(w, 0x000F000Fu, magic)) + h2{ z, z };
}
__device__ __forceinline__ h2 codes_hi(uint32_t w, uint32_t magic, float zero) {
    const _Float16 z = (_Float16)(-64.0f - zero), f = (_Float16)0.0625f;
    return __builtin_elementwise_fma(__builtin_bit_cast(h2, and_or(w, 0x00F000F0u, magic)), h2{ f, f }, h2{ z, z });
}
// Two f32 as f16. The word is made once: left to itself the compiler rounds an operand of the matrix instruction and the
// same value in the residual that follows it by different instructions, once and twice, which differ in rare ties.
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
    uint32_t w = __builtin_bit_cast(uint32_t, h2{ (_Float16)a, (_Float16)b });
    asm("" : "+v"(w));
    return w;
}
__device__ __forceinline__ h8 of_words(const uint32_t (&w)[4]) { return __builtin_bit_cast(h8, make_uint4(w[0], w[1], w[2], w[3])); }
__device__ __forceinline__ h8 four(h2 a, h2 b, h2 c, h2 d) { return h8{ a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1] }; }
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
#ifndef FENCE
#define FENCE 256
#endif
constexpr int kFence = FENCE;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 6.0f;                  // weights are at most 2^6: a maximum is followed when it is passed by more

// A tile of one plane as a lane holds it: the codes, and of the scales the words of one cell (the lane's place in its row of
// 16 lanes says which): the others are fetched from the row's lanes when they are needed.
template <int D, uint32_t TYPE>
struct Tile {
    uint4 w[D / 64];                            // K: two groups of 16 cells x two blocks; V: two blocks x two groups
    uint32_t d[D / 64];                         // {d, d of the next cell}
    uint32_t m[TYPE == kKvQ4_1 ? D / 64 : 1];
};
// The word that lane I of the row of 16 lanes holds: block I / 4, group of 16 cells I / 2 % 2, cells 4 g + 2 (I % 2) and
// the next.
template <int I>
__device__ __forceinline__ uint32_t from_row(uint32_t w) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)w, 0x150 + I, 0xF, 0xF, true);
}
__device__ __forceinline__ void all_cells(uint32_t w, uint32_t (&x)[2][4]) {
    x[0][0] = from_row<0>(w); x[0][1] = from_row<1>(w); x[0][2] = from_row<2>(w); x[0][3] = from_row<3>(w);
    x[1][0] = from_row<4>(w); x[1][1] = from_row<5>(w); x[1][2] = from_row<6>(w); x[1][3] = from_row<7>(w);
}

// SPLIT: the four waves of a workgroup have the same rows and take different tiles; else each has rows of its own.
template <int D, int NT, uint32_t TYPE, bool SPLIT>
struct Attn4 {
    static constexpr int NB = D / 32;                              // blocks of a head
    static constexpr int AHEAD = D >= 512 ? 1 : 2;                 // tiles loaded ahead
    using Tl = Tile<D, TYPE>;
    struct Row {                                                   // of the lane's query row in each group of 16
        uint32_t lo0, hi0, lo1, hi1, t;
    };
    Row row[NT];
    float qs[NT][TYPE == kKvQ4_1 ? NB : 1];                        // q4_1: sum of the block's q
    float csc[NT];                                                 // the scores' unit, base 2
    f4 o[NT][2 * NB];
    float bias[NT][TYPE == kKvQ4_1 ? NB : 1];                      // q4_1: sum p (m + 8 d)
    float m[NT], l[NT];
    uint32_t magic;                                                // 0x64006400 (f16 1024) in a vector register

    __device__ __forceinline__ bool sees(int n, uint32_t c) const {
        return (c >= row[n].lo0 && c < row[n].hi0) || (c >= row[n].lo1 && c < row[n].hi1);
    }

    // The rows' runs and queries; put: this wave writes the queries' pieces to `lds` (the caller's barrier follows).
    __device__ __forceinline__ void load_rows(const Attn4Args & a, uint32_t h, uint32_t r0, uint32_t lane, h8 * lds, bool put) {
        const uint32_t g = lane >> 4;
        asm("v_mov_b32 %0, 0x64006400" : "=v"(magic));
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
            float top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float4 u = *(const float4 *)(q + 32 * b), v = *(const float4 *)(q + 32 * b + 16);
                top = fmaxf(fmaxf(fmaxf(top, fabsf(u.x)), fmaxf(fabsf(u.y), fabsf(u.z))), fabsf(u.w));
                top = fmaxf(fmaxf(fmaxf(top, fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
            }
            top = rows_max(top);
            asm volatile("" : "+v"(q));                            // (read again rather than kept: D 512 has no registers for it)
            const int e = 140 - (int)(fb(top) >> 23);              // 2^e top in [2^13, 2^14)
            csc[n] = __builtin_ldexpf(a.scale * kLog2e, -e);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float4 u = *(const float4 *)(q + 32 * b), v = *(const float4 *)(q + 32 * b + 16);
                const float x[8] = { u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w };
                float sum = 0.0f;
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    y[i] = __builtin_ldexpf(x[i], e);
                    sum += y[i];
                }
                if constexpr (TYPE == kKvQ4_1) qs[n][b] = rows_sum(sum);
                if (put) {
                    const float z[8] = { y[0], y[2], y[4], y[6], y[1], y[3], y[5], y[7] };
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        hi[i] = pair_of(z[2 * i], z[2 * i + 1]);
                        lo[i] = pair_of(z[2 * i] - half_of(hi[i], 0), z[2 * i + 1] - half_of(hi[i], 1));
                    }
                    lds[((n * NB + b) * 2 + 0) * 64 + lane] = of_words(hi);
                    lds[((n * NB + b) * 2 + 1) * 64 + lane] = of_words(lo);
                }
            }
#pragma unroll
            for (int b = 0; b < (TYPE == kKvQ4_1 ? NB : 1); ++b) bias[n][b] = 0.0f;
#pragma unroll
            for (int j = 0; j < 2 * NB; ++j) o[n][j] = f4{ 0.0f, 0.0f, 0.0f, 0.0f };
            m[n] = -__builtin_inff();
            l[n] = 0.0f;
        }
    }

    template <bool V>
    static __device__ __forceinline__ void load(Tl & k, const uint8_t * p, size_t pair, uint32_t lane) {
        const uint32_t word = 8u * (lane >> 4) + (lane & 7u);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            const uint8_t * t = p + j * pair;
            if constexpr (V) {
                k.w[j] = *(const uint4 *)(t + 16u * lane);
            } else {
                const uint2 x = *(const uint2 *)(t + 8u * lane), y = *(const uint2 *)(t + 512u + 8u * lane);
                k.w[j] = make_uint4(x.x, x.y, y.x, y.y);
            }
            if constexpr (TYPE == kKvQ4_1) {
                const uint2 z = *(const uint2 *)(t + 1024u + 8u * word);
                k.d[j] = z.x;
                k.m[j] = z.y;
            } else {
                k.d[j] = *(const uint32_t *)(t + 1024u + 4u * word);
            }
        }
    }

    __device__ __forceinline__ void scores(const Tl & k, const h8 * q, f4 (&s)[NT][2]) const {
        constexpr float zero = TYPE == kKvQ4_0 ? 8.0f : 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = f4{ 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            uint32_t dw[2][4], mw[2][4];
            all_cells(k.d[j], dw);
            if constexpr (TYPE == kKvQ4_1) all_cells(k.m[j], mw);
#pragma unroll
            for (int bb = 0; bb < 2; ++bb) {
                const int b = 2 * j + bb;
                if constexpr (D >= kFence) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t w = u ? (bb ? k.w[j].w : k.w[j].z) : (bb ? k.w[j].y : k.w[j].x);
                    const h8 n8 = four(codes_lo(w, magic, zero), codes_hi(w, magic, zero), codes_lo(w >> 8, magic, zero), codes_hi(w >> 8, magic, zero));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        f4 x = mfma(n8, q[((n * NB + b) * 2 + 0) * 64], f4{ 0.0f, 0.0f, 0.0f, 0.0f });
                        x = mfma(n8, q[((n * NB + b) * 2 + 1) * 64], x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int y = 2 * u + (i >> 1);
                            s[n][u][i] = __builtin_fmaf(half_of(dw[bb][y], i & 1), x[i], s[n][u][i]);
                            if constexpr (TYPE == kKvQ4_1) s[n][u][i] = __builtin_fmaf(half_of(mw[bb][y], i & 1), qs[n][b], s[n][u][i]);
                        }
                    }
                }
            }
        }
    }

    // The weights of a tile from its scores: s becomes p 2^k. MASKED when some row does not see all of it (or a mask is
    // given): vis gets the cells that the lane's row sees (bit 4 u + i: its cell i of group u). c0: the first cell.
    template <bool MASKED>
    __device__ __forceinline__ void weights(const Attn4Args & a, f4 (&s)[NT][2], uint32_t (&vis)[NT], uint32_t c0, uint32_t lane,
                                            float kexp) {
        const uint32_t g = lane >> 4;
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
            }
            float x = fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3]));
            x = fmaxf(x, fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
            top[n] = MASKED ? x : x * csc[n];
            grow |= top[n] > m[n] + kSlack;
        }
        if (__ballot(grow)) {                                      // a larger maximum: what is summed so far shrinks
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float mn = fmaxf(m[n], rows_max(top[n]));
                const float f = mn == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - mn);
                m[n] = mn;
                l[n] *= f;
#pragma unroll
                for (int b = 0; b < (TYPE == kKvQ4_1 ? NB : 1); ++b) bias[n][b] *= f;
#pragma unroll
                for (int j = 0; j < 2 * NB; ++j) o[n][j] *= f;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float sub = kexp - (m[n] == -__builtin_inff() ? 0.0f : m[n]), unit = MASKED ? 1.0f : csc[n];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[n][u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][u][i], unit, sub));
                    l[n] += s[n][u][i];
                }
        }
    }

    template <bool MASKED>
    __device__ __forceinline__ void values(const Tl & v, const f4 (&s)[NT][2], const uint32_t (&vis)[NT]) {
        uint32_t p16[NT][4], in[NT][4];                            // of the cells 2 x, 2 x + 1 of the lane's eight
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                p16[n][x] = pair_of(s[n][x >> 1][2 * (x & 1)], s[n][x >> 1][2 * (x & 1) + 1]);
                in[n][x] = ((vis[n] >> (2 * x)) & 1u ? 0x0000FFFFu : 0u) | ((vis[n] >> (2 * x)) & 2u ? 0xFFFF0000u : 0u);
            }
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            uint32_t dw[2][4], mw[2][4];
            all_cells(v.d[j], dw);
            if constexpr (TYPE == kKvQ4_1) all_cells(v.m[j], mw);
#pragma unroll
            for (int bb = 0; bb < 2; ++bb) {
                const int b = 2 * j + bb;
                if constexpr (D >= kFence) __builtin_amdgcn_sched_barrier(0);
                const uint32_t w0 = bb ? v.w[j].z : v.w[j].x, w1 = bb ? v.w[j].w : v.w[j].y;
                const h8 clo = four(codes_lo(w0, magic, 8.0f), codes_lo(w0 >> 8, magic, 8.0f), codes_lo(w1, magic, 8.0f), codes_lo(w1 >> 8, magic, 8.0f));
                const h8 chi = four(codes_hi(w0, magic, 8.0f), codes_hi(w0 >> 8, magic, 8.0f), codes_hi(w1, magic, 8.0f), codes_hi(w1 >> 8, magic, 8.0f));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint32_t ph[4], pl[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float p0 = s[n][x >> 1][2 * (x & 1)], p1 = s[n][x >> 1][2 * (x & 1) + 1];
                        const uint32_t d = MASKED ? dw[bb][x] & in[n][x] : dw[bb][x];
                        const h2 hi = __builtin_bit_cast(h2, p16[n][x]) * __builtin_bit_cast(h2, d);
                        ph[x] = __builtin_bit_cast(uint32_t, hi);
                        pl[x] = pair_of(__builtin_fmaf(p0, half_of(d, 0), -half_of(ph[x], 0)), __builtin_fmaf(p1, half_of(d, 1), -half_of(ph[x], 1)));
                        if constexpr (TYPE == kKvQ4_1) {
                            const uint32_t m = MASKED ? mw[bb][x] & in[n][x] : mw[bb][x];
                            bias[n][b] = __builtin_fmaf(p0, __builtin_fmaf(half_of(d, 0), 8.0f, half_of(m, 0)), bias[n][b]);
                            bias[n][b] = __builtin_fmaf(p1, __builtin_fmaf(half_of(d, 1), 8.0f, half_of(m, 1)), bias[n][b]);
                        }
                    }
                    o[n][2 * b] = mfma(clo, of_words(ph), o[n][2 * b]);
                    o[n][2 * b + 1] = mfma(chi, of_words(ph), o[n][2 * b + 1]);
                    o[n][2 * b] = mfma(clo, of_words(pl), o[n][2 * b]);
                    o[n][2 * b + 1] = mfma(chi, of_words(pl), o[n][2 * b + 1]);
                }
            }
        }
    }

    // The next tile at or after i (in steps) that all rows of the wave see whole (WHOLE; none under a mask), or that a row
    // sees and not all see whole; t1 when there is none.
    template <bool WHOLE>
    __device__ __forceinline__ uint32_t next(const Attn4Args & a, uint32_t i, uint32_t t1, uint32_t step) const {
        for (; i < t1; i += step) {
            const uint32_t c0 = 32u * i, c1 = c0 + 32u;
            bool any = false, all = a.mask == nullptr;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                all = all && ((row[n].lo0 <= c0 && row[n].hi0 >= c1) || (row[n].lo1 <= c0 && row[n].hi1 >= c1));
                any |= (row[n].lo0 < row[n].hi0 && row[n].lo0 < c1 && row[n].hi0 > c0) ||
                       (row[n].lo1 < row[n].hi1 && row[n].lo1 < c1 && row[n].hi1 > c0);
            }
            const bool whole = __ballot(!all) == 0ull;
            if (WHOLE ? whole : (!whole && __ballot(any) != 0ull)) break;
        }
        return min(i, t1);
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
        t1 = (hi + 31u) / 32u;                                     // (cells stay below 2^31)
    }

    // The tiles t0, t0 + parts, .. below t1 that are (not) whole, the next two loaded ahead.
    template <bool WHOLE>
    __device__ __forceinline__ void tiles(const Attn4Args & a, const uint8_t * kp, const uint8_t * vp, size_t pair, uint32_t t0,
                                          uint32_t t1, uint32_t parts, float kexp, const h8 * lds, uint32_t lane) {
        constexpr size_t tb = kv4_tile_bytes(TYPE);
        uint32_t i0 = next<WHOLE>(a, t0, t1, parts);
        if (i0 >= t1) return;
        uint32_t i1 = next<WHOLE>(a, i0 + parts, t1, parts);
        Tl k0, v0, k1, v1;
        load<false>(k0, kp + i0 * tb, pair, lane);
        load<true>(v0, vp + i0 * tb, pair, lane);
        if constexpr (AHEAD == 2) {
            const size_t c1 = (i1 < t1 ? i1 : i0) * tb;            // (past the last tile: the one before again)
            load<false>(k1, kp + c1, pair, lane);
            load<true>(v1, vp + c1, pair, lane);
        }
        auto one = [&](Tl & k, Tl & v, uint32_t i, uint32_t ahead) {
            uint32_t ql = lane;                                    // the pieces of q are read from LDS for every tile: kept in
            asm volatile("" : "+v"(ql));                           // registers they would spill
            f4 s[NT][2];
            uint32_t vis[NT];
            const size_t c = (ahead < t1 ? ahead : i) * tb;
            scores(k, lds + ql, s);
            load<false>(k, kp + c, pair, lane);
            weights<!WHOLE>(a, s, vis, 32u * i, lane, kexp);
            values<!WHOLE>(v, s, vis);
            load<true>(v, vp + c, pair, lane);
        };
        if constexpr (AHEAD == 1) {
            for (;;) {
                one(k0, v0, i0, i1);
                if (i1 >= t1) return;
                i0 = i1;
                i1 = next<WHOLE>(a, i0 + parts, t1, parts);
            }
        }
        for (;;) {
            const uint32_t i2 = next<WHOLE>(a, i1 + parts, t1, parts);
            one(k0, v0, i0, i2);
            if (i1 >= t1) break;
            const uint32_t i3 = next<WHOLE>(a, i2 + parts, t1, parts);
            one(k1, v1, i1, i3);
            if (i2 >= t1) break;
            i0 = i2;
            i1 = i3;
        }
    }
    __device__ __forceinline__ void run(const Attn4Args & a, uint32_t h, uint32_t part, uint32_t parts, const h8 * lds, uint32_t lane) {
        const size_t pair = (size_t)a.n_tiles * kv4_tile_bytes(TYPE);
        const uint8_t * kp = a.k + kKv4Header + (size_t)h * (D / 64) * pair, * vp = a.v + kKv4Header + (size_t)h * (D / 64) * pair;
        // 2^k: the largest |d| of the V plane times 2^k in [2^8, 2^9) (an infinite one counts as the largest finite), k <= 9
        const uint32_t dm = *(const uint32_t *)a.v;
        const float top = (float)__builtin_bit_cast(_Float16, (uint16_t)min(dm, 0x7BFFu));
        const float kexp = top == 0.0f ? 0.0f : (float)min(8 - ((int)(fb(top) >> 23) - 127), 9);
        uint32_t t0, t1;
        hull(t0, t1);
        tiles<true>(a, kp, vp, pair, t0 + part, t1, parts, kexp, lds, lane);
        tiles<false>(a, kp, vp, pair, t0 + part, t1, parts, kexp, lds, lane);
    }

    // Rows summed over their lanes; o becomes sum p v (2^k times), value 32 b + 16 c + 4 g + i in o[2 b + c][i].
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            l[n] = rows_sum(l[n]);
            if constexpr (TYPE == kKvQ4_1)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float z = rows_sum(bias[n][b]);
                    o[n][2 * b] += z;
                    o[n][2 * b + 1] += z;
                }
        }
    }
};

// Workgroup (KV head, split, group of rows), KV heads fastest: with eight of them every XCD's L2 holds one head.
template <int D, int NT, uint32_t TYPE, bool SPLIT>
__global__ __launch_bounds__(256, D == 64 ? 4 : D <= 256 ? 2 : 1) void k_attn4(Attn4Args a) {
    using A = Attn4<D, NT, TYPE, SPLIT>;
    constexpr uint32_t kRows = 16u * NT * (SPLIT ? 1u : kWaves);
    const uint32_t h = blockIdx.x % a.n_head_kv, rest = blockIdx.x / a.n_head_kv, split = rest % a.S;
    const uint32_t n_rg = gridDim.x / a.n_head_kv / a.S, rg = n_rg - 1u - rest / a.S;   // causal: the long rows first
    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x & 63u, g = lane >> 4;
    const uint32_t r0 = rg * kRows + (SPLIT ? 0u : 16u * NT * wave), R = a.T * a.G;
    __shared__ h8 lq[(SPLIT ? 1 : kWaves) * NT * A::NB * 2 * 64];
    A w;
    w.load_rows(a, h, r0, lane, lq + (SPLIT ? 0u : wave) * NT * A::NB * 2 * 64, !SPLIT || wave == 0u);
    __syncthreads();
    if constexpr (SPLIT) w.run(a, h, split * kWaves + wave, a.S * kWaves, lq, lane);
    else w.run(a, h, split, a.S, lq + wave * NT * A::NB * 2 * 64, lane);
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

// The splits of a row joined: a workgroup a row, 256 / (D / 4) threads of the same four values take splits in turn, then
// meet in LDS; the order of the additions is fixed.
template <int D>
__global__ __launch_bounds__(256) void k_attn4_join(Attn4Args a) {
    constexpr uint32_t W = D / 4, NG = 256u / W;
    __shared__ float4 acc[256];
    __shared__ float wt[64];
    const uint32_t ro = blockIdx.x, nh = a.G * a.n_head_kv, c = threadIdx.x % W, s0 = threadIdx.x / W;
    const size_t nr = (size_t)a.T * nh;
    const float4 * po = (const float4 *)(a.part + 2u * a.S * nr + (size_t)ro * D) + c;
    if (threadIdx.x < 64u) {                                       // S <= 64: a lane a split
        float2 e = make_float2(-__builtin_inff(), 0.0f);
        if (threadIdx.x < a.S) e = ((const float2 *)a.part)[threadIdx.x * nr + ro];
        float M = e.x;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) M = fmaxf(M, __shfl_xor(M, d));
        const float f = e.x == M ? 1.0f : __builtin_amdgcn_exp2f(e.x - M);
        float L = e.y * f;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) L += __shfl_xor(L, d);
        wt[threadIdx.x] = L == 0.0f ? 0.0f : f / L;
    }
    float4 x[64 / NG];
#pragma unroll
    for (uint32_t i = 0; i < 64u / NG; ++i)                        // all loads in flight at once
        x[i] = s0 + NG * i < a.S ? po[(size_t)(s0 + NG * i) * nr * W] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __syncthreads();
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (uint32_t i = 0; i < 64u / NG; ++i) {
        const float f = wt[s0 + NG * i];
        if (s0 + NG * i < a.S) { y.x += x[i].x * f; y.y += x[i].y * f; y.z += x[i].z * f; y.w += x[i].w * f; }
    }
    acc[threadIdx.x] = y;
    __syncthreads();
    if (s0 == 0u) {
#pragma unroll
        for (uint32_t i = 1; i < NG; ++i) {
            const float4 z = acc[i * W + c];
            y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
        }
        *((float4 *)(a.out + (size_t)(ro / nh) * a.out_stride + (size_t)(ro % nh) * D) + c) = y;
    }
}

template <int D, int NT, uint32_t TYPE, bool SPLIT>
static int launch(const Attn4Args & a, hipStream_t s) {
    const uint32_t rows = 16u * NT * (SPLIT ? 1u : kWaves), n_rg = (a.T * a.G + rows - 1u) / rows;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_attn4<D, NT, TYPE, SPLIT>), dim3(n_rg * a.S * a.n_head_kv), dim3(256), 0, s, a);
    if (a.S > 1u) hipLaunchKernelGGL(k_attn4_join<D>, dim3(a.T * a.G * a.n_head_kv), dim3(256), 0, s, a);
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
