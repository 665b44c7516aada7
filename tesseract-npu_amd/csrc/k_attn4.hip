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
//   P V      O^T[value][row]: the first operand are n - 8 again, the second p d[cell] of a block in two f16 pieces, f16(p) d
//            rounded once and what p d leaves of it. Sums of raw codes would be large and nearly cancel: an error that grows
//            with the root of the cells. p d carries 2^e with 2^e max|d| in [2^5, 2^9), max|d| the largest finite scale that
//            the row has seen so far, followed like the maximum of its scores; p takes k = min(e, 9) of it and d, exactly, the
//            rest. p is at most 2^6 (the maximum follows when it is passed by that), so that no piece overflows and the
//            pieces keep 2^-30 of the largest. What a row does not see has no part in e: cells of other rows, heads and
//            times change no result's precision. Following e takes 1 to 3 % of a call (512 tokens behind 1536 cells 48.9 ->
//            49.8 us, a token behind 8192 cells 12.7 -> 13.0; heads of 512 over q4_1 up to 17 %, whose registers spill).
//            q4_1: sum p (m + 8 d) is summed aside in f32.
// The scales meet the f32 sums only, where a cell that its row does not see is replaced by nothing: an infinity or a
// NaN in a masked cell reaches no result. Sums, maxima and results are f32; both splits keep 22 bits of f32's 24.
//
// Bound. Few rows: the cells' bytes and two launches: a token of 32 heads of 128 (8 KV heads) takes 13.1 us behind 8192
// cells (a call of a graph of them: 7 the cells, 2.8 the join, the rest between launches) and 43 us behind 131071 of q4_1
// (168 MB, 3.9 TB/s; a plain read of them 29 us). Many rows: vector instructions, about 130 a 16 x 16 tile of scores and
// D 128 (a third the unpacking, a quarter the pieces of p d) against 16 matrix instructions: 2048 tokens behind 6144
// cells take 553 to 574 us (418 to 435 TFLOP/s), vector units 80 %, matrix units 35 % busy. Unpacking once for four waves through LDS,
// V in two pieces, left 270 vector instructions of 466 a tile of 32 rows and was no faster: with 239 registers two waves a
// SIMD hide neither kind behind the other; four groups of rows a workgroup gave nothing.
#include "attn4_plan.hpp"
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

constexpr uint32_t kWaves = 4;                  // of a workgroup
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 6.0f;                  // weights are at most 2^6: a maximum is followed when it is passed by more

// A tile of one plane as a lane holds it: the codes, and the scales. Where a column of the matrix instruction is a query row
// (C 1): of each pair of blocks one word {d, d of the next cell} (the lane's place in its row of 16 lanes says which; the
// others are fetched from the row's lanes when they are needed). Where C columns share a row: the words of the lane's
// eight cells for the blocks C k + c of its column.
template <int D, int C, uint32_t TYPE>
struct Tile {
    uint4 w[D / 64];                            // K: two groups of 16 cells x two blocks; V: two blocks x two groups
    uint32_t d[C == 1 ? D / 64 : 1];
    uint32_t m[C == 1 && TYPE == kKvQ4_1 ? D / 64 : 1];
    uint4 sc[C == 1 ? 1 : D / 32 / C][TYPE == kKvQ4_1 ? 2 : 1];
    // {d, d of the next cell} of the lane's cells 2 x, 2 x + 1 for its k-th block, and {m, m}
    __device__ __forceinline__ uint32_t dk(int k, int x) const {
        const uint4 & u = sc[k][0];
        if constexpr (TYPE == kKvQ4_1) return x == 0 ? u.x : x == 1 ? u.z : x == 2 ? sc[k][TYPE == kKvQ4_1].x : sc[k][TYPE == kKvQ4_1].z;
        return x == 0 ? u.x : x == 1 ? u.y : x == 2 ? u.z : u.w;
    }
    __device__ __forceinline__ uint32_t mk(int k, int x) const {
        const uint4 & u = sc[k][0], & v = sc[k][TYPE == kKvQ4_1];
        return x == 0 ? u.y : x == 1 ? u.w : x == 2 ? v.y : v.w;
    }
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

// The scales of two cells by their size (|d|'s bits), without those that are not finite where FINITE.
typedef uint16_t u2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u2 larger(u2 a, u2 b) { return __builtin_elementwise_max(a, b); }
__device__ __forceinline__ uint32_t larger(u2 a) { return max((uint32_t)a[0], (uint32_t)a[1]); }
template <bool FINITE>
__device__ __forceinline__ u2 sizes(uint32_t w) {
    u2 x = __builtin_bit_cast(u2, w & 0x7FFF7FFFu);
    if constexpr (FINITE) x = u2{ x[0] < 0x7C00u ? x[0] : (uint16_t)0u, x[1] < 0x7C00u ? x[1] : (uint16_t)0u };
    return x;
}
// e of a largest scale: the largest of 21, 17 .. 9 .. -7 with 2^e |d| < 2^9 (steps of 2^4, so that it seldom changes). A wave starts
// with 9, right for 2^-4 <= |d| < 1. The least size for which e is too large, and whether one is small enough for the next.
constexpr int kMostE = 21, kMostK = 9, kFirstE = 9;
__device__ __forceinline__ int e_of(uint32_t size) { return ((30 - (int)(size >> 10)) & ~3) - 7; }
__device__ __forceinline__ uint32_t beyond(int e) { return (uint32_t)(24 - e) << 10; }
__device__ __forceinline__ bool below(uint32_t size, int e) { return e < kMostE && size < beyond(e + 4); }
__device__ __forceinline__ int k_of(int e) { return min(e, kMostK); }
// 2^(e - k), as an f16 pair
__device__ __forceinline__ h2 rest_of(int e) {
    return __builtin_bit_cast(h2, (uint32_t)(15 + e - k_of(e)) * 0x04000400u);
}
__device__ __forceinline__ uint32_t rows_max_u(uint32_t x) {      // over the four lanes that hold one row
    auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(a[0], a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(b[0], b[1]);
}
// The token of row r of a KV head: r / G by a product (r < 2^22, G <= 64: exact).
__device__ __forceinline__ uint32_t token(const Attn4Args & a, uint32_t r) {
    return a.T == 1u ? 0u : a.inv_G == 0u ? r : __umulhi(r, a.inv_G);
}
// Over the wave, by DPP inside the rows of 16 lanes (the four rows hold the same values).
__device__ __forceinline__ uint32_t rows16_min(uint32_t v) {
    v = min(v, (uint32_t)dpp_i<kDppXor1>((int)v));
    v = min(v, (uint32_t)dpp_i<kDppXor2>((int)v));
    v = min(v, (uint32_t)dpp_i<kDppRowHalfMirror>((int)v));
    v = min(v, (uint32_t)dpp_i<kDppRowMirror>((int)v));
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ uint32_t rows16_max(uint32_t v) { return ~rows16_min(~v); }
// Maximum over the C columns of a row (aligned groups of C lanes).
template <int C>
__device__ __forceinline__ uint32_t columns_max(uint32_t x) {
    if constexpr (C >= 2) x = max(x, (uint32_t)dpp_i<kDppXor1>((int)x));
    if constexpr (C >= 4) x = max(x, (uint32_t)dpp_i<kDppXor2>((int)x));
    return x;
}
// Sum over the C columns of a row (aligned groups of C lanes).
template <int C>
__device__ __forceinline__ float columns_sum(float x) {
    if constexpr (C >= 2) x += dpp_f<kDppXor1>(x);
    if constexpr (C >= 4) x += dpp_f<kDppXor2>(x);
    if constexpr (C >= 8) x += dpp_f<kDppRowHalfMirror>(x);
    return x;
}

// The waves of a workgroup have the same rows and take different tiles.
// C: columns of the matrix instruction a query row. With few rows (a decode token's G query heads) 16 / C rows fill the
// 16 columns: column C r + c is row r and meets the blocks C k + c alone (its q is zero for the others, and of its results
// for the values of other blocks nothing is used), so that a lane scales the products and splits the weights of D / 32 / C
// blocks and not of all D / 32.
template <int D, int NT, int C, uint32_t TYPE>
struct Attn4 {
    static constexpr int NB = D / 32, NK = NB / C;                 // blocks of a head, of a column
    static constexpr int RW = 16 / C;                              // query rows of a group of 16 columns
    static constexpr int AHEAD = D >= 256 ? 1 : 2;                 // tiles loaded ahead
    using Tl = Tile<D, C, TYPE>;
    struct Row {                                                   // of the lane's query row in each group of 16
        uint32_t lo0, hi0, lo1, hi1, t;
    };
    Row row[NT];
    const float * qp[NT];
    float qs[NT][TYPE == kKvQ4_1 ? NK : 1];                        // q4_1: sum of the block's q
    float csc[NT];                                                 // the scores' unit, base 2
    f4 o[NT][2 * NB];
    float bias[NT][TYPE == kKvQ4_1 ? NK : 1];                      // q4_1: sum p (m + 8 d)
    float m[NT], l[NT];
    int e[NT];                                                     // o is 2^e, l and bias are 2^min(e, 9) times their sums (until finish)
    uint32_t magic;                                                // 0x64006400 (f16 1024) in a vector register

    __device__ __forceinline__ bool sees(int n, uint32_t c) const {
        return (c >= row[n].lo0 && c < row[n].hi0) || (c >= row[n].lo1 && c < row[n].hi1);
    }

    // The rows' runs, and where the lane's parts of their queries are.
    __device__ __forceinline__ void load_runs(const Attn4Args & a, uint32_t h, uint32_t r0, uint32_t lane) {
        asm("v_mov_b32 %0, 0x64006400" : "=v"(magic));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t r = r0 + RW * n + (lane & 15u) / C;
            const uint32_t ru = min(r, a.T * a.G - 1u), t = token(a, ru), hq = h * a.G + ru - t * a.G;   // (past the last: its copies)
            Row & w = row[n];
            w.t = t;
            uint4 u = make_uint4(0u, a.n_kv, 0u, 0u);
            if (a.runs != nullptr) u = *(const uint4 *)(a.runs + (a.T == 1u ? 0u : 4u * (size_t)t));
            w.lo0 = u.x;
            w.hi0 = min(u.y, a.n_kv);
            w.lo1 = u.z;
            w.hi1 = min(u.w, a.n_kv);
            qp[n] = a.q + (size_t)t * a.q_stride + (size_t)hq * D + 4u * (lane >> 4);
#pragma unroll
            for (int k = 0; k < (TYPE == kKvQ4_1 ? NK : 1); ++k) bias[n][k] = 0.0f;
#pragma unroll
            for (int j = 0; j < 2 * NB; ++j) o[n][j] = f4{ 0.0f, 0.0f, 0.0f, 0.0f };
            m[n] = -__builtin_inff();
            l[n] = 0.0f;
        }
    }
    // The queries; their pieces go to `lds`, [row group][block][piece][lane], the blocks shared out over the waves.
    __device__ __forceinline__ void load_queries(float scale, uint32_t lane, h8 * lds, uint32_t wave) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float * q = qp[n];
            float top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float4 u = *(const float4 *)(q + 32 * b), v = *(const float4 *)(q + 32 * b + 16);
                top = fmaxf(fmaxf(fmaxf(top, fabsf(u.x)), fmaxf(fabsf(u.y), fabsf(u.z))), fabsf(u.w));
                top = fmaxf(fmaxf(fmaxf(top, fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
            }
            top = rows_max(top);
            if constexpr (D > 128) asm volatile("" : "+v"(q));     // (read again rather than kept: no registers for it)
            const int e = 140 - (int)(fb(top) >> 23);              // 2^e top in [2^13, 2^14)
            csc[n] = __builtin_ldexpf(scale, -e) * kLog2e;         // (in this order: scale log2(e) may pass f32's range)
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
                const bool mine = C == 1 || (lane & (C - 1u)) == b % C;
                if constexpr (TYPE == kKvQ4_1) {
                    const float z = rows_sum(sum);
                    if (mine) qs[n][b / C] = z;
                }
                if (b % kWaves == wave) {
                    const float z[8] = { y[0], y[2], y[4], y[6], y[1], y[3], y[5], y[7] };
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        hi[i] = pair_of(z[2 * i], z[2 * i + 1]);
                        lo[i] = pair_of(z[2 * i] - half_of(hi[i], 0), z[2 * i + 1] - half_of(hi[i], 1));
                        if (!mine) hi[i] = lo[i] = 0u;
                    }
                    lds[((n * NB + b) * 2 + 0) * 64 + lane] = of_words(hi);
                    lds[((n * NB + b) * 2 + 1) * 64 + lane] = of_words(lo);
                }
            }
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
            if constexpr (C == 1 && TYPE == kKvQ4_1) {
                const uint2 z = *(const uint2 *)(t + 1024u + 8u * word);
                k.d[j] = z.x;
                k.m[j] = z.y;
            } else if constexpr (C == 1) {
                k.d[j] = *(const uint32_t *)(t + 1024u + 4u * word);
            }
        }
        if constexpr (C > 1)
#pragma unroll
            for (int y = 0; y < NK; ++y) {
                const uint32_t b = C * y + (lane & (C - 1u));
                constexpr uint32_t n = TYPE == kKvQ4_1 ? 2u : 1u;
                const uint8_t * t = p + (b >> 1) * pair + 1024u + 4u * n * (8u * (lane >> 4) + 4u * (b & 1u));
#pragma unroll
                for (uint32_t i = 0; i < n; ++i) k.sc[y][i] = *(const uint4 *)(t + 16u * i);
            }
    }

    __device__ __forceinline__ void scores(const Tl & k, const h8 * q, f4 (&s)[NT][2]) const {
        constexpr float zero = TYPE == kKvQ4_0 ? 8.0f : 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = f4{ 0.0f, 0.0f, 0.0f, 0.0f };
        if constexpr (C > 1) {
#pragma unroll
            for (int y = 0; y < NK; ++y) {
                f4 x[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) x[n][0] = x[n][1] = f4{ 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int b = C * y + c;
                    const uint4 & w4 = k.w[b >> 1];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t w = u ? (b & 1 ? w4.w : w4.z) : (b & 1 ? w4.y : w4.x);
                        const h8 n8 = four(codes_lo(w, magic, zero), codes_hi(w, magic, zero), codes_lo(w >> 8, magic, zero),
                                           codes_hi(w >> 8, magic, zero));
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            x[n][u] = mfma(n8, q[((n * NB + b) * 2 + 0) * 64], x[n][u]);
                            x[n][u] = mfma(n8, q[((n * NB + b) * 2 + 1) * 64], x[n][u]);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int z = 2 * u + (i >> 1);
                            s[n][u][i] = __builtin_fmaf(half_of(k.dk(y, z), i & 1), x[n][u][i], s[n][u][i]);
                            if constexpr (TYPE == kKvQ4_1) s[n][u][i] = __builtin_fmaf(half_of(k.mk(y, z), i & 1), qs[n][y], s[n][u][i]);
                        }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][u][i] = columns_sum<C>(s[n][u][i]);
        } else
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            uint32_t dw[2][4], mw[2][4];
            all_cells(k.d[j], dw);
            if constexpr (TYPE == kKvQ4_1) all_cells(k.m[j], mw);
#pragma unroll
            for (int bb = 0; bb < 2; ++bb) {
                const int b = 2 * j + bb;
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

    // The scales' sizes of a tile of V: of the lane's cells 2 x, 2 x + 1 (MASKED, C > 1), or of all that the lane holds.
    template <bool MASKED>
    using Sizes = u2[MASKED || C > 1 ? 4 : 1];
    template <bool MASKED, bool FINITE>
    static __device__ __forceinline__ void sizes_of(const Tl & v, Sizes<MASKED> & size) {
        if constexpr (C > 1) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                size[x] = sizes<FINITE>(v.dk(0, x));
#pragma unroll
                for (int y = 1; y < NK; ++y) size[x] = larger(size[x], sizes<FINITE>(v.dk(y, x)));
            }
        } else {
            size[0] = sizes<FINITE>(v.d[0]);
#pragma unroll
            for (int j = 1; j < D / 64; ++j) size[0] = larger(size[0], sizes<FINITE>(v.d[j]));
            if constexpr (MASKED) {
                uint32_t z = __builtin_bit_cast(uint32_t, size[0]);    // (the other block of a pair is four lanes on in a row)
                z = __builtin_bit_cast(uint32_t, larger(size[0], __builtin_bit_cast(u2, (uint32_t)__builtin_amdgcn_mov_dpp((int)z, 0x124, 0xF, 0xF, true))));
                size[0] = __builtin_bit_cast(u2, from_row<0>(z));
                size[1] = __builtin_bit_cast(u2, from_row<1>(z));
                size[2] = __builtin_bit_cast(u2, from_row<2>(z));
                size[3] = __builtin_bit_cast(u2, from_row<3>(z));
            }
        }
    }

    // The bits of the lane's cells 2 x, 2 x + 1 that its row sees, as a mask of halves.
    static __device__ __forceinline__ uint32_t cells_in(uint32_t vis, int x) {
        return ((vis >> (2 * x)) & 1u ? 0x0000FFFFu : 0u) | ((vis >> (2 * x)) & 2u ? 0xFFFF0000u : 0u);
    }
    // The largest of them; of the cells that the lane's row sees.
    template <bool MASKED>
    static __device__ __forceinline__ uint32_t all_of(const Sizes<MASKED> & size) {
        if constexpr (C > 1) return larger(larger(larger(size[0], size[1]), larger(size[2], size[3])));
        else return larger(size[0]);
    }
    static __device__ __forceinline__ uint32_t all_seen(const Sizes<true> & size, uint32_t vis) {
        u2 z = { 0, 0 };
#pragma unroll
        for (int y = 0; y < 4; ++y) z = larger(z, __builtin_bit_cast(u2, __builtin_bit_cast(uint32_t, size[y]) & cells_in(vis, y)));
        return larger(z);
    }
    // The weights of a tile from its scores: s becomes p 2^k. MASKED when some row does not see all of it (or a mask is
    // given): vis gets the cells that the lane's row sees (bit 4 u + i: its cell i of group u). c0: the first cell. A larger
    // maximum of the scores, or of the scales of V that a row sees, shrinks what is summed so far: `whole` is e of the
    // tiles that every row sees, the same for all of them.
    template <bool MASKED>
    __device__ __forceinline__ void weights(const Attn4Args & a, f4 (&s)[NT][2], uint32_t (&vis)[NT], const Tl & v, const Sizes<MASKED> & size,
                                            int & whole, bool & first, uint32_t c0, uint32_t lane) {
        const uint32_t g = lane >> 4;
        bool grow = false;
        float top[NT];
        if constexpr (!MASKED) grow = all_of<false>(size) >= beyond(whole);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            vis[n] = 0xFFu;
            if constexpr (MASKED) {
                vis[n] = 0u;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t c = c0 + 16u * u + 4u * g;
                    uint2 w = make_uint2(0u, 0u);                  // the mask's four values
                    if (a.mask != nullptr) {
                        const uint16_t * mp = a.mask + (size_t)row[n].t * a.mask_stride + c;
                        if (a.mask_by4 && c + 4u <= a.n_kv) {
                            w = *(const uint2 *)mp;
                        } else {
                            if (c < a.n_kv) w.x = mp[0];
                            if (c + 1u < a.n_kv) w.x |= (uint32_t)mp[1] << 16;
                            if (c + 2u < a.n_kv) w.y = mp[2];
                            if (c + 3u < a.n_kv) w.y |= (uint32_t)mp[3] << 16;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float z = half_of(i < 2 ? w.x : w.y, i & 1);
                        const bool in = sees(n, c + i) && z != -__builtin_inff();
                        const float x = __builtin_fmaf(z, kLog2e, s[n][u][i] * csc[n]);
                        vis[n] |= in ? 1u << (4 * u + i) : 0u;
                        s[n][u][i] = in ? x : -__builtin_inff();
                    }
                }
            }
            float x = fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3]));
            x = fmaxf(x, fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
            top[n] = MASKED ? x : x * csc[n];
            grow |= top[n] > m[n] + kSlack;
            if constexpr (MASKED) grow |= all_seen(size, vis[n]) >= beyond(e[n]);
        }
        if (__ballot(grow)) {
            bool fresh[NT];                                        // nothing was summed yet
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float mn = fmaxf(m[n], rows_max(top[n]));
                const float f = mn == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - mn);
                fresh[n] = m[n] == -__builtin_inff() && mn != m[n];
                m[n] = mn;
                l[n] *= f;
#pragma unroll
                for (int k = 0; k < (TYPE == kKvQ4_1 ? NK : 1); ++k) bias[n][k] *= f;
#pragma unroll
                for (int j = 0; j < 2 * NB; ++j) o[n][j] *= f;
            }
            bool other;                                            // another e for a row, perhaps
            if constexpr (MASKED) {
                other = false;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint32_t z = columns_max<C>(rows_max_u(all_seen(size, vis[n])));
                    other |= z >= beyond(e[n]) || (fresh[n] && below(z, e[n]));
                }
                other = __ballot(other) != 0ull;
            } else {
                const uint32_t z = all_of<false>(size);
                other = __ballot(z >= beyond(whole)) != 0ull || (first && __ballot(!below(z, whole)) == 0ull);
            }
            if (other) {
                Sizes<MASKED> finite;
                sizes_of<MASKED, true>(v, finite);
                const int was = whole;
                if constexpr (!MASKED) {
                    whole = e_of(rows16_max(rows_max_u(all_of<false>(finite))));
                    if (!first) whole = min(whole, was);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    int e0 = was, e1 = whole;
                    if constexpr (MASKED) {
                        e0 = e[n];
                        e1 = e_of(columns_max<C>(rows_max_u(all_seen(finite, vis[n]))));
                        e[n] = e1 = fresh[n] ? e1 : min(e0, e1);
                    }
                    const float fk = __builtin_ldexpf(1.0f, k_of(e1) - k_of(e0)), fe = __builtin_ldexpf(1.0f, e1 - e0);
                    l[n] *= fk;
#pragma unroll
                    for (int k = 0; k < (TYPE == kKvQ4_1 ? NK : 1); ++k) bias[n][k] *= fk;
#pragma unroll
                    for (int j = 0; j < 2 * NB; ++j) o[n][j] *= fe;
                }
            }
            first = false;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float sub = (float)k_of(MASKED ? e[n] : whole) - (m[n] == -__builtin_inff() ? 0.0f : m[n]), unit = MASKED ? 1.0f : csc[n];
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
    __device__ __forceinline__ void values(const Tl & v, const f4 (&s)[NT][2], const uint32_t (&vis)[NT], int whole) {
        // the scales times their part of 2^e: a tile's, or where the rows differ in it a row's
        h2 rest[NT];
        float eight[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int en = MASKED ? e[n] : whole;
            rest[n] = rest_of(en);
            eight[n] = __builtin_ldexpf(8.0f, k_of(en) - en);
        }
        auto scaled = [&](uint32_t d, int n) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, d) * rest[n]); };
        auto of_tile = [&](uint32_t d) { return MASKED ? d : scaled(d, 0); };
        uint32_t p16[NT][4], in[NT][4];                            // of the cells 2 x, 2 x + 1 of the lane's eight
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                p16[n][x] = pair_of(s[n][x >> 1][2 * (x & 1)], s[n][x >> 1][2 * (x & 1) + 1]);
                in[n][x] = cells_in(vis[n], x);
            }
        // the pieces of the weights times the scales of a block, {d, d of the next cell} in d and {m, m} in mm
        auto pieces = [&](int n, int k, const uint32_t (&dd)[4], const uint32_t (&mm)[4], uint32_t (&ph)[4], uint32_t (&pl)[4]) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float p0 = s[n][x >> 1][2 * (x & 1)], p1 = s[n][x >> 1][2 * (x & 1) + 1];
                const uint32_t d = MASKED ? scaled(dd[x] & in[n][x], n) : dd[x];
                ph[x] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, p16[n][x]) * __builtin_bit_cast(h2, d));
                pl[x] = pair_of(__builtin_fmaf(p0, half_of(d, 0), -half_of(ph[x], 0)), __builtin_fmaf(p1, half_of(d, 1), -half_of(ph[x], 1)));
                if constexpr (TYPE == kKvQ4_1) {
                    const uint32_t m = MASKED ? mm[x] & in[n][x] : mm[x];
                    bias[n][k] = __builtin_fmaf(p0, __builtin_fmaf(half_of(d, 0), eight[n], half_of(m, 0)), bias[n][k]);
                    bias[n][k] = __builtin_fmaf(p1, __builtin_fmaf(half_of(d, 1), eight[n], half_of(m, 1)), bias[n][k]);
                }
            }
        };
        auto add = [&](int b, const uint32_t (&ph)[NT][4], const uint32_t (&pl)[NT][4]) {
            const uint4 & w = v.w[b >> 1];
            const uint32_t w0 = b & 1 ? w.z : w.x, w1 = b & 1 ? w.w : w.y;
            const h8 clo = four(codes_lo(w0, magic, 8.0f), codes_lo(w0 >> 8, magic, 8.0f), codes_lo(w1, magic, 8.0f), codes_lo(w1 >> 8, magic, 8.0f));
            const h8 chi = four(codes_hi(w0, magic, 8.0f), codes_hi(w0 >> 8, magic, 8.0f), codes_hi(w1, magic, 8.0f), codes_hi(w1 >> 8, magic, 8.0f));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                o[n][2 * b] = mfma(clo, of_words(ph[n]), o[n][2 * b]);
                o[n][2 * b + 1] = mfma(chi, of_words(ph[n]), o[n][2 * b + 1]);
                o[n][2 * b] = mfma(clo, of_words(pl[n]), o[n][2 * b]);
                o[n][2 * b + 1] = mfma(chi, of_words(pl[n]), o[n][2 * b + 1]);
            }
        };
        uint32_t ph[NT][4], pl[NT][4];
        if constexpr (C > 1) {
#pragma unroll
            for (int y = 0; y < NK; ++y) {
                const uint32_t dd[4] = { of_tile(v.dk(y, 0)), of_tile(v.dk(y, 1)), of_tile(v.dk(y, 2)), of_tile(v.dk(y, 3)) };
                uint32_t mm[4] = {};
                if constexpr (TYPE == kKvQ4_1)
#pragma unroll
                    for (int x = 0; x < 4; ++x) mm[x] = v.mk(y, x);
#pragma unroll
                for (int n = 0; n < NT; ++n) pieces(n, y, dd, mm, ph[n], pl[n]);
#pragma unroll
                for (int c = 0; c < C; ++c) add(C * y + c, ph, pl);
            }
        } else {
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                uint32_t dw[2][4], mw[2][4] = {};
                all_cells(of_tile(v.d[j]), dw);
                if constexpr (TYPE == kKvQ4_1) all_cells(v.m[j], mw);
#pragma unroll
                for (int bb = 0; bb < 2; ++bb) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) pieces(n, 2 * j + bb, dw[bb], mw[bb], ph[n], pl[n]);
                    add(2 * j + bb, ph, pl);
                }
            }
        }
    }

    // Whether a row of the wave sees a cell of tile i.
    __device__ __forceinline__ bool any(uint32_t i) const {
        const uint32_t c0 = 32u * i, c1 = c0 + 32u;
        bool x = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
            x |= (row[n].lo0 < row[n].hi0 && row[n].lo0 < c1 && row[n].hi0 > c0) ||
                 (row[n].lo1 < row[n].hi1 && row[n].lo1 < c1 && row[n].hi1 > c0);
        return __ballot(x) != 0ull;
    }
    struct Span {                                                  // tiles [lo, hi)
        uint32_t lo, hi;
        __device__ __forceinline__ uint32_t size() const { return hi - lo; }
    };
    // The tiles that every row sees whole by its first (second) run; the tiles that hold all cells that any row sees.
    __device__ __forceinline__ void spans(const Attn4Args & a, Span & w0, Span & w1, Span & all) const {
        uint32_t l0 = 0u, h0 = 0xFFFFFFFFu, l1 = 0u, h1 = 0xFFFFFFFFu, lo = 0xFFFFFFFFu, hi = 0u;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const Row & r = row[n];
            l0 = max(l0, r.lo0); h0 = min(h0, r.hi0);
            l1 = max(l1, r.lo1); h1 = min(h1, r.hi1);
            if (r.lo0 < r.hi0) { lo = min(lo, r.lo0); hi = max(hi, r.hi0); }
            if (r.lo1 < r.hi1) { lo = min(lo, r.lo1); hi = max(hi, r.hi1); }
        }
        if (a.T != 1u) {
            l0 = rows16_max(l0); h0 = rows16_min(h0);
            l1 = rows16_max(l1); h1 = rows16_min(h1);
            lo = rows16_min(lo); hi = rows16_max(hi);
        } else {                                                   // (the lanes agree)
            l0 = __builtin_amdgcn_readfirstlane(l0); h0 = __builtin_amdgcn_readfirstlane(h0);
            l1 = __builtin_amdgcn_readfirstlane(l1); h1 = __builtin_amdgcn_readfirstlane(h1);
            lo = __builtin_amdgcn_readfirstlane(lo); hi = __builtin_amdgcn_readfirstlane(hi);
        }
        all = Span{ min(lo, hi) / 32u, (hi + 31u) / 32u };         // (cells stay below 2^31)
        w0 = Span{ (min(l0, 0x7FFFFFFFu) + 31u) / 32u, h0 / 32u };
        w1 = Span{ (min(l1, 0x7FFFFFFFu) + 31u) / 32u, h1 / 32u };
        if (w0.lo >= w0.hi || a.mask != nullptr) w0 = Span{ all.lo, all.lo };
        if (w1.lo >= w1.hi || a.mask != nullptr) w1 = Span{ all.hi, all.hi };
        if (w1.lo < w0.lo) { const Span x = w0; w0 = w1; w1 = x; }
        w1.lo = max(w1.lo, w0.hi);                                 // (runs that overlap: each tile once)
        w1.hi = max(w1.hi, w1.lo);
    }

    // The scores and the values of one tile, its registers loaded again from tile `ahead` behind their last use.
    template <bool WHOLE>
    __device__ __forceinline__ void one(const Attn4Args & a, Tl & k, Tl & v, uint32_t i, uint32_t ahead, const uint8_t * kp,
                                        const uint8_t * vp, size_t pair, int & whole, bool & first, const h8 * lds, uint32_t lane) {
        uint32_t ql = lane;                                        // q's pieces: read from LDS for every tile where registers
        if constexpr (D * NT > 128) asm volatile("" : "+v"(ql));   // would spill, kept where they do not
        f4 s[NT][2];
        uint32_t vis[NT];
        const size_t c = (size_t)ahead * kv4_tile_bytes(TYPE);
        Sizes<!WHOLE> size;
        sizes_of<!WHOLE, false>(v, size);
        scores(k, lds + ql, s);
        if constexpr (!WHOLE)                                      // (made here: moved behind the mask's branches they would
#pragma unroll                                                     // keep the products and scales of every block in registers)
            for (int n = 0; n < NT; ++n) asm volatile("" : "+v"(s[n][0]), "+v"(s[n][1]));
        load<false>(k, kp + c, pair, lane);
        weights<!WHOLE>(a, s, vis, v, size, whole, first, 32u * i, lane);
        if constexpr (C == 1) {                                    // (from here on: scaled and spread before the softmax they would
#pragma unroll                                                     // take registers of every block)
            for (int j = 0; j < D / 64; ++j) asm volatile("" : "+v"(v.d[j]));
        } else {
#pragma unroll
            for (int y = 0; y < NK; ++y)
#pragma unroll
                for (int z = 0; z < (TYPE == kKvQ4_1 ? 2 : 1); ++z)
                    asm volatile("" : "+v"(v.sc[y][z].x), "+v"(v.sc[y][z].y), "+v"(v.sc[y][z].z), "+v"(v.sc[y][z].w));
        }
        values<!WHOLE>(v, s, vis, whole);
        load<true>(v, vp + c, pair, lane);
    }
    // The tiles that the rows see, every parts-th: those that all rows see whole with the next AHEAD tiles loaded ahead,
    // then the others. `lds`: room for the queries' pieces.
    __device__ __forceinline__ void run(const Attn4Args & a, uint32_t h, uint32_t part, uint32_t parts, h8 * lds, uint32_t wave,
                                        uint32_t lane) {
        constexpr size_t tb = kv4_tile_bytes(TYPE);
        const size_t pair = (size_t)a.n_tiles * tb;
        const uint8_t * kp = a.k + kKv4Header + (size_t)h * (D / 64) * pair, * vp = a.v + kKv4Header + (size_t)h * (D / 64) * pair;
        Span w0, w1, all;
        spans(a, w0, w1, all);
        const uint32_t n0 = w0.size(), nw = n0 + w1.size();
        auto whole = [&](uint32_t j) { return j < n0 ? w0.lo + j : w1.lo + (j - n0); };
        // two tiles ahead: tiles 0, 1 of an even count go to the registers 0, 1; of an odd count tile 0 goes to 1 and is done
        // first, so that the loop is whole pairs and its waits count the loads behind the ones they wait for
        Tl k0, v0, k1, v1;
        const uint32_t cnt = part < nw ? (nw - 1u - part) / parts + 1u : 0u, odd = AHEAD == 2 ? cnt & 1u : 0u;
        auto nth = [&](uint32_t x) { return whole(part + min(x, cnt - 1u) * parts); };   // (past the last: it again)
        if (cnt != 0u) {
            load<false>(k0, kp + nth(odd) * tb, pair, lane);
            load<true>(v0, vp + nth(odd) * tb, pair, lane);
            if constexpr (AHEAD == 2) {
                load<false>(k1, kp + nth(1u - odd) * tb, pair, lane);
                load<true>(v1, vp + nth(1u - odd) * tb, pair, lane);
            }
        }
        load_queries(a.scale, lane, lds, wave);
        __syncthreads();
        int whole_e = kFirstE;
        bool first = true;                                         // no tile has been summed
        if (odd) one<true>(a, k1, v1, nth(0u), nth(2u), kp, vp, pair, whole_e, first, lds, lane);
        for (uint32_t x = odd; x < cnt; x += AHEAD) {
            one<true>(a, k0, v0, nth(x), nth(x + AHEAD), kp, vp, pair, whole_e, first, lds, lane);
            if constexpr (AHEAD == 2) one<true>(a, k1, v1, nth(x + 1u), nth(x + 3u), kp, vp, pair, whole_e, first, lds, lane);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) e[n] = whole_e;
        // the others: the hull without w0 and w1, dealt on from the wave after the one that took the last whole tile
        const uint32_t g0 = w0.lo - all.lo, g1 = g0 + (w1.lo - w0.hi), np = all.size() - nw;
        uint32_t x = part + parts - nw % parts;
        x = x >= parts ? x - parts : x;
        auto other = [&](uint32_t y) { return y < g0 ? all.lo + y : y < g1 ? w0.hi + (y - g0) : w1.hi + (y - g1); };
        while (x < np && !any(other(x))) x += parts;
        if (x >= np) return;
        load<false>(k0, kp + other(x) * tb, pair, lane);
        load<true>(v0, vp + other(x) * tb, pair, lane);
        for (;;) {
            uint32_t nx = x + parts;
            while (nx < np && !any(other(nx))) nx += parts;
            one<false>(a, k0, v0, other(x), other(nx < np ? nx : x), kp, vp, pair, whole_e, first, lds, lane);
            if (nx >= np) break;
            x = nx;
        }
    }

    // Rows summed over their lanes; o becomes sum p v, value 32 b + 16 c + 4 g + i in o[2 b + c][i]. What leaves the wave
    // carries no power of two: waves differ in it, and the joins weigh by the maxima alone.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float unit = __builtin_ldexpf(1.0f, -k_of(e[n])), ounit = __builtin_ldexpf(1.0f, -e[n]);
            l[n] = rows_sum(l[n]) * unit;
#pragma unroll
            for (int j = 0; j < 2 * NB; ++j) o[n][j] *= ounit;
            if constexpr (TYPE == kKvQ4_1)
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    const float z = rows_sum(bias[n][k]) * unit;   // (used where column and block belong together)
#pragma unroll
                    for (int j = 2 * C * k; j < 2 * C * (k + 1); ++j) o[n][j] += z;
                }
        }
    }
};

constexpr uint32_t values_at_once(uint32_t D, uint32_t most) { return D <= most ? D : values_at_once(D / 2u, most); }

// Waves a SIMD that a kernel has registers for: the most that need no spills, but for heads of 512 over q4_1 with two columns a
// row, which keep 78 of one wave's 512 in memory (the scales and sums of 16 blocks: 60 rows behind 500 cells, 8 heads on 1, 41
// us against 30 over q4_0).
constexpr int waves_of(int D, int NT, int C, uint32_t TYPE) {
    if (D * NT == 64) return 4;
    if (NT == 1 && (D == 128 ? C == 4 || (C == 1 && TYPE == kKvQ4_0) : D == 256 && C == 1 && TYPE == kKvQ4_0)) return 3;
    return D <= 256 ? 2 : 1;
}

// Workgroup (KV head, split, group of rows), KV heads fastest: with eight of them every XCD's L2 holds one head.
template <int D, int NT, int C, uint32_t TYPE>
__global__ __launch_bounds__(256, waves_of(D, NT, C, TYPE)) void k_attn4(Attn4Args a) {
    using A = Attn4<D, NT, C, TYPE>;
    constexpr uint32_t RT = A::RW * NT;                            // rows of the workgroup
    const uint32_t h = blockIdx.x, split = blockIdx.y, rg = gridDim.z - 1u - blockIdx.z;   // causal: the long rows first
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), lane = threadIdx.x & 63u, g = lane >> 4;
    const uint32_t c = lane & (C - 1u), rl = (lane & 15u) / C;
    const uint32_t r0 = rg * RT, R = a.T * a.G, nh = a.G * a.n_head_kv;
    const size_t nr = (size_t)a.T * nh;
    // the queries' pieces, then the waves' sums, DC values of every row at a time
    constexpr uint32_t kQ = NT * A::NB * 2u * 64u * 16u, kRoom = kQ < 16384u ? 16384u : kQ;
    constexpr uint32_t DC = values_at_once(D, kRoom / (16u * RT));
    __shared__ __align__(16) uint8_t room[kRoom];
    h8 * lq = (h8 *)room;
    A w;
    w.load_runs(a, h, r0, lane);
    w.run(a, h, split * kWaves + wave, a.S * kWaves, lq, wave, lane);
    w.finish();
    // where row r's result goes: the output, or its place in the split's partial rows
    auto place = [&](uint32_t r) {
        const uint32_t t = token(a, r), hq = h * a.G + r - t * a.G;
        return a.S > 1u ? a.part + attn4_part_row(nr, D, split, (size_t)t * nh + hq)
                        : a.out + (size_t)t * a.out_stride + (size_t)hq * D;
    };
    auto sums = [&](uint32_t r, float m, float l) {
        const uint32_t t = token(a, r);
        *(float2 *)(a.part + attn4_part_sum(nr, D, a.S, split, (size_t)t * nh + h * a.G + r - t * a.G)) = make_float2(m, l);
    };
    // the waves' sums joined
    static_assert(DC % 16u == 0u && D % DC == 0u, "whole groups of 16 values");
    __shared__ float2 ml[kWaves * RT];
    float * lo = (float *)room;
#pragma unroll
    for (uint32_t z = 0; z < D / DC; ++z) {
        __syncthreads();                                       // (the queries, the values before have been read)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (z == 0u && g == 0u && c == 0u) ml[wave * RT + A::RW * n + rl] = make_float2(w.m[n], w.l[n]);
#pragma unroll
            for (uint32_t j = 0; j < DC / 16; ++j) {
                const f4 x = w.o[n][z * (DC / 16) + j];
                if (C == 1 || ((z * (DC / 16) + j) / 2u) % C == c)
                    *(float4 *)(lo + (wave * RT + A::RW * n + rl) * DC + 16 * j + 4 * g) = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < RT * (DC / 4); e += 64u * kWaves) {
            const uint32_t r = e / (DC / 4), d = 4u * (e % (DC / 4));
            if (r0 + r >= R) continue;
            float2 u[kWaves];
            float M = -__builtin_inff(), L = 0.0f;
#pragma unroll
            for (uint32_t x = 0; x < kWaves; ++x) { u[x] = ml[x * RT + r]; M = fmaxf(M, u[x].x); }
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t x = 0; x < kWaves; ++x) {
                const float f = u[x].x == M ? 1.0f : __builtin_amdgcn_exp2f(u[x].x - M);
                const float4 v = *(const float4 *)(lo + (x * RT + r) * DC + d);
                L += u[x].y * f;
                y.x += v.x * f; y.y += v.y * f; y.z += v.z * f; y.w += v.w * f;
            }
            const float il = a.S > 1u ? 1.0f : L == 0.0f ? 0.0f : 1.0f / L;
            *(float4 *)(place(r0 + r) + z * DC + d) = make_float4(y.x * il, y.y * il, y.z * il, y.w * il);
            if (a.S > 1u && z == 0u && d == 0u) sums(r0 + r, M, L);
        }
    }
}

// The splits of a row joined: a workgroup a row. 256 / (D / 4) groups of threads take splits in turn, then meet in LDS; the
// order of the additions is fixed.
template <int D>
__global__ __launch_bounds__(256) void k_attn4_join(Attn4Args a) {
    constexpr uint32_t W = D / 4, NG = 256u / W, N = 8;            // N: loads in flight
    __shared__ float4 acc[256];
    __shared__ float wt[kSplitsMax], red[8];
    const uint32_t ro = blockIdx.x, nh = a.G * a.n_head_kv, tid = threadIdx.x, c = tid % W, s0 = tid / W;
    const size_t nr = (size_t)a.T * nh;
    const float4 * po = (const float4 *)(a.part + attn4_part_row(nr, D, 0u, ro)) + c;
    float4 x[N];
    auto fetch = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            const uint32_t sp = s0 + NG * (i0 + i);
            x[i] = sp < a.S ? po[(size_t)sp * nr * W] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    };
    fetch(0u);
    static_assert(kSplitsMax == 256u, "a thread a split");
    float2 e = make_float2(-__builtin_inff(), 0.0f);
    if (tid < a.S) e = *(const float2 *)(a.part + attn4_part_sum(nr, D, a.S, tid, ro));
    float M = e.x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) M = fmaxf(M, __shfl_xor(M, d));
    if ((tid & 63u) == 0u) red[tid / 64u] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float f = e.x == M ? 1.0f : __builtin_amdgcn_exp2f(e.x - M);
    float L = e.y * f;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) L += __shfl_xor(L, d);
    if ((tid & 63u) == 0u) red[4u + tid / 64u] = L;
    wt[tid] = f;
    __syncthreads();
    L = (red[4] + red[5]) + (red[6] + red[7]);
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t i0 = 0;;) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            const uint32_t sp = s0 + NG * (i0 + i);
            const float w = sp < a.S ? wt[sp] : 0.0f;
            y.x += x[i].x * w; y.y += x[i].y * w; y.z += x[i].z * w; y.w += x[i].w * w;
        }
        i0 += N;
        if (i0 * NG >= a.S) break;
        fetch(i0);
    }
    acc[tid] = y;
    __syncthreads();
    if (s0 == 0u) {
#pragma unroll
        for (uint32_t i = 1; i < NG; ++i) {
            const float4 z = acc[i * W + c];
            y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
        }
        const float il = L == 0.0f ? 0.0f : 1.0f / L;
        *((float4 *)(a.out + (size_t)(ro / nh) * a.out_stride + (size_t)(ro % nh) * D) + c) =
            make_float4(y.x * il, y.y * il, y.z * il, y.w * il);
    }
}

template <int D, int NT, int C, uint32_t TYPE>
static int launch(const Attn4Args & a, hipStream_t s) {
    const uint32_t rows = 16u / C * NT, n_rg = (a.T * a.G + rows - 1u) / rows;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_attn4<D, NT, C, TYPE>), dim3(a.n_head_kv, a.S, n_rg), dim3(64u * kWaves), 0, s, a);
    if (a.S > 1u) hipLaunchKernelGGL(k_attn4_join<D>, dim3(a.T * a.G * a.n_head_kv), dim3(256), 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

template <int D, uint32_t TYPE>
static int launch_d(const Attn4Args & a, const Attn4Plan & p, hipStream_t s) {
    if constexpr (D <= 128)
        if (p.NT == 2u) return launch<D, 2, 1, TYPE>(a, s);
    switch (p.C) {
        case 2: return launch<D, 1, 2, TYPE>(a, s);
        case 4:
            if constexpr (D >= 128) return launch<D, 1, 4, TYPE>(a, s);
        default: return launch<D, 1, 1, TYPE>(a, s);
    }
}

template <uint32_t TYPE>
static int launch_t(const Attn4Args & a, const Attn4Plan & p, hipStream_t s) {
    switch (a.D) {
        case 64: return launch_d<64, TYPE>(a, p, s);
        case 128: return launch_d<128, TYPE>(a, p, s);
        case 256: return launch_d<256, TYPE>(a, p, s);
        case 512: return launch_d<512, TYPE>(a, p, s);
        default: return -2;
    }
}

}  // namespace tsr

int tsr_launch_attn4(const tsr::Attn4Args & a, const tsr::Attn4Plan & p, hipStream_t s) {
    return a.type == tsr::kKvQ4_0 ? tsr::launch_t<tsr::kKvQ4_0>(a, p, s) : tsr::launch_t<tsr::kKvQ4_1>(a, p, s);
}
