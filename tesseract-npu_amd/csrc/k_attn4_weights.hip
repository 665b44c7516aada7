// k_attn4_weights.hip -- the attention weight that each cell of a 4-bit K cache gets, summed over tokens and query heads:
// out[c] = decay before[c] + sum over rows of exp(s[row][c] - max[row]) / sum[row], s the scores of attn4.hpp.
//
// A row's sum has to be known before any of its weights is, and the weights of all rows are too many to keep (64 tokens of 32 heads
// behind 32768 cells: 268 MB), so that the scores are made twice, from the codes, which stay in the caches:
//   k_attn4_rowsums  every row's maximum and sum of exp2, a lane a row and a quarter of the cells, joined over lanes and waves
//   k_attn4_weights  the weights of a workgroup's rows, summed over them: a lane sums its row of each group of 16, the 16 lanes
//                    then meet; 32 sums a tile and row set go to memory
//   k_attn4_cells    the row sets' sums added up, in their order: no atomic decides a rounding
// or, for one group of rows of few heads, both at once: k_attn4_weights_one.
// A workgroup's waves have the same rows (up to four groups of 16: nothing but scores to hold) and take tiles in turn.
//
// Bound: a decode token's three launches (32 heads of 128 over 8 KV heads behind 8192 cells: 13.0 us, 5.7 + 6.8 + 2.5 by themselves, the
// codes' 9 MB in 2); for many rows the f32 operations on the scores, 4 for every product of 16 x 16 x 32 and then 4 and an exponential
// a score: 64 such tokens behind 32768 cells of q4_1 take 108 to 111 us, 61 + 60, of which the matrix instruction is busy for 14 each.
// Its time and theirs add up here. K in two f16 pieces with its scales, shared by a workgroup's waves through LDS, needs none of the
// four and three products for two: 110 us, and 121 for q4_0, which takes 98 so.
#include "attn4.hpp"
#include "long_grid.hpp"
#include "weights4_plan.hpp"

namespace tsr {

template <int D, int NT, uint32_t TYPE>
struct Weights4 : Attn4<D, NT, 1, TYPE> {
    using A = Attn4<D, NT, 1, TYPE>;
    using typename A::Tl;
    using typename A::Span;
    static constexpr bool MIN = TYPE == kKvQ4_1;
    static constexpr int NB = D / 32, NW = (NB + 3) / 4;

    // A tile's codes and scales, and q4_1's minima as an operand of the matrix instruction has them: of a group of 16 cells the lane's
    // cell lane & 15 in blocks 4 k + g. They meet the sums of the blocks' q, in two pieces, in one product for all blocks: 64 tokens
    // of 32 heads behind 32768 cells take 110 us, with a product and a sum in f32 for every block 125.
    struct Codes {
        Tl t;
        uint32_t m[2][MIN ? NW : 1];
    };
    h8 qm[NT];
    static __device__ __forceinline__ void load(Codes & k, const uint8_t * p, size_t pair, uint32_t lane) {
        const uint32_t word = 8u * (lane >> 4) + (lane & 7u), c = lane & 15u;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            const uint8_t * t = p + j * pair;
            const uint2 x = *(const uint2 *)(t + 8u * lane), y = *(const uint2 *)(t + 512u + 8u * lane);
            k.t.w[j] = make_uint4(x.x, x.y, y.x, y.y);
            k.t.d[j] = *(const uint32_t *)(t + 1024u + (MIN ? 8u : 4u) * word);
        }
        if constexpr (MIN)
#pragma unroll
            for (uint32_t u = 0; u < 2u; ++u)
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    const uint32_t b = (4u * i + (lane >> 4)) & (NB - 1u);   // (heads of 64: blocks 2 and 3 meet sums of 0)
                    k.m[u][i] = *(const uint16_t *)(p + (b >> 1) * pair + 1028u + 8u * (8u * (c >> 2) + 4u * (b & 1u) + 2u * u + ((c >> 1) & 1u)) + 2u * (c & 1u));
                }
    }
    __device__ __forceinline__ void scores(const Codes & k, const h8 * q, f4 (&s)[NT][2]) const {
        if constexpr (MIN) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t w[4] = {};
#pragma unroll
                for (int i = 0; i < NW; ++i) w[i] = k.m[u][i] * 0x10001u;
#pragma unroll
                for (int n = 0; n < NT; ++n) s[n][u] = mfma(of_words(w), qm[n], f4{ 0.0f, 0.0f, 0.0f, 0.0f });
            }
        }
        A::template scores<!MIN>(k.t, q, s);
    }
    template <bool OWN>
    __device__ __forceinline__ void load_queries(float scale, uint32_t lane, h8 * lds, uint32_t wave) {
        A::template load_queries<MIN ? 135 : 140, OWN>(scale, lane, lds, wave);   // (135: the sum of a block fits f16)
        // The unit of a row of zeros under a small scale leaves f32's range, and infinities, which the maxima start from and cells that are
        // not seen get, would meet a 0. Sums of codes stay below 2^45, whose exp2 in a unit of 2^-126 or less is 1.
#pragma unroll
        for (int n = 0; n < NT; ++n) this->csc[n] = fmaxf(this->csc[n], 0x1p-126f);
        if constexpr (MIN)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t w[4] = {};
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    float z = 0.0f;
#pragma unroll
                    for (int g = 0; g < 4 && 4 * i + g < NB; ++g) z = (lane >> 4) == (uint32_t)g ? this->qs[n][4 * i + g] : z;
                    const uint32_t hi = pair_of(z, 0.0f), lo = pair_of(z - half_of(hi, 0), 0.0f);
                    w[i] = (hi & 0xFFFFu) | (lo << 16);
                }
                qm[n] = of_words(w);
            }
    }

    // The lane's cells of tile i that its row n sees: bit 4 u + k its cell 16 u + 4 g + k.
    __device__ __forceinline__ uint32_t seen(int n, uint32_t i, uint32_t g) const {
        uint32_t v = 0u;
#pragma unroll
        for (uint32_t u = 0; u < 2u; ++u)
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) v |= this->sees(n, 32u * i + 16u * u + 4u * g + k) ? 1u << (4u * u + k) : 0u;
        return v;
    }

    // Each row's maximum and the inverse of its sum over the splits, the four lanes of a row taking them in turn.
    float top[NT], il[NT];
    __device__ __forceinline__ void load_sums(const Attn4Args & a, const Weights4Plan & p, uint32_t h, uint32_t rg, uint32_t lane) {
        const uint32_t g = lane >> 4;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float2 * pairs = (const float2 *)a.part + weights4_pair(p, a.n_head_kv, 0u, h, rg, 16u * n + (lane & 15u));
            const size_t step = weights4_pair(p, a.n_head_kv, 1u, 0u, 0u, 0u);
            float2 x[kWeightsSplits / 4];                          // (all on their way at once)
#pragma unroll
            for (uint32_t j = 0; j < kWeightsSplits / 4; ++j)
                x[j] = g + 4u * j < a.S ? pairs[(g + 4u * j) * step] : make_float2(-__builtin_inff(), 0.0f);
            float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < kWeightsSplits / 4; ++j) m = fmaxf(m, x[j].x);
#pragma unroll
            for (uint32_t j = 0; j < kWeightsSplits / 4; ++j) l += x[j].y * (x[j].x == m ? 1.0f : __builtin_amdgcn_exp2f(x[j].x - m));
            top[n] = rows_max(m);
            l = rows_sum(l * (m == top[n] ? 1.0f : __builtin_amdgcn_exp2f(m - top[n])));
            const bool empty = l == 0.0f || rg * 16u * NT + 16u * n + (lane & 15u) >= a.T * a.G;
            il[n] = empty ? 0.0f : 1.0f / l;
            top[n] = empty ? __builtin_inff() : top[n];            // (weights of 0, whatever the scores are)
        }
    }
    // The rows' weights of tile i, summed: of its cell place(lane), in the lanes without bit 3.
    static __device__ __forceinline__ uint32_t place(uint32_t lane) { return 16u * ((lane >> 2) & 1u) + 4u * (lane >> 4) + (lane & 3u); }
    __device__ __forceinline__ float sums(const Codes & k, uint32_t i, bool whole, const h8 * lds, uint32_t lane) const {
        f4 s[NT][2];
        uint32_t ql = lane;
        asm volatile("" : "+v"(ql));
        scores(k, lds + ql, s);
        float x[8] = {};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t in = whole ? 0xFFu : seen(n, i, lane >> 4);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][c >> 2][c & 3], this->csc[n], -top[n]));
                const float z = __builtin_fmaf(e, il[n], x[c]);
                x[c] = whole || ((in >> c) & 1u) ? z : x[c];
            }
        }
        // over the 16 lanes of a row of the wave: halves handed over between lanes 7 - x and x, 2 and 1 apart; then all eight
        const bool b2 = (lane & 4u) != 0u, b1 = (lane & 2u) != 0u, b0 = (lane & 1u) != 0u;
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = (b2 ? x[c + 4] : x[c]) + dpp_f<kDppRowHalfMirror>(b2 ? x[c] : x[c + 4]);
#pragma unroll
        for (int c = 0; c < 2; ++c) x[c] = (b1 ? x[c + 2] : x[c]) + dpp_f<kDppXor2>(b1 ? x[c] : x[c + 2]);
        x[0] = (b0 ? x[1] : x[0]) + dpp_f<kDppXor1>(b0 ? x[0] : x[1]);
        return x[0] + dpp_f<kDppRowMirror>(dpp_f<kDppRowHalfMirror>(x[0]));   // (lane l and l ^ 8)
    }

    // one(tile's codes, its number, whether every row sees all of it) for the wave's tiles, every parts-th; none(number) for
    // those that no row sees. `lds`: the queries' pieces go there first (OWN: the wave's own room and rows).
    template <bool OWN = false, class One, class None>
    __device__ __forceinline__ void walk(const Attn4Args & a, uint32_t h, uint32_t part, uint32_t parts, h8 * lds, uint32_t wave, uint32_t lane,
                                         One one, None none) {
        constexpr size_t tb = kv4_tile_bytes(TYPE);
        const size_t pair = (size_t)a.n_tiles * tb;
        const uint8_t * kp = a.k + kKv4Header + (size_t)h * (D / 64) * pair;
        Span w0, w1, all;
        this->spans(a, w0, w1, all);
        const uint32_t n0 = w0.size(), nw = n0 + w1.size();
        const uint32_t cnt = part < nw ? (nw - 1u - part) / parts + 1u : 0u;
        auto nth = [&](uint32_t x) {                               // (past the last: it again)
            const uint32_t j = part + min(x, cnt - 1u) * parts;
            return j < n0 ? w0.lo + j : w1.lo + (j - n0);
        };
        Codes k0, k1;
        if (cnt != 0u) {
            load(k0, kp + nth(0u) * tb, pair, lane);
            load(k1, kp + nth(1u) * tb, pair, lane);
        }
        load_queries<OWN>(a.scale, lane, lds, wave);
        __syncthreads();
        for (uint32_t x = 0; x < cnt; x += 2u) {                   // two tiles ahead
            one(k0, nth(x), true);
            load(k0, kp + nth(x + 2u) * tb, pair, lane);
            if (x + 1u < cnt) one(k1, nth(x + 1u), true);
            load(k1, kp + nth(x + 3u) * tb, pair, lane);
        }
        // the others: what is left of all tiles, dealt on from the wave after the one that took the last whole tile
        const uint32_t g0 = w0.lo, g1 = g0 + (w1.lo - w0.hi), np = (a.n_kv + 31u) / 32u - nw;
        auto other = [&](uint32_t y) { return y < g0 ? y : y < g1 ? w0.hi + (y - g0) : w1.hi + (y - g1); };
        uint32_t x = part + parts - nw % parts;
        x = x >= parts ? x - parts : x;
        for (; x < np; x += parts) {
            const uint32_t i = other(x);
            if (!this->any(i)) {
                none(i);
                continue;
            }
            load(k0, kp + i * tb, pair, lane);
            one(k0, i, false);
        }
    }
};

constexpr int weights_waves(int D, int NT) { return D * NT <= 64 ? 4 : D * NT <= 128 ? 3 : 2; }

// Workgroup (KV head, split, row set), KV heads fastest.
template <int D, int NT, uint32_t TYPE>
__global__ __launch_bounds__(256, weights_waves(D, NT)) void k_attn4_rowsums(Attn4Args a, Weights4Plan p) {
    using W = Weights4<D, NT, TYPE>;
    __shared__ __align__(16) uint8_t room[W::kQ];
    __shared__ float2 ml[kWaves][16 * NT];
    const uint32_t h = blockIdx.x, split = blockIdx.y, rg = blockIdx.z, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4;
    W w;
    w.load_runs(a, h, rg * 16u * NT, lane);
    float sub[NT] = {};                                            // the maxima in base 2 (0: none yet)
    w.walk(a, h, split * kWaves + wave, a.S * kWaves, (h8 *)room, wave, lane,
           [&](const typename W::Codes & k, uint32_t i, bool whole) {
               f4 s[NT][2];
               uint32_t ql = lane;                                 // (q's pieces: read from LDS for every tile)
               asm volatile("" : "+v"(ql));
               w.scores(k, (h8 *)room + ql, s);
               // maxima of the scores in the row's own unit, which is positive; a lane's sum is in units of its maximum's exp2
#pragma unroll
               for (int n = 0; n < NT; ++n) {
                   if (!whole) {
                       const uint32_t in = w.seen(n, i, g);
#pragma unroll
                       for (int c = 0; c < 8; ++c) s[n][c >> 2][c & 3] = (in >> c) & 1u ? s[n][c >> 2][c & 3] : -__builtin_inff();
                   }
                   float top = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])), s[n][1][0]);
                   top = fmaxf(fmaxf(fmaxf(top, s[n][1][1]), s[n][1][2]), s[n][1][3]);
                   if (__ballot(top > w.m[n])) {
                       const float m = fmaxf(w.m[n], top);
                       w.l[n] = w.m[n] == m ? w.l[n] : w.l[n] * __builtin_amdgcn_exp2f((w.m[n] - m) * w.csc[n]);
                       w.m[n] = m;
                       sub[n] = m == -__builtin_inff() ? 0.0f : m * w.csc[n];
                   }
#pragma unroll
                   for (int c = 0; c < 8; ++c) w.l[n] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][c >> 2][c & 3], w.csc[n], -sub[n]));
               }
           },
           [](uint32_t) {});
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const float m0 = w.m[n] == -__builtin_inff() ? w.m[n] : sub[n], m = rows_max(m0);
        const float l = rows_sum(w.l[n] * (m0 == m ? 1.0f : __builtin_amdgcn_exp2f(m0 - m)));
        if (g == 0u) ml[wave][16 * n + lane] = make_float2(m, l);
    }
    __syncthreads();
    const uint32_t r = threadIdx.x;
    if (r < 16u * NT) {
        float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
        for (uint32_t v = 0; v < kWaves; ++v) m = fmaxf(m, ml[v][r].x);
#pragma unroll
        for (uint32_t v = 0; v < kWaves; ++v) l += ml[v][r].y * (ml[v][r].x == m ? 1.0f : __builtin_amdgcn_exp2f(ml[v][r].x - m));
        ((float2 *)a.part)[weights4_pair(p, a.n_head_kv, split, h, rg, r)] = make_float2(m, l);
    }
}

template <int D, int NT, uint32_t TYPE>
__global__ __launch_bounds__(256, weights_waves(D, NT)) void k_attn4_weights(Attn4Args a, Weights4Plan p) {
    using W = Weights4<D, NT, TYPE>;
    __shared__ __align__(16) uint8_t room[W::kQ];
    const uint32_t h = blockIdx.x, split = blockIdx.y, rg = blockIdx.z, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const uint32_t lane = threadIdx.x & 63u;
    W w;
    w.load_runs(a, h, rg * 16u * NT, lane);
    w.load_sums(a, p, h, rg, lane);
    float * sums = (float *)((uint8_t *)a.part + p.sums) + ((size_t)h * p.n_rg + rg) * p.n_pad;
    w.walk(a, h, split * kWaves + wave, a.S * kWaves, (h8 *)room, wave, lane,
           [&](const typename W::Codes & k, uint32_t i, bool whole) {
               const float x = w.sums(k, i, whole, (h8 *)room, lane);
               if ((lane & 8u) == 0u) sums[32u * i + W::place(lane)] = x;
           },
           [&](uint32_t i) {
               if (lane < 32u) sums[32u * i + lane] = 0.0f;
           });
}

// The last two passes in one for rows that are one group of 16 (a decode token's) of few KV heads and cells (weights4_plan.hpp): a wave a KV
// head, the waves' sums of a tile meet in LDS and are results.
template <int D, uint32_t TYPE>
__global__ __launch_bounds__(65536 / D) void k_attn4_weights_one(Attn4Args a, Weights4Plan p, const float * before, float decay) {
    using W = Weights4<D, 1, TYPE>;
    __shared__ __align__(16) uint8_t room[1024 / D][W::kQ];
    __shared__ float part[2][1024 / D][32];
    const uint32_t h = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), lane = threadIdx.x & 63u;
    W w;
    w.load_runs(a, h, 0u, lane);
    w.load_sums(a, p, h, 0u, lane);
    uint32_t buf = 0u;
    auto out = [&](uint32_t i, bool any) {
        const uint32_t c = 32u * i + lane;
        if (h != 0u || lane >= 32u || c >= a.n_kv) return;
        float x = 0.0f;
        if (any)
            for (uint32_t v = 0; v < a.n_head_kv; ++v) x += part[buf][v][lane];
        a.out[c] = before == nullptr ? x : __builtin_fmaf(decay, before[c], x);
    };
    w.template walk<true>(a, h, blockIdx.x, gridDim.x, (h8 *)room[h], 0u, lane,
           [&](const typename W::Codes & k, uint32_t i, bool whole) {
               const float x = w.sums(k, i, whole, (h8 *)room[h], lane);
               if ((lane & 8u) == 0u) part[buf][h][W::place(lane)] = x;
               lds_barrier();                                      // (the waves see the same cells: they come here as often)
               out(i, true);
               buf ^= 1u;
           },
           [&](uint32_t i) { out(i, false); });
}

// Cells' sums over n row sets: 64 cells a workgroup, its four waves every fourth row set, joined in their order.
__global__ __launch_bounds__(256) void k_attn4_cells(const float * sums, uint32_t n, uint32_t n_pad, uint32_t n_kv, const float * before, float decay,
                                                     float * out) {
    __shared__ float part[4][64];
    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x & 63u, c = long_block() * 64u + lane;
    float x = 0.0f;
    if (c < n_kv)
        for (uint32_t i = wave; i < n; i += 32u) {                 // (eight on their way at once)
            float v[8];
#pragma unroll
            for (uint32_t j = 0; j < 8u; ++j) v[j] = i + 4u * j < n ? sums[(size_t)(i + 4u * j) * n_pad + c] : 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < 8u; ++j) x += v[j];
        }
    part[wave][lane] = x;
    __syncthreads();
    if (wave == 0u && c < n_kv) {
        x = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
        out[c] = before == nullptr ? x : __builtin_fmaf(decay, before[c], x);
    }
}

template <int D, int NT, uint32_t TYPE>
static int launch_weights(const Attn4Args & a, const Weights4Plan & p, const float * before, float decay, hipStream_t s) {
    const dim3 grid(a.n_head_kv, a.S, (a.T * a.G + 16u * NT - 1u) / (16u * NT)), wg(64u * kWaves);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_attn4_rowsums<D, NT, TYPE>), grid, wg, 0, s, a, p);
    if constexpr (NT == 1 && D <= 256)
        if (p.one != 0u) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_attn4_weights_one<D, TYPE>), dim3(p.one), dim3(64u * a.n_head_kv), 0, s, a, p, before, decay);
            return hipGetLastError() == hipSuccess ? 0 : -4;
        }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_attn4_weights<D, NT, TYPE>), grid, wg, 0, s, a, p);
    const uint32_t n = a.n_head_kv * p.n_rg;
    hipLaunchKernelGGL(k_attn4_cells, long_grid(((uint64_t)a.n_kv + 63u) / 64u), dim3(256), 0, s, (const float *)((uint8_t *)a.part + p.sums), n, p.n_pad, a.n_kv, before,
                       decay, a.out);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

template <uint32_t TYPE>
static int launch_weights_t(const Attn4Args & a, const Weights4Plan & p, const float * before, float decay, hipStream_t s) {
    switch (a.D * 8u + p.NT) {
        case 64 * 8 + 1: return launch_weights<64, 1, TYPE>(a, p, before, decay, s);
        case 64 * 8 + 2: return launch_weights<64, 2, TYPE>(a, p, before, decay, s);
        case 64 * 8 + 4: return launch_weights<64, 4, TYPE>(a, p, before, decay, s);
        case 128 * 8 + 1: return launch_weights<128, 1, TYPE>(a, p, before, decay, s);
        case 128 * 8 + 2: return launch_weights<128, 2, TYPE>(a, p, before, decay, s);
        case 128 * 8 + 4: return launch_weights<128, 4, TYPE>(a, p, before, decay, s);
        case 256 * 8 + 1: return launch_weights<256, 1, TYPE>(a, p, before, decay, s);
        case 512 * 8 + 1: return launch_weights<512, 1, TYPE>(a, p, before, decay, s);
        default: return -2;
    }
}

}  // namespace tsr

int tsr_launch_attn4_weights(const tsr::Attn4Args & a, const tsr::Weights4Plan & p, const float * before, float decay, hipStream_t s) {
    if (a.n_kv == 0u) return 0;
    return a.type == tsr::kKvQ4_0 ? tsr::launch_weights_t<tsr::kKvQ4_0>(a, p, before, decay, s) : tsr::launch_weights_t<tsr::kKvQ4_1>(a, p, before, decay, s);
}
