// k_kv4_select.hip -- for every token and KV head the blocks of cells whose bounds (k_kv4_bounds.hip) allow the largest
// scores.
//
// The score of a block is max over the KV head's query heads of sum over channels of max(q lo, q hi) = max(q, 0) hi + min(q, 0) lo.
// It decides between blocks that may lie close together, so that it is f64: products of f32 and bf16 are exact there
// and a sum of 512 is off by 2^-52 of its terms, far below what tells two blocks apart. Equal scores go to the lowest block.
//
// k_kv4_scores is a matrix product of bounds and queries on the f64 matrix instruction 16x16x4 (the rate of f64's vector units,
// without their registers): rows 16 blocks, columns 16 query heads (whole tokens), each channel once with hi and
// once with lo. What leaves is a key a block, an unsigned number in the order of the scores. k_kv4_pick_blocks then finds the
// cut: the keys' range is counted into 1024 bins, the bin with the cut becomes the range, until all of a bin is taken or it
// is one value; two passes do for a few thousand keys.
#include "kernels.hpp"
#include "tsr_dev.hpp"
#include "wave_lds.hpp"

namespace tsr {

typedef double d4 __attribute__((ext_vector_type(4)));

// The order of f64 as unsigned numbers; a NaN is the lowest.
__device__ __forceinline__ uint64_t order_of(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return x != x ? 0u : u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}

constexpr uint32_t kScoreWaves = 4u;

// The blocks that cells [lo, hi) touch.
struct BlockRange { uint32_t lo, hi; };
__device__ __forceinline__ BlockRange blocks_of(uint32_t lo, uint32_t hi, uint32_t n_kv, uint32_t block) {
    hi = min(hi, n_kv);
    return lo < hi ? BlockRange{ lo / block, (hi + block - 1u) / block } : BlockRange{ 0u, 0u };
}

// Workgroup (64 blocks, KV heads fastest; tokens), a wave 16 blocks. C columns hold 16 / G tokens' G query heads, or a token's 16 at
// a time where G > 16.
template <int D>
__global__ __launch_bounds__(64 * kScoreWaves) void k_kv4_scores(Kv4SelectArgs a) {
    __shared__ double room[kScoreWaves][16 * 17];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
    const uint32_t h = blockIdx.x % a.n_head_kv, b0 = (blockIdx.x / a.n_head_kv * kScoreWaves + wave) * 16u;
    const uint32_t tpt = a.G <= 16u ? 16u / a.G : 1u, t0 = blockIdx.y * tpt;
    if (b0 >= a.n_blocks) return;
    if (a.runs != nullptr) {                                       // a tile that no token's runs touch
        bool any = false;
        if (lane < tpt && t0 + lane < a.T) {
            const uint4 u = *(const uint4 *)(a.runs + 4u * (size_t)(t0 + lane));
            const BlockRange x = blocks_of(u.x, u.y, a.n_kv, a.block), y = blocks_of(u.z, u.w, a.n_kv, a.block);
            any = (x.lo < b0 + 16u && x.hi > b0) || (y.lo < b0 + 16u && y.hi > b0);
        }
        if (__ballot(any) == 0ull) return;
    }
    // the bounds: of block b0 + r the channels 16 m + 4 g .. + 3
    const uint32_t * bp = a.bounds + ((size_t)h * a.stride + min(b0 + r, a.n_blocks - 1u)) * D + 4u * g;
    constexpr int AT = D / 16 <= 8 ? D / 16 : 8;                   // loads of 16 channels in flight
    double * mine = room[wave];
    const uint32_t items = tpt * 16u;
    double best[4];                                                // of the items that the lane stores
#pragma unroll
    for (int i = 0; i < 4; ++i) best[i] = -__builtin_inf();
    bool nan[4] = {};
    for (uint32_t c0 = 0u; c0 < a.G; c0 += 16u) {                  // (one round where G <= 16)
        const uint32_t tt = a.G <= 16u ? r / a.G : 0u, gq = a.G <= 16u ? r - tt * a.G : c0 + r;
        const bool real = tt < tpt && t0 + tt < a.T && gq < a.G;
        const float * qp = a.q + (size_t)min(t0 + tt, a.T - 1u) * a.q_stride + ((size_t)h * a.G + min(gq, a.G - 1u)) * D + 4u * g;
        d4 acc = { 0.0, 0.0, 0.0, 0.0 };
#pragma unroll 1
        for (int m0 = 0; m0 < D / 16; m0 += AT) {
            uint4 w[AT];
            float4 q[AT];
#pragma unroll
            for (int m = 0; m < AT; ++m) {
                w[m] = *(const uint4 *)(bp + 16 * (m0 + m));
                q[m] = *(const float4 *)(qp + 16 * (m0 + m));
            }
#pragma unroll
            for (int m = 0; m < AT; ++m) {
                const uint32_t x[4] = { w[m].x, w[m].y, w[m].z, w[m].w };
                const float y[4] = { q[m].x, q[m].y, q[m].z, q[m].w };
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float up = y[i] < 0.0f ? 0.0f : y[i], down = y[i] > 0.0f ? 0.0f : y[i];   // (a NaN stays one)
                    acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)bf(x[i] & 0xFFFF0000u), (double)up, acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)bf(x[i] << 16), (double)down, acc, 0, 0, 0);
                }
            }
        }
        // lane (column r, row group g) holds the rows 4 i + g; the most of a token's columns
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[r * 17u + 4u * i + g] = real ? acc[i] : -__builtin_inf();
        own_room();
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            const uint32_t e = lane + 64u * k, b = e & 15u, first = (e >> 4) * (a.G <= 16u ? a.G : 0u);
            if (e < items)
                for (uint32_t j = 0; j < min(a.G, 16u); ++j) {
                    const double s = mine[(first + j) * 17u + b];
                    nan[k] |= s != s;
                    best[k] = fmax(best[k], s);
                }
        }
        own_room();
    }
#pragma unroll
    for (uint32_t k = 0; k < 4u; ++k) {
        const uint32_t e = lane + 64u * k, b = b0 + (e & 15u), t = t0 + (e >> 4);
        if (e < items && t < a.T && b < a.n_blocks)
            a.keys[((size_t)t * a.n_head_kv + h) * a.n_blocks + b] = nan[k] ? 0u : order_of(best[k]);
    }
}

__device__ __forceinline__ uint64_t lesser(uint64_t a, uint64_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a < b ? b : a; }

constexpr uint32_t kPickWaves = 4u, kBins = 1024u;

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t x, int d) {
    return (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)x, d) | (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)(x >> 32), d) << 32;
}

// Workgroup (KV head, token). The keys of the candidates between the first and the last ones lie in the waves' registers, wave
// w the w-th quarter, rows of 64; where they are more than ROWS rows a wave, they are read from memory whenever they are needed.
template <uint32_t ROWS>
__global__ __launch_bounds__(64 * kPickWaves) void k_kv4_pick_blocks(Kv4SelectArgs a) {
    __shared__ uint32_t bins[kBins], part[kPickWaves][2], found[3];
    __shared__ uint64_t ends[kPickWaves][2];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), lane = threadIdx.x & 63u;
    const uint32_t h = blockIdx.x, t = blockIdx.y;
    BlockRange x = { 0u, (a.n_kv + a.block - 1u) / a.block }, y = { 0u, 0u };
    if (a.runs != nullptr) {
        const uint4 u = *(const uint4 *)(a.runs + 4u * (size_t)t);
        x = blocks_of(u.x, u.y, a.n_kv, a.block);
        y = blocks_of(u.z, u.w, a.n_kv, a.block);
        if (y.lo < y.hi && (y.lo < x.lo || x.lo >= x.hi)) { const BlockRange z = x; x = y; y = z; }
        y.lo = max(y.lo, x.hi);
        if (y.lo > y.hi) y.hi = y.lo;
    }
    const uint32_t nx = x.hi - x.lo, n = nx + (y.hi - y.lo);
    auto block = [&](uint32_t i) { return i < nx ? x.lo + i : y.lo + (i - nx); };
    int32_t * out = a.blocks + ((size_t)t * a.n_head_kv + h) * a.n_sel;
    const uint32_t nf = min(a.n_first, n), take = min(n, a.n_sel);
    for (uint32_t i = threadIdx.x; i < a.n_sel; i += 64u * kPickWaves) {
        if (n <= a.n_sel) out[i] = i < n ? (int32_t)block(i) : -1;
        else if (i < nf) out[i] = (int32_t)block(i);
        else if (i >= a.n_sel - a.n_last) out[i] = (int32_t)block(n - (a.n_sel - i));
    }
    uint32_t m = take - nf - a.n_last;                             // wanted of the others
    if (n <= a.n_sel || m == 0u) return;
    const uint32_t others = n - nf - a.n_last, rows = (others + 64u * kPickWaves - 1u) / (64u * kPickWaves), first = wave * rows * 64u;
    const uint64_t * keys = a.keys + ((size_t)t * a.n_head_kv + h) * a.n_blocks;
    auto fetch = [&](uint32_t j) {
        const uint32_t i = first + 64u * j + lane;
        return i < others ? keys[block(nf + i)] : 0u;
    };
    uint64_t mine[ROWS == 0u ? 1u : ROWS];
    if constexpr (ROWS != 0u)
#pragma unroll
        for (uint32_t j = 0; j < ROWS; ++j) mine[j] = j < rows ? fetch(j) : 0u;
    // f(place, key, whether there is one) for every row of the wave, the lanes together
    auto each = [&](auto f) {
        if constexpr (ROWS != 0u) {
#pragma unroll
            for (uint32_t j = 0; j < ROWS; ++j)
                if (j < rows) f(first + 64u * j + lane, mine[j], first + 64u * j + lane < others);
        } else {
            for (uint32_t j = 0; j < rows; ++j) f(first + 64u * j + lane, fetch(j), first + 64u * j + lane < others);
        }
    };
    uint64_t lo = ~0ull, hi = 0u;
    each([&](uint32_t, uint64_t k, bool real) {
        lo = real ? lesser(lo, k) : lo;
        hi = real ? larger(hi, k) : hi;
    });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        lo = lesser(lo, shfl_xor64(lo, d));
        hi = larger(hi, shfl_xor64(hi, d));
    }
    if (lane == 0u) { ends[wave][0] = lo; ends[wave][1] = hi; }
    __syncthreads();
#pragma unroll
    for (uint32_t v = 0; v < kPickWaves; ++v) { lo = lesser(lo, ends[v][0]); hi = larger(hi, ends[v][1]); }
    // keys above hi are taken, those below lo are not, m of those between are
    bool whole = others == m;
    while (!whole && lo != hi) {
        const uint32_t bits = 64u - (uint32_t)__builtin_clzll(hi - lo), shift = bits > 10u ? bits - 10u : 0u;
        for (uint32_t i = threadIdx.x; i < kBins; i += 64u * kPickWaves) bins[i] = 0u;
        __syncthreads();
        each([&](uint32_t, uint64_t k, bool real) {
            if (real && k >= lo && k <= hi) atomicAdd(&bins[(uint32_t)((k - lo) >> shift)], 1u);
        });
        __syncthreads();
        // thread i has four bins from the top down: how many keys lie above them, and where m is passed
        uint32_t c[4], sum = 0u;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) { c[i] = bins[kBins - 1u - (4u * threadIdx.x + i)]; sum += c[i]; }
        uint32_t above = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t v = (uint32_t)__shfl_up((int)above, d);
            above += lane >= (uint32_t)d ? v : 0u;
        }
        if (lane == 63u) part[wave][0] = above;
        __syncthreads();
        above -= sum;
#pragma unroll
        for (uint32_t v = 0; v < kPickWaves; ++v) above += v < wave ? part[v][0] : 0u;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            if (above < m && above + c[i] >= m) { found[0] = kBins - 1u - (4u * threadIdx.x + i); found[1] = above; found[2] = c[i]; }
            above += c[i];
        }
        __syncthreads();
        lo += (uint64_t)found[0] << shift;
        hi = lesser(hi, lo + (((uint64_t)1 << shift) - 1u));
        m -= found[1];
        whole = found[2] == m;
    }
    // the cut: keys above hi, and of those from lo to hi all or, equal ones, the first m
    uint32_t n_above = 0u, n_in = 0u;
    each([&](uint32_t, uint64_t k, bool real) {
        n_above += (uint32_t)__popcll(__ballot(real && k > hi));
        n_in += (uint32_t)__popcll(__ballot(real && k >= lo && k <= hi));
    });
    if (lane == 0u) { part[wave][0] = n_above; part[wave][1] = n_in; }
    __syncthreads();
    uint32_t at = 0u, in = 0u;
#pragma unroll
    for (uint32_t v = 0; v < kPickWaves; ++v) {
        at += v < wave ? part[v][0] : 0u;
        in += v < wave ? part[v][1] : 0u;
    }
    at += nf + min(in, m);
    const uint64_t below = (1ull << lane) - 1u;
    each([&](uint32_t i, uint64_t k, bool real) {
        const bool mid = real && k >= lo && k <= hi;
        const uint64_t mids = __ballot(mid);
        const bool sel = (real && k > hi) || (mid && in + (uint32_t)__popcll(mids & below) < m);
        const uint64_t sels = __ballot(sel);
        if (sel) out[at + (uint32_t)__popcll(sels & below)] = (int32_t)block(nf + i);
        at += (uint32_t)__popcll(sels);
        in += (uint32_t)__popcll(mids);
    });
}

template <int D>
static void launch_scores(const Kv4SelectArgs & a, hipStream_t s) {
    const uint32_t tpt = a.G <= 16u ? 16u / a.G : 1u;
    hipLaunchKernelGGL(k_kv4_scores<D>, dim3(a.n_head_kv * ((a.n_blocks + 16u * kScoreWaves - 1u) / (16u * kScoreWaves)), (a.T + tpt - 1u) / tpt),
                       dim3(64u * kScoreWaves), 0, s, a);
}

}  // namespace tsr

int tsr_launch_kv4_select(const tsr::Kv4SelectArgs & a, hipStream_t s) {
    if (a.n_blocks > a.n_sel && a.n_sel > a.n_first + a.n_last) {   // (else no score decides)
        switch (a.D) {
            case 64: tsr::launch_scores<64>(a, s); break;
            case 128: tsr::launch_scores<128>(a, s); break;
            case 256: tsr::launch_scores<256>(a, s); break;
            case 512: tsr::launch_scores<512>(a, s); break;
            default: return -2;
        }
    }
    const dim3 grid(a.n_head_kv, a.T), wg(64u * tsr::kPickWaves);
    const uint32_t rows = (a.n_blocks + 64u * tsr::kPickWaves - 1u) / (64u * tsr::kPickWaves);
    if (rows <= 2u) hipLaunchKernelGGL(tsr::k_kv4_pick_blocks<2>, grid, wg, 0, s, a);
    else if (rows <= 16u) hipLaunchKernelGGL(tsr::k_kv4_pick_blocks<16>, grid, wg, 0, s, a);
    else hipLaunchKernelGGL(tsr::k_kv4_pick_blocks<0>, grid, wg, 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
