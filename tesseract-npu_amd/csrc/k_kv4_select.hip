// k_kv4_select.hip -- for every token and KV head the blocks of cells whose bounds (k_kv4_bounds.hip) allow the largest
// scores.
//
// The score of a block is max over the KV head's query heads of sum over channels of max(q lo, q hi).
// It decides between blocks that may lie close together, so that it is f64, made as max(q, 0) hi + min(q, 0) lo: products are
// exact, sums off by 2^-53 of their terms, far below what tells two blocks apart, and the bound that q does not meet adds 0, so
// that blocks whose scores are equal by the formula are so here. Equal scores go to the lowest block.
//
// k_kv4_scores is a product of bounds and queries on the f64 matrix instruction 4x4x4 (four of them at once: 16 blocks by
// four query heads, each channel once with hi and once with lo), 18 cycles an instruction; k_kv4_scores_many on 16x16x4, 64 cycles,
// whose 16 columns several tokens fill that look at the same blocks. What leaves is a key a block, an unsigned number in
// the order of the scores. k_kv4_pick_blocks then finds the cut (pick.hpp). Both are a few microseconds of waiting for memory
// and for each other's steps, not work: reductions and scans run on DPP, keys are asked for before the runs that say which
// of them count. A token of 32 heads of 128 over 8 KV heads, 2048 blocks: scores 4.8 us, cut 6.9 (an empty kernel 1.7); 33 sequences' tokens
// of 8 heads of 256 over 4, 94 blocks: 10.1 and 6.4. 512 tokens of 32 heads of 128 behind 120 blocks take 27.0 for the scores, bound by
// the matrix instruction (13.7 at what an 8192^3 product reaches, 66 TFLOP/s); with 4x4x4 they took 51 to 54.
#include "kernels.hpp"
#include "long_grid.hpp"
#include "pick.hpp"

namespace tsr {

typedef double d4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kScoreWaves = 4u;

// The blocks that cells [lo, hi) touch.
struct BlockRange {
    uint32_t lo, hi;
    __device__ __forceinline__ bool has(uint32_t b) const { return b >= lo && b < hi; }
    __device__ __forceinline__ bool meets(uint32_t b0, uint32_t b1) const { return lo < b1 && hi > b0 && lo < hi; }
};
__device__ __forceinline__ BlockRange blocks_of(uint32_t lo, uint32_t hi, uint32_t n_kv, uint32_t block) {
    hi = min(hi, n_kv);
    return lo < hi ? BlockRange{ lo / block, (hi + block - 1u) / block } : BlockRange{ 0u, 0u };
}

// The bounds of a word.
struct Bounds2 { double hi, lo; };
__device__ __forceinline__ Bounds2 bounds2(uint32_t w) { return Bounds2{ (double)bf(w & 0xFFFF0000u), (double)bf(w << 16) }; }
// The parts of q that meet hi and lo, by its sign.
struct Query2 { double up, down; };
__device__ __forceinline__ Query2 query2(float q) {
    const uint32_t u = fb(q), m = (uint32_t)((int32_t)u >> 31);
    return Query2{ (double)bf(u & ~m), (double)bf(u & m) };
}

// Few tokens: workgroup (KV heads fastest, part of the blocks; token), a wave 16 blocks at a time and the token's query heads, NG
// groups of four at a time. Lane 16 k + 4 u + i of the instruction's operands: block 4 u + i (query head i), channels 4 k .. 4
// k + 3 of every 16, one a step; of its result: block 4 u + k, query head i. One token: a part is 64 blocks, whose bounds are asked
// for ahead of the runs. Several may be sequences of their own, which look at a few of the blocks: the parts share a token's out.
template <int D, int NG>
__global__ __launch_bounds__(64 * kScoreWaves) void k_kv4_scores(Kv4SelectArgs a, uint32_t parts) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), lane = threadIdx.x & 63u, g = lane >> 4;
    const uint32_t h = blockIdx.x % a.n_head_kv, t = blockIdx.y;
    constexpr int most = 16 / NG, AT = D / 16 < most ? D / 16 : most;   // loads of 16 channels in flight
    const uint32_t * hp = a.bounds + (size_t)h * a.stride * D + 4u * g;
    uint32_t b0 = (blockIdx.x / a.n_head_kv * kScoreWaves + wave) * 16u, end = a.n_blocks;
    auto row = [&](uint32_t b) { return hp + (size_t)min(b + (lane & 15u), a.n_blocks - 1u) * D; };
    uint4 w[AT];
    if (a.T == 1u)
#pragma unroll
        for (int m = 0; m < AT; ++m) w[m] = *(const uint4 *)(row(b0) + 16 * m);
    BlockRange x = { 0u, end }, y = { 0u, 0u };
    if (a.runs != nullptr) {
        const uint4 u = *(const uint4 *)(a.runs + 4u * (size_t)t);
        x = blocks_of(u.x, u.y, a.n_kv, a.block);
        y = blocks_of(u.z, u.w, a.n_kv, a.block);
        const uint32_t lo = min(x.lo < x.hi ? x.lo : end, y.lo < y.hi ? y.lo : end);
        end = max(x.lo < x.hi ? x.hi : 0u, y.lo < y.hi ? y.hi : 0u);
        if (a.T != 1u) b0 += lo & ~15u;
    }
    bool here = a.T == 1u;                                         // w holds this tile's first bounds
    for (; b0 < end; b0 += parts * kScoreWaves * 16u) {
        if (!x.meets(b0, b0 + 16u) && !y.meets(b0, b0 + 16u)) {
            here = false;
            continue;
        }
        const uint32_t * bp = row(b0);
        double best = -__builtin_inf();                                // over the lane's query heads
        bool nan = false;
        for (uint32_t q0 = 0; q0 < a.G; q0 += 4u * NG) {
            const float * qp[NG];
#pragma unroll
            for (int n = 0; n < NG; ++n)                               // (past the last: it again)
                qp[n] = a.q + (size_t)t * a.q_stride + ((size_t)h * a.G + min(q0 + 4u * n + (lane & 3u), a.G - 1u)) * D + 4u * g;
            double acc[NG][2];
#pragma unroll
            for (int n = 0; n < NG; ++n) acc[n][0] = acc[n][1] = 0.0;
#pragma unroll 1
            for (int m0 = 0; m0 < D / 16; m0 += AT) {
                if (!here || m0 != 0 || (D / 16 > AT && q0 != 0u))
#pragma unroll
                    for (int m = 0; m < AT; ++m) w[m] = *(const uint4 *)(bp + 16 * (m0 + m));
                float4 q[NG][AT];
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int m = 0; m < AT; ++m) q[n][m] = *(const float4 *)(qp[n] + 16 * (m0 + m));
#pragma unroll
                for (int m = 0; m < AT; ++m) {
                    const uint32_t x[4] = { w[m].x, w[m].y, w[m].z, w[m].w };
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const Bounds2 z = bounds2(x[i]);
#pragma unroll
                        for (int n = 0; n < NG; ++n) {
                            const float y[4] = { q[n][m].x, q[n][m].y, q[n][m].z, q[n][m].w };
                            const Query2 v = query2(y[i]);
                            acc[n][0] = __builtin_amdgcn_mfma_f64_4x4x4f64(z.hi, v.up, acc[n][0], 0, 0, 0);
                            acc[n][1] = __builtin_amdgcn_mfma_f64_4x4x4f64(z.lo, v.down, acc[n][1], 0, 0, 0);
                        }
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                const double s = acc[n][0] + acc[n][1];
                nan |= s != s;
                best = fmax(best, s);
            }
        }
        // the most over the four lanes of a block
        auto xor_of = [](double v, auto f) {
            const uint64_t u = __builtin_bit_cast(uint64_t, v);
            return __builtin_bit_cast(double, (uint64_t)(uint32_t)f((int)(uint32_t)u) | (uint64_t)(uint32_t)f((int)(uint32_t)(u >> 32)) << 32);
        };
        best = fmax(best, xor_of(best, [](int v) { return dpp_i<kDppXor1>(v); }));
        best = fmax(best, xor_of(best, [](int v) { return dpp_i<kDppXor2>(v); }));
        const bool none = ((__ballot(nan) >> (lane & 60u)) & 15u) != 0u;
        const uint32_t b = b0 + (lane & 12u) + g;
        if ((lane & 3u) == 0u && b < a.n_blocks)
            a.keys[((size_t)t * a.n_head_kv + h) * a.n_blocks + b] = none ? kNan64 : order_of(best);
        here = false;
    }
}

// Many tokens: workgroup (64 blocks, KV heads fastest; tokens), a wave 16 blocks. The instruction's 16 columns hold 16 / G tokens' G query heads, or a token's 16 at
// a time where G > 16.
template <int D>
__global__ __launch_bounds__(64 * kScoreWaves) void k_kv4_scores_many(Kv4SelectArgs a) {
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
            any = x.meets(b0, b0 + 16u) || y.meets(b0, b0 + 16u);
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
                    const Bounds2 z = bounds2(x[i]);
                    const Query2 v = query2(y[i]);
                    acc = __builtin_amdgcn_mfma_f64_16x16x4f64(z.hi, v.up, acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f64_16x16x4f64(z.lo, v.down, acc, 0, 0, 0);
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
            a.keys[((size_t)t * a.n_head_kv + h) * a.n_blocks + b] = nan[k] ? kNan64 : order_of(best[k]);
    }
}

constexpr uint32_t pick_waves(uint32_t WAVES) { return WAVES == 1u ? 4u : WAVES; }   // of a workgroup

// WAVES 16: a workgroup a token and KV head; WAVES 1: each of its four waves. The keys lie in the waves' registers, wave w of a
// list the w-th part of the blocks, rows of 64; where they are more than ROWS rows (ROWS 0), they are read from memory whenever they
// are needed.
template <uint32_t ROWS, uint32_t WAVES>
__global__ __launch_bounds__(64 * pick_waves(WAVES)) void k_kv4_pick_blocks(Kv4SelectArgs a) {
    constexpr uint32_t LISTS = pick_waves(WAVES) / WAVES;
    __shared__ __align__(16) PickRoom<WAVES> room[LISTS];
    const uint32_t wv = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), lane = threadIdx.x & 63u;
    const uint32_t list = WAVES == 1u ? wv : 0u, wave = WAVES == 1u ? 0u : wv, tid = 64u * wave + lane;
    const uint32_t id = blockIdx.x * LISTS + list;                 // token and KV head
    if (id >= a.T * a.n_head_kv) return;
    const uint32_t t = id / a.n_head_kv;
    const uint64_t * keys = a.keys + (size_t)id * a.n_blocks;
    uint32_t from = 0u, rows = (a.n_blocks + 64u * WAVES - 1u) / (64u * WAVES);
    uint64_t mine[ROWS == 0u ? 1u : ROWS];
    if constexpr (ROWS != 0u)
#pragma unroll
        for (uint32_t j = 0; j < ROWS; ++j) {
            const uint32_t b = (wave * rows + j) * 64u + lane;
            mine[j] = j < rows && b < a.n_blocks ? keys[b] : 0u;
        }
    BlockRange x = { 0u, a.n_blocks }, y = { 0u, 0u };
    if (a.runs != nullptr) {
        const uint4 u = *(const uint4 *)(a.runs + 4u * (size_t)t);
        x = blocks_of(u.x, u.y, a.n_kv, a.block);
        y = blocks_of(u.z, u.w, a.n_kv, a.block);
        if (y.lo < y.hi && (y.lo < x.lo || x.lo >= x.hi)) { const BlockRange z = x; x = y; y = z; }
        y.lo = max(y.lo, x.hi);
        if (y.lo > y.hi) y.hi = y.lo;
    }
    if constexpr (ROWS == 0u) {                                    // the candidates' hull
        from = x.lo;
        rows = (max(x.hi, y.lo < y.hi ? y.hi : 0u) - from + 64u * WAVES - 1u) / (64u * WAVES);
    }
    const uint32_t nx = x.hi - x.lo, n = nx + (y.hi - y.lo);
    auto block = [&](uint32_t i) { return i < nx ? x.lo + i : y.lo + (i - nx); };
    int32_t * out = a.blocks + (size_t)id * a.n_sel;
    const uint32_t nf = min(a.n_first, n);
    for (uint32_t i = tid; i < a.n_sel; i += 64u * WAVES) {
        if (n <= a.n_sel) out[i] = i < n ? (int32_t)block(i) : -1;
        else if (i < nf) out[i] = (int32_t)block(i);
        else if (i >= a.n_sel - a.n_last) out[i] = (int32_t)block(n - (a.n_sel - i));
    }
    if (n <= a.n_sel || a.n_sel == nf + a.n_last) return;
    // f(block, key) for every row of the wave, the lanes together; key 0: not one of them
    auto each = [&](auto f) {
        auto one = [&](uint32_t j, uint64_t k) {
            const uint32_t b = from + (wave * rows + j) * 64u + lane;
            const uint32_t i = x.has(b) ? b - x.lo : y.has(b) ? nx + (b - y.lo) : ~0u;
            f(b, i >= nf && i < n - a.n_last ? k : 0u);
        };
        if constexpr (ROWS != 0u) {
#pragma unroll
            for (uint32_t j = 0; j < ROWS; ++j)
                if (j < rows) one(j, mine[j]);
        } else {
            for (uint32_t j = 0; j < rows; ++j) one(j, keys[min(from + (wave * rows + j) * 64u + lane, a.n_blocks - 1u)]);
        }
    };
    Pick<WAVES>{ room[list], wave, lane }.template run<uint64_t>(a.n_sel - nf - a.n_last, each, [&](uint32_t at, uint32_t b, uint64_t) { out[nf + at] = (int32_t)b; });
}

template <int D>
static void launch_scores(const Kv4SelectArgs & a, hipStream_t s) {
    const uint32_t all = (a.n_blocks + 16u * kScoreWaves - 1u) / (16u * kScoreWaves), tpt = a.G <= 16u ? 16u / a.G : 1u;
    const uint32_t lists = a.T * a.n_head_kv, parts = min(all, a.T == 1u ? kAxisGroups / a.n_head_kv : max(1u, 1024u / lists));
    const dim3 grid(a.n_head_kv * parts, a.T), wg(64u * kScoreWaves);
    // The host does not know whether tokens share their blocks. Scores and cut in us, 4x4x4 / 16x16x4, tokens of one sequence; of
    // sequences side by side: 32 heads of 128 over 8, 1024 blocks: 32 tokens 38.1 / 19.6; 11.4 / 11.2, 64 tokens 68.7 / 33.1; 11.7 / 15.9; 120
    // blocks: 32 tokens 9.5 / 9.1; 7.6 / 8.4, 64 tokens 13.3 / 9.2; 7.4 / 7.7; 8 heads of 256 over 4, 94 blocks: 32 tokens 9.5 / 11.9; 7.0 / 10.1,
    // 64 tokens 13.2 / 11.9; 9.5 / 10.3. Workgroups of 4x4x4 in all, 256, 1024, 4096: 33 tokens behind 1024 blocks 67.9, 49.4, 44.4;
    // 12.1, 12.0, 16.8; 63 tokens 70.2, 68.5, 68.2; 12.4, 13.6, 19.9.
    if (a.T >= 64u) hipLaunchKernelGGL(k_kv4_scores_many<D>, dim3(a.n_head_kv * all, (a.T + tpt - 1u) / tpt), wg, 0, s, a);
    else if (a.G <= 4u) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_kv4_scores<D, 1>), grid, wg, 0, s, a, parts);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_kv4_scores<D, 2>), grid, wg, 0, s, a, parts);
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
    const uint32_t lists = a.T * a.n_head_kv;
    const dim3 grid(lists), grid4((lists + 3u) / 4u), wg(1024), wg4(256);
    if (a.n_blocks <= 128u) hipLaunchKernelGGL(HIP_KERNEL_NAME(tsr::k_kv4_pick_blocks<2, 1>), grid4, wg4, 0, s, a);
    else if (a.n_blocks <= 512u) hipLaunchKernelGGL(HIP_KERNEL_NAME(tsr::k_kv4_pick_blocks<8, 1>), grid4, wg4, 0, s, a);
    else if (a.n_blocks <= 2048u) hipLaunchKernelGGL(HIP_KERNEL_NAME(tsr::k_kv4_pick_blocks<2, 16>), grid, wg, 0, s, a);
    else if (a.n_blocks <= 8192u) hipLaunchKernelGGL(HIP_KERNEL_NAME(tsr::k_kv4_pick_blocks<8, 16>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(tsr::k_kv4_pick_blocks<0, 16>), grid, wg, 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
