// k_attn4.hip -- attention of f32 query rows over a 4-bit KV cache, the cells of each token's runs (attn4.hpp has the
// mathematics and what a wave does).
//
// Bound. Few rows: the cells' bytes and two launches: a token of 32 heads of 128 (8 KV heads) takes 13.1 us behind 8192
// cells (a call of a graph of them: 7 the cells, 2.8 the join, the rest between launches) and 43 us behind 131071 of q4_1
// (168 MB, 3.9 TB/s; a plain read of them 29 us). Many rows: vector instructions, about 130 a 16 x 16 tile of scores and
// D 128 (a third the unpacking, a quarter the pieces of p d) against 16 matrix instructions: 2048 tokens behind 6144
// cells take 553 to 574 us (418 to 435 TFLOP/s), vector units 80 %, matrix units 35 % busy. Unpacking once for four waves through LDS,
// V in two pieces, left 270 vector instructions of 466 a tile of 32 rows and was no faster: with 239 registers two waves a
// SIMD hide neither kind behind the other; four groups of rows a workgroup gave nothing.
#include "attn4.hpp"

namespace tsr {

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
    constexpr uint32_t DC = A::DC;
    __shared__ __align__(16) uint8_t room[A::kRoom];
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
    // the waves' sums joined (here and not in a function, whose reads of w.o end up in private memory or otherwise before the loop's
    // waits: a token of 8 heads of 256 behind 65536 cells 22.6 us, 24.5 so)
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
    if (a.S > 1u) return tsr_launch_attn4_join(a, s);
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

int tsr_launch_attn4_join(const tsr::Attn4Args & a, hipStream_t s) {
    const dim3 grid(a.T * a.G * a.n_head_kv), wg(256);
    switch (a.D) {
        case 64: hipLaunchKernelGGL(tsr::k_attn4_join<64>, grid, wg, 0, s, a); break;
        case 128: hipLaunchKernelGGL(tsr::k_attn4_join<128>, grid, wg, 0, s, a); break;
        case 256: hipLaunchKernelGGL(tsr::k_attn4_join<256>, grid, wg, 0, s, a); break;
        case 512: hipLaunchKernelGGL(tsr::k_attn4_join<512>, grid, wg, 0, s, a); break;
        default: return -2;
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
