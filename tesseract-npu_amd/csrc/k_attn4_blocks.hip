// k_attn4_blocks.hip -- attention of f32 query rows over listed blocks of a 4-bit KV cache (attn4.hpp has the mathematics and
// what a wave does): a token's query heads of one KV head share a list and are the rows of its workgroups, whose waves take
// the lists' tiles in turn, those that the rows see whole first (gathered 64 entries at a time), the list asked for ahead of all else.
//
// Bound: a token's latency (32 heads of 128 over 8 KV heads, 32 blocks of 64 in 16 splits: 7.2 us and the join 3.9, its 9.4 MB in 2). Many
// tokens: vector instructions, since the codes of a list are unpacked for its few rows alone (512 such tokens 160 us of a call's 194;
// the products would take 14). 33 sequences' tokens of two heads of 256 a list: 22 us, one tile ahead a wave.
#include "attn4.hpp"

namespace tsr {

// Workgroup (KV head, split, token and group of its rows).
template <int D, int C, uint32_t TYPE>
__global__ __launch_bounds__(256, waves_of(D, 1, C, TYPE)) void k_attn4_blocks(Attn4BlocksArgs b) {
    using A = Attn4<D, 1, C, TYPE>;
    Attn4Args a = b.a;
    const uint32_t n_rg = (a.G + A::RW - 1u) / A::RW, t = blockIdx.z / n_rg, r0 = (blockIdx.z - t * n_rg) * A::RW;
    const uint32_t h = blockIdx.x, split = blockIdx.y, nh = a.G * a.n_head_kv;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), lane = threadIdx.x & 63u;
    const size_t nr = (size_t)a.T * nh, row0 = (size_t)t * nh + h * a.G;
    float * out = a.out + (size_t)t * a.out_stride + (size_t)h * a.G * D;
    a.T = 1u;                                                      // the token alone
    a.mask = nullptr;
    a.q += (size_t)t * a.q_stride;
    if (a.runs != nullptr) a.runs += 4u * (size_t)t;
    __shared__ __align__(16) uint8_t room[A::kRoom];
    __shared__ float2 ml[kWaves * A::RT];
    __shared__ uint32_t list[kWaves][64];
    const int32_t * ids = b.blocks + ((size_t)t * a.n_head_kv + h) * b.n_sel;
    const uint32_t per = b.block / 32u, n_blocks = (a.n_kv + b.block - 1u) / b.block;
    auto entry = [&](uint32_t j) {
        const uint32_t i = j / per, id = (uint32_t)ids[i];
        return id < n_blocks ? id * per + (j - i * per) : ~0u;
    };
    const uint32_t part = split * kWaves + wave, parts = a.S * kWaves, total = b.n_sel * per;
    const uint32_t e0 = entry(min(part + parts * lane, total - 1u));
    A w;
    w.load_runs(a, h, r0, lane);
    w.run_list(a, h, part, parts, total, e0, entry, list[wave], (h8 *)room, wave, lane);
    w.finish();
    auto place = [&](uint32_t r) { return a.S > 1u ? a.part + attn4_part_row(nr, D, split, row0 + r) : out + (size_t)r * D; };
    auto sums = [&](uint32_t r, float m, float l) { *(float2 *)(a.part + attn4_part_sum(nr, D, a.S, split, row0 + r)) = make_float2(m, l); };
    // the waves' sums joined, as k_attn4.hip has it
    constexpr uint32_t RT = A::RT, DC = A::DC;
    const uint32_t g = lane >> 4, c = lane & (C - 1u), rl = (lane & 15u) / C;
    float * lo = (float *)room;
#pragma unroll
    for (uint32_t z = 0; z < D / DC; ++z) {
        __syncthreads();                                       // (the queries, the values before have been read)
        if (z == 0u && g == 0u && c == 0u) ml[wave * RT + rl] = make_float2(w.m[0], w.l[0]);
#pragma unroll
        for (uint32_t j = 0; j < DC / 16; ++j) {
            const f4 x = w.o[0][z * (DC / 16) + j];
            if (C == 1 || ((z * (DC / 16) + j) / 2u) % C == c)
                *(float4 *)(lo + (wave * RT + rl) * DC + 16 * j + 4 * g) = make_float4(x[0], x[1], x[2], x[3]);
        }
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < RT * (DC / 4); e += 64u * kWaves) {
            const uint32_t r = e / (DC / 4), d = 4u * (e % (DC / 4));
            if (r0 + r >= a.G) continue;
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

template <int D, int C, uint32_t TYPE>
static int launch_blocks(const Attn4BlocksArgs & b, hipStream_t s) {
    const uint32_t n_rg = (b.a.G + 16u / C - 1u) / (16u / C);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_attn4_blocks<D, C, TYPE>), dim3(b.a.n_head_kv, b.a.S, b.a.T * n_rg), dim3(64u * kWaves), 0, s, b);
    if (b.a.S > 1u) return tsr_launch_attn4_join(b.a, s);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

template <int D, uint32_t TYPE>
static int launch_blocks_d(const Attn4BlocksArgs & b, uint32_t C, hipStream_t s) {
    switch (C) {
        case 2: return launch_blocks<D, 2, TYPE>(b, s);
        case 4:
            if constexpr (D >= 128) return launch_blocks<D, 4, TYPE>(b, s);
        default: return launch_blocks<D, 1, TYPE>(b, s);
    }
}

template <uint32_t TYPE>
static int launch_blocks_t(const Attn4BlocksArgs & b, uint32_t C, hipStream_t s) {
    switch (b.a.D) {
        case 64: return launch_blocks_d<64, TYPE>(b, C, s);
        case 128: return launch_blocks_d<128, TYPE>(b, C, s);
        case 256: return launch_blocks_d<256, TYPE>(b, C, s);
        case 512: return launch_blocks_d<512, TYPE>(b, C, s);
        default: return -2;
    }
}

}  // namespace tsr

int tsr_launch_attn4_blocks(const tsr::Attn4BlocksArgs & b, uint32_t C, hipStream_t s) {
    return b.a.type == tsr::kKvQ4_0 ? tsr::launch_blocks_t<tsr::kKvQ4_0>(b, C, s) : tsr::launch_blocks_t<tsr::kKvQ4_1>(b, C, s);
}
