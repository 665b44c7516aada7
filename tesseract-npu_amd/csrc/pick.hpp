// pick.hpp -- the m largest of many keys, in the order of their places: by a wave or a workgroup of them. Equal keys: the
// lowest places.
//
// The keys' range is counted into bins, the bin with the cut becomes the range, until all of a bin is taken or it is one value:
// two or three passes do for thousands of keys. The bins' counts are integers: no order of additions shows.
#pragma once

#include "tsr_dev.hpp"
#include "wave_lds.hpp"

namespace tsr {

// The order of f64 and f32 as unsigned numbers; a NaN is the lowest, zeros are equal. Nothing but what takes no part is 0 (of f64:
// in the high word).
constexpr uint64_t kNan64 = (uint64_t)1 << 32;
constexpr uint32_t kNan32 = 1u;
__device__ __forceinline__ uint64_t order_of(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
    return x != x ? kNan64 : u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = fb(x + 0.0f);
    return x != x ? kNan32 : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// The number of an order (a NaN for a NaN's, 0 for zeros').
__device__ __forceinline__ float of_order(uint32_t k) { return bf(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Over the wave: the least, and the sum of the lanes up to each (row shifts, then broadcasts of the rows' ends).
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
    v = min(v, (uint32_t)dpp_i<kDppXor1>((int)v));
    v = min(v, (uint32_t)dpp_i<kDppXor2>((int)v));
    v = min(v, (uint32_t)dpp_i<kDppRowHalfMirror>((int)v));
    v = min(v, (uint32_t)dpp_i<kDppRowMirror>((int)v));
    auto x = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = min(x[0], x[1]);
    auto y = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return min(y[0], y[1]);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}

// A list's room in LDS. WAVES 16: its workgroup's; WAVES 1: its wave's own.
template <uint32_t WAVES>
struct PickRoom {
    uint32_t bins[256u * WAVES], part[WAVES][2], found[3];
};

// The wave's place in the list's workgroup, and the workgroup's barrier.
template <uint32_t WAVES>
struct Pick {
    static constexpr uint32_t kBins = 256u * WAVES, kBits = WAVES == 1u ? 8u : 12u;
    static_assert(kBins == 1u << kBits, "bins");
    PickRoom<WAVES> & room;
    uint32_t wave, lane;
    static __device__ __forceinline__ void sync() {
        if constexpr (WAVES == 1u) own_room();
        else __syncthreads();
    }

    // each(f) calls f(place, key) for every row of the wave, the lanes together, rows and waves in the order of the places; key 0
    // takes no part, at least m others do, m >= 1. put(position, place, key) for the m that are taken, positions from 0 on in the
    // order of the places.
    template <class Key, class Each, class Put>
    __device__ __forceinline__ void run(uint32_t m, Each each, Put put) {
        constexpr uint32_t kHigh = 8u * sizeof(Key) - 32u;
        const uint32_t tid = 64u * wave + lane;
        uint32_t (*part)[2] = room.part, * found = room.found;
        uint32_t least = ~0u, most = 0u;                           // of the keys' high words, the least less one
        each([&](uint32_t, Key k) {
            least = min(least, (uint32_t)(k >> kHigh) - 1u);
            most = max(most, (uint32_t)(k >> kHigh));
        });
        least = wave_min(least);
        most = ~wave_min(~most);
        if constexpr (WAVES > 1u) {
            if (lane == 0u) { part[wave][0] = least; part[wave][1] = most; }
            sync();
#pragma unroll
            for (uint32_t v = 0; v < WAVES; ++v) { least = min(least, part[v][0]); most = max(most, part[v][1]); }
        }
        const Key ones = ((Key)1 << kHigh) - 1u;
        Key lo = (Key)(least + 1u) << kHigh, hi = ((Key)most << kHigh) | ones;   // (lo > 0)
        // keys above hi are taken, those below lo are not, m of those between are
        bool whole = false;
        while (!whole && lo != hi) {
            const uint32_t bits = 64u - (uint32_t)__builtin_clzll((uint64_t)(hi - lo)), shift = bits > kBits ? bits - kBits : 0u;
            *(uint4 *)(room.bins + 4u * tid) = make_uint4(0u, 0u, 0u, 0u);
            sync();
            each([&](uint32_t, Key k) {
                if (k - lo <= hi - lo) atomicAdd(&room.bins[(uint32_t)((k - lo) >> shift)], 1u);
            });
            sync();
            // thread i has four bins from the top down: how many keys lie above them, and where m is passed
            const uint4 z = *(const uint4 *)(room.bins + kBins - 4u - 4u * tid);
            const uint32_t c[4] = { z.w, z.z, z.y, z.x }, sum = (z.x + z.y) + (z.z + z.w);
            uint32_t above = wave_scan(sum);
            if constexpr (WAVES > 1u) {
                if (lane == 63u) part[wave][0] = above;
                sync();
#pragma unroll
                for (uint32_t v = 0; v < WAVES; ++v) above += v < wave ? part[v][0] : 0u;
            }
            above -= sum;
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                if (above < m && above + c[i] >= m) { found[0] = kBins - 1u - (4u * tid + i); found[1] = above; found[2] = c[i]; }
                above += c[i];
            }
            sync();
            lo += (Key)found[0] << shift;
            const Key span = ((Key)1 << shift) - 1u;
            hi = hi - lo < span ? hi : lo + span;
            m -= found[1];
            whole = found[2] == m;
        }
        // all keys from lo on are taken or, where lo is the only one left, those above it and its first m
        uint32_t at = 0u, in = 0u;
        if constexpr (WAVES > 1u) {
            uint32_t n_from = 0u, n_in = 0u;                       // keys from lo on, those that are lo
            each([&](uint32_t, Key k) { n_from += k >= lo ? 1u : 0u; });
            if (!whole) each([&](uint32_t, Key k) { n_in += k == lo ? 1u : 0u; });
            n_from = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(n_from), 63);
            n_in = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(n_in), 63);
            sync();                                                // (the bins' partial sums have been read)
            if (lane == 0u) { part[wave][0] = n_from - n_in; part[wave][1] = n_in; }
            sync();
#pragma unroll
            for (uint32_t v = 0; v < WAVES; ++v) {
                at += v < wave ? part[v][0] : 0u;
                in += v < wave ? part[v][1] : 0u;
            }
            at += min(in, m);
        }
        auto rank = [](uint64_t lanes) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0u)); };
        if (whole) {
            each([&](uint32_t b, Key k) {
                const uint64_t sels = __ballot(k >= lo);
                if (k >= lo) put(at + rank(sels), b, k);
                at += (uint32_t)__builtin_popcountll(sels);
            });
        } else {
            each([&](uint32_t b, Key k) {
                const uint64_t mids = __ballot(k == lo);
                const bool sel = k > lo || (k == lo && in + rank(mids) < m);
                const uint64_t sels = __ballot(sel);
                if (sel) put(at + rank(sels), b, k);
                at += (uint32_t)__builtin_popcountll(sels);
                in += (uint32_t)__builtin_popcountll(mids);
            });
        }
    }
};

}  // namespace tsr
