// Selection over rows of logits: order-preserving bit patterns, joins over a
// wave's lanes, bounds of the nth largest lane, and vectors that start anywhere.
// Shared by beam search (beam.hip) and the token scores (scoring.hip).
#pragma once

#include <type_traits>

#include "bdm_common.h"

namespace bdm {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// ------------------------------------------------------------------ ordered bit patterns
// Unsigned integers in the order of the floating values; -0 counts as +0.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint64_t ordered(double x) {
    const uint64_t u = uint64_t(__double_as_longlong(x + 0.0));
    return u ^ (uint64_t(int64_t(u) >> 63) | 0x8000000000000000ull);
}

// The wave's lanes joined by op, which leaves x as it is beside `none`, in
// every lane: a row's 16 lanes by shifts, then the rows, none of it through LDS.
template <typename F>
__device__ __forceinline__ uint32_t wave_join(uint32_t x, uint32_t none, F op) {
    auto with = [&](auto step) {
        x = op(x, uint32_t(__builtin_amdgcn_update_dpp(int(none), int(x), decltype(step)::value, 0xf, 0xf, false)));
    };
    with(std::integral_constant<int, 0x111>{});  // row_shr by 1, 2, 4, 8
    with(std::integral_constant<int, 0x112>{});
    with(std::integral_constant<int, 0x114>{});
    with(std::integral_constant<int, 0x118>{});
    with(std::integral_constant<int, 0x142>{});  // row_bcast of lanes 15, 31
    with(std::integral_constant<int, 0x143>{});
    return uint32_t(__builtin_amdgcn_readlane(int(x), kWave - 1));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    return wave_join(x, 0, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ uint32_t wave_min(uint32_t x) {
    return wave_join(x, UINT32_MAX, [](uint32_t a, uint32_t b) { return min(a, b); });
}
__device__ __forceinline__ float wave_max(float x) {
    return __uint_as_float(wave_join(__float_as_uint(x), __float_as_uint(-INFINITY), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ float wave_sum(float x) {
    return __uint_as_float(wave_join(__float_as_uint(x), 0, [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
// The sum of the first row's 16 lanes.
__device__ __forceinline__ uint32_t row_sum(uint32_t x) {
    auto with = [&](auto step) {
        x += uint32_t(__builtin_amdgcn_update_dpp(0, int(x), decltype(step)::value, 0xf, 0xf, false));
    };
    with(std::integral_constant<int, 0x111>{});
    with(std::integral_constant<int, 0x112>{});
    with(std::integral_constant<int, 0x114>{});
    with(std::integral_constant<int, 0x118>{});
    return uint32_t(__builtin_amdgcn_readlane(int(x), 15));
}
__device__ __forceinline__ int popcount(uint64_t m) { return __popcll(m); }

// Lower bounds of the nth largest of the lanes' ordered values (0: the lane has
// none) for several n, each one of them itself; 0 where fewer lanes have one.
// Bisected, a ballot a bit, over where the values lie between the lowest and
// the highest of them, in 256 parts: 9 ballots in the place of the 16 of the
// patterns' top half, and as near where the lanes are like each other (8
// prompts of 8 beams over 50,257 BF16 logits: 13.6 -> 12.2 us, 64 of 16: 45.4
// -> 40.9).
template <int N>
struct Bounds {
    uint32_t at[N];
};
template <int N>
__device__ __forceinline__ Bounds<N> nth_of_lanes(uint32_t value, Bounds<N> nth) {
    const uint32_t high = wave_max(value), low = wave_min(value ? value : UINT32_MAX), range = high - low;
    const int shift = max(0, 24 - __clz(int(range | 1)));
    const uint32_t part = value ? ((value - low) >> shift) + 1 : 0;
    Bounds<N> bound{};
#pragma unroll
    for (int bit = 8; bit >= 0; --bit) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t next = bound.at[n] | (1u << bit);
            if (uint32_t(popcount(__ballot(part >= next))) >= nth.at[n]) bound.at[n] = next;
        }
    }
    // parts of more than an eighth of their values, as where the lanes lie on both sides of zero: the one of the bound
    // in 256 parts again (64 prompts of 8 beams over 1,024 tokens around zero: 19.8 -> 7.4 us)
    const bool coarse = shift > 20;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (!bound.at[n]) continue;
        bool reaches = part >= bound.at[n];
        if (coarse) {
            const uint32_t within = value - (low + ((bound.at[n] - 1) << shift));
            const uint32_t finer = part > bound.at[n] ? 512 : reaches ? (within >> (shift - 8)) + 1 : 0;
            uint32_t found = 0;
#pragma unroll
            for (int bit = 8; bit >= 0; --bit) {
                const uint32_t next = found | (1u << bit);
                if (uint32_t(popcount(__ballot(finer >= next))) >= nth.at[n]) found = next;
            }
            reaches = finer >= found;
        }
        bound.at[n] = wave_min(reaches ? value : UINT32_MAX);
    }
    return bound;
}

// The team's waves wait for each other and see each other's LDS writes.
template <int WAVES>
__device__ __forceinline__ void team_sync() {
    if constexpr (WAVES > 1) {
        __syncthreads();
    } else {
        // one wave: its LDS accesses are in order, the compiler has to keep them so
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T> struct Vec;
template <> struct Vec<bf16_t> {
    static constexpr int kSize = 8;
    static __device__ __forceinline__ void widen(u32x4 u, float *out) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            out[2 * i] = __uint_as_float(u[i] << 16);
            out[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
};
template <> struct Vec<float> {
    static constexpr int kSize = 4;
    static __device__ __forceinline__ void widen(u32x4 u, float *out) {
        out[0] = __uint_as_float(u.x), out[1] = __uint_as_float(u.y);
        out[2] = __uint_as_float(u.z), out[3] = __uint_as_float(u.w);
    }
};

// 16 bytes that start at any element.  A row's values are dealt to lanes by their tokens, wherever the row starts: the
// sum of exponentials, whose last bits follow its order, is the same for equal rows, so that beams with equal logits
// and scores tie.  (64 prompts of 16 beams over 50,257 BF16 logits, half the rows at odd addresses: 39.7 us; dealt from
// each row's own boundary 39.7, over 50,256, all of them aligned, 39.5.)
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) AnyVector {
    u32x4 bits;
};
static_assert(alignof(AnyVector<bf16_t>) == 2 && alignof(AnyVector<float>) == 4 && sizeof(AnyVector<bf16_t>) == 16);

}  // namespace bdm
