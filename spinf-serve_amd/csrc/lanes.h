// Sums and the like over the lanes of a wave by lane permutations, without LDS.
#pragma once
#include <hip/hip_runtime.h>

template <int CTRL>
__device__ __forceinline__ unsigned permuted(unsigned x) { return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false); }

// f (commutative, associative as far as it matters) over each N lanes in a row, N = 2 .. 64: neighbours, pairs, quads and eights within a row of 16 lanes, then the rows
template <int N = 64, class T, class F>
__device__ __forceinline__ T over_lanes(T x, F f) {
    constexpr int WORDS = sizeof(T) / 4;
    struct Words { unsigned w[WORDS]; };
    const auto step = [&](auto move) __attribute__((always_inline)) {
        const Words a = __builtin_bit_cast(Words, x);
        Words b, c;
#pragma unroll
        for (int i = 0; i < WORDS; i++) move(a.w[i], b.w[i], c.w[i]);
        x = f(__builtin_bit_cast(T, b), __builtin_bit_cast(T, c));
    };
    if constexpr (N >= 2) step([](unsigned a, unsigned& b, unsigned& c) __attribute__((always_inline)) { b = a; c = permuted<0xb1>(a); });
    if constexpr (N >= 4) step([](unsigned a, unsigned& b, unsigned& c) __attribute__((always_inline)) { b = a; c = permuted<0x4e>(a); });
    if constexpr (N >= 8) step([](unsigned a, unsigned& b, unsigned& c) __attribute__((always_inline)) { b = a; c = permuted<0x141>(a); });
    if constexpr (N >= 16) step([](unsigned a, unsigned& b, unsigned& c) __attribute__((always_inline)) { b = a; c = permuted<0x140>(a); });
    if constexpr (N >= 32) step([](unsigned a, unsigned& b, unsigned& c) __attribute__((always_inline)) { const auto y = __builtin_amdgcn_permlane16_swap(a, a, false, false); b = y[0]; c = y[1]; });
    if constexpr (N >= 64) step([](unsigned a, unsigned& b, unsigned& c) __attribute__((always_inline)) { const auto y = __builtin_amdgcn_permlane32_swap(a, a, false, false); b = y[0]; c = y[1]; });
    return x;
}
