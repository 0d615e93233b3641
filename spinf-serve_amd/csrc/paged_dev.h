// Device pieces that the paged cache's kernels share: scalar loads, the division by the page size, the DMA of a 32-key tile.
#pragma once
#include <hip/hip_runtime.h>

#include "attn_tiles.h"
#include "paged.h"

constexpr int TK = PAGED_TILE;
constexpr float LOG2E = 1.4426950408889634f;

typedef const __attribute__((address_space(4))) int* scalar_ints;
// a value at a wave-uniform address, through the scalar cache
__device__ __forceinline__ int sload(const int* p, int i) { return ((scalar_ints)(size_t)p)[__builtin_amdgcn_readfirstlane(i)]; }

// The lane's index, found anew (two instructions): for code outside a tile loop, where a value kept in a register across the loop would be spilled.
__device__ __forceinline__ int lane_now() {
    int lane;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
    return lane;
}

// Division of n < 2^31 by a number known when the kernel is launched, as the high word of a product: the multiplier ceil(2^(31 + b) / d), b = ceil(log2 d), and the
// shift b - 1 (exact: the multiplier is too large by less than one, which is less than 2^b / n of a unit of the quotient's last place).
struct Div {
    int d; unsigned mul; int shift;   // mul 0: divide by 1
    static Div by(int d) {
        Div x = {d, 0, 0};
        if (d > 1) {
            int b = 0;
            while ((1 << b) < d) b++;
            x.mul = (unsigned)(((1ull << (31 + b)) + d - 1) / d);
            x.shift = b - 1;
        }
        return x;
    }
    __device__ __forceinline__ int of(int n) const { return mul ? (int)(__umulhi((unsigned)n, mul) >> shift) : n; }
};
// of the page size, in pieces of 16 keys
struct PageDiv : Div {
    static PageDiv of_page(int page) { return {Div::by(page / 16)}; }
};

// The soft cap, cap tanh(scale s / cap): what becomes of a score here is the tanh; `unit` is what it is worth in units of log 2 (without a cap: the score stays, and is worth
// scale log2 e).  With z = scale s / cap, tanh z = 1 - 2 / (exp(2 z) + 1): the subtraction leaves an error of 2^-24, that is of the cap, whatever the score.  That is
// nothing under a cap of up to 64 (4e-6 on a score), and 0.1 on every score under one of 10^6: there tanh z is z (1 + q P(q)) for z below a third, q = z^2, P the
// polynomial of degree 2 of least largest relative error (2^-25, found by Remez' exchange), and the other form from there on; a score keeps its 21 bits.
// A score's result depends on that score alone.  (With the polynomial under every cap, 7 x 517 new tokens under a window of 1,024 took 115 us where scores lie about
// the cap, 101 with the exponentials alone.)
struct SoftCap {
    float in, two_in, edge, unit;   // scale / cap; 2 log2 e scale / cap; a third of cap / scale; cap log2 e
    bool on, narrow;
    // false: numbers that fp32 does not hold
    static bool of(float scale, float softcap, SoftCap& x) {
        x = {0.f, 0.f, 0.f, scale * LOG2E, softcap > 0.f && softcap <= 0x1p100f, false};   // (a larger cap changes no score below 2^88, and fp32 would not hold z)
        if (x.on) x = {scale / softcap, 2.0f * LOG2E * (scale / softcap), softcap / (3.0f * scale), softcap * LOG2E, true, softcap <= 64.f};
        return x.two_in < INFINITY && x.unit < INFINITY;
    }
    __device__ __forceinline__ float small(float s) const {
        const float z = s * in, q = z * z;
        return z * __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, -0.049570475f, 0.13305548f), -0.33332828f), 1.0f);
    }
    __device__ __forceinline__ float large(float s) const { return 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * two_in) + 1.0f); }
    __device__ __forceinline__ float mixed(float s) const { return __builtin_fabsf(s) < edge ? small(s) : large(s); }
    __device__ __forceinline__ float of(float s) const { return narrow ? large(s) : mixed(s); }
    __device__ __forceinline__ void of(f32x16& s) const {   // of a tile's scores
        if (narrow) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = large(s[i]);
            return;
        }
        float far = __builtin_fabsf(s[0]);
#pragma unroll
        for (int i = 1; i < 16; i++) far = fmaxf(far, __builtin_fabsf(s[i]));
        if (__builtin_amdgcn_ballot_w64(!(far < edge)) == 0) {   // (the usual case: caps lie far above most scores)
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = small(s[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = mixed(s[i]);
        }
    }
};

constexpr int vmcnt_imm(int n) { return 0x0f70 | (n & 15) | ((n >> 4) << 14); }   // waits for all but the n youngest vector memory operations

// DMA of regions reg0 .. reg0 + N - 1 of a tile (32 rows of W dims) into the LDS tile at `lds`; RS: distance of its regions
template <int W, int N, int RS>
__device__ __forceinline__ void fetch(const char* b0, const char* b1, long row, int last, int reg0, unsigned lds, int lane) {
    using G = Geo<W, TK>;
    const int slot = lane / G::CPR, chunk = lane % G::CPR;
    if (last == TK - 1 && b1 == b0 + 16 * row) {   // 32 rows, one after the other: a uniform base and a constant per lane
        const unsigned off = (unsigned)(slot * G::NREG * (int)row + chunk * 16);
#pragma unroll
        for (int i = 0; i < N; i++) dma16_uniform(b0 + (reg0 + i) * row, off, lds + (reg0 + i) * RS);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            int r = reg0 + i + G::NREG * slot;
            r = r < last ? r : last;
            const char* b = r >= 16 ? b1 : b0;
            dma16_lane(b + (r & 15) * row + chunk * 16, lds + (reg0 + i) * RS);
        }
    }
}
