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
