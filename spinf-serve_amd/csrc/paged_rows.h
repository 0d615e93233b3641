// What a wave of the paged cache's attention kernels holds of its 32 rows, and what it does with a tile of 32 keys: scores, softmax, product with the values.  Which
// keys a row sees is the kernels' own.
#pragma once
#include "paged_dev.h"

constexpr float TAU = 8.f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int LGKM0 = 0xc07f;                                                     // waits for every LDS operation

// A wave's 32 rows: queries, output accumulators, softmax state
template <int D, int DV, bool CAP>
struct RowTile {
    using GK = Geo<D, TK>;
    using GV = Geo<DV, TK>;
    static constexpr int NS = D / 16, NDT = DV / 32;
    static constexpr int KAHEAD = D >= 256 ? 3 : 4, VAHEAD = D >= 256 ? 3 : 4;   // fragments read ahead of the products
    bf16x8 qf[NS];
    f32x16 o[NDT];
    float M, l, over;   // reference (0 before a row's first key), sum, score above which the reference is raised (-inf: no key so far)
    int lane, m, g;

    __device__ __forceinline__ void reset() {
        M = 0.f;
        l = 0.f;
        over = -INFINITY;
#pragma unroll
        for (int dt = 0; dt < NDT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[dt][i] = 0.f;
    }
    // scores of a tile; register i holds key 8 (i / 4) + 4 g + i % 4
    __device__ __forceinline__ void scores(const char* kt_lds, f32x16& s) {
        const char* krow = kt_lds + GK::k_off(m) + 16 * g;
        constexpr int PF = NS < KAHEAD ? NS : KAHEAD;
        bf16x8 kf[PF];
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.f;
#pragma unroll
        for (int st = 0; st < PF; st++) kf[st] = *(const bf16x8*)(krow + 32 * st);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < NS; st++) {
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[st % PF], qf[st], s, 0, 0, 0);
            if (st + PF < NS) kf[st % PF] = *(const bf16x8*)(krow + 32 * (st + PF));
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // scores (with a cap: their tanh) -> probabilities.  The reference stays while no score lies more than TAU above it, which one comparison per lane with `over` (the score that
    // far above, in the scores' own units) tells; where one does, or a row meets its first keys, it is raised and what was summed is rescaled.
    __device__ __forceinline__ void softmax(const SoftCap& cap, f32x16& s, bf16x8 (&pb)[2]) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; i++) mx = fmaxf(mx, s[i]);
        if (__builtin_amdgcn_ballot_w64(mx > over) != 0) {
            mx = lane32_max(mx);
            const float t = mx * cap.unit;
            const bool fresh = over == -INFINITY, up = mx > -INFINITY && (fresh || t > M + TAU);
            const float alpha = up && !fresh ? __builtin_amdgcn_exp2f(M - t) : 1.0f;
            if (__builtin_amdgcn_ballot_w64(up && !fresh) != 0) {   // (rows without a key so far hold zeros)
#pragma unroll
                for (int dt = 0; dt < NDT; dt++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[dt][i] *= alpha;
            }
            l *= alpha;
            M = up ? t : M;
            over = up ? (M + TAU) / cap.unit : over;
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], cap.unit, -M));
            sum += pr;
            pb[i >> 3][i & 7] = (__bf16)pr;
        }
        l += sum;
    }
    __device__ __forceinline__ void values(const char* vt_lds, const bf16x8 (&pb)[2]) {
        const int tr_a = lane & 3, tr_j = (lane >> 2) & 3, tr_mb = (lane >> 4) & 1;
        const char* vrow = vt_lds + GV::v_off(4 * g + tr_j) + 32 * tr_mb + 8 * tr_a;
        constexpr int NF = 2 * NDT, PF = NF < VAHEAD ? NF : VAHEAD;
        s16x4 lo[PF], hi[PF];
        auto ask = [&](const int f) __attribute__((always_inline)) {
            const char* vp = vrow + GV::v_off(16 * (f / NDT)) + 64 * (f % NDT);
            lo[f % PF] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)vp);
            hi[f % PF] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vp + GV::v_off(8)));
        };
#pragma unroll
        for (int f = 0; f < PF; f++) ask(f);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < NF; f++) {
            const bf16x8 a = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo[f % PF], hi[f % PF], 0, 1, 2, 3, 4, 5, 6, 7));
            o[f % NDT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, pb[f / NDT], o[f % NDT], 0, 0, 0);
            if (f + PF < NF) ask(f + PF);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // is some result of the wave's rows not finite?
    __device__ __forceinline__ bool spoilt(int rows_left) const {
        float t = 0.f;
#pragma unroll
        for (int dt = 0; dt < NDT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) t += o[dt][i] * 0.f;
        return __builtin_amdgcn_ballot_w64((lane_now() & 31) < rows_left && !(t == 0.f)) != 0;
    }
};

// 1 / sum; rows that saw nothing come out as zeros
__device__ __forceinline__ float inverse(float sum) { return sum == 0.f ? 0.f : 1.0f / sum; }
__device__ __forceinline__ float log_sum(float M, float sum) { return sum == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(sum)) * LN2; }
