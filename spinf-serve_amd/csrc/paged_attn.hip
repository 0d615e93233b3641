// Attention of new tokens over a paged cache of keys and values for gfx950 (MI355X): single tokens, chunks, trees of questions below a
// stored content.  No counterpart in the reference, whose contents are read anew with every request.
//
// Mathematics.  Row = new token x query head; out = sum_s p_s v_s / sum_s p_s over the stored keys s that the row sees, p_s = exp(t_s - ref), t_s the
// (capped) scaled score, ref a running maximum that is raised, and what was summed so far rescaled, only where a tile's maximum exceeds it by more
// than TAU (exponents in units of log 2; probabilities stay below 2^TAU).  Sums, maxima and accumulators are fp32; the p_s are rounded to bf16 once, for the matrix product with V
// (their sum takes the unrounded ones): an error of at most 2^-8 of each term, of either sign, as the output's own rounding.
//
// Tiles.  32 keys; S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16_bf16 (a lane owns one row; V^T through ds_read_b64_tr_b16), K and V
// global -> LDS by DMA in the padded layout of attn_tiles.h.  A tile is two halves of 16 keys and a page a multiple of 16, so a half lies in one
// page: two scalar reads of the page list per tile, no per-key lookup.  Rows behind the stored keys are never read (the last key is read in their place).
//
// Two kernels over the items of csrc/pagedplan.cpp:
//   wave   few rows: the workgroup's waves share 32 rows and divide the tiles, each with a tile buffer of its own and no barrier; joined at the end.
//          Bound by HBM where the GPU is full (64 requests of ~3,000 keys, one token, 24 heads on 4 of 256 dims: 863 MB in 164 us, 5.3 TB/s; one of 131,071 keys of
//          512 dims 46 us, 5.8), by a tile's latency where it is not (a request's 350 questions' tokens on 301 keys, 16 on 8 of 256: 15.5 us).
//   block  many rows: four waves with 32 rows each on the same double-buffered tiles, one barrier per tile.  Bound by what a wave cannot overlap: products,
//          softmax and LDS reads of one tile follow each other, and the two or three waves of a SIMD hide only part of it (two documents of 8,192 new on
//          8,192 stored tokens, 32 on 16 of 128: 3.10 ms, 1.06 PFLOP/s, matrix pipe busy 45 %; 8 of 256 dims: 2.84 ms, 1.16 PFLOP/s).
// and paged_join_kernel where an item's keys were cut into pieces.
// 512 dims: a wave's registers hold the accumulators of half of them.  In the wave kernel an item is two workgroups, each with all of S and half of the output's dims
// (bound by the keys' bytes, which the L2 gives the second one); in the block kernel two waves share their rows, each with half of the products on either side.
//
// Keys that a row does not see have p = 0 exactly; 0 x inf or NaN in the matrix product would still be NaN.  Nothing is spent on that in the usual
// case: a workgroup that masked some tile and whose results are not all finite looks whether those tiles hold such values (rubbish), and if so computes its rows again
// one by one, over the keys that each of them sees (slow_row).
#include <hip/hip_runtime.h>

#include <climits>

#include "spinf_tree.h"
#include "common.h"
#include "paged.h"
#include "attn_tiles.h"
#include "paged_dev.h"

namespace {

constexpr float TAU = 8.f;
constexpr float LN2 = 0.6931471805599453f;

struct Params {
    const __bf16* q; __bf16* out; float* lse;
    long q_tok, q_head, o_tok, o_head;
    const char* k; const char* v;
    unsigned k_page, k_row, v_page, v_row; long k_head, v_head;   // bytes
    bool same;                                                    // keys and values have the same strides
    const int* table; const int* end; const int* pos;
    const PagedItem* items; const PagedRun* runs; const PagedJoin* joins;
    float* part_o; float2* part_ml;
    int n_items, hq, group, window;
    PageDiv page;
    SoftCap cap;
};

__device__ __forceinline__ PagedItem load_item(const PagedItem* items, int i) {
    PagedItem it;
    const int* p = (const int*)(items + i);
    it.cu = sload(p, 0); it.T = sload(p, 1); it.L = sload(p, 2); it.tab = sload(p, 3);
    it.kvh = sload(p, 4); it.row0 = sload(p, 5); it.first = sload(p, 6); it.runs = sload(p, 7);
    it.tiles = sload(p, 8); it.part = sload(p, 9);
    return it;
}

// the tiles of an item, in order
struct Walk {
    const int* at;
    int kt, count, bits, off, tiles;
    __device__ __forceinline__ void load() {
        kt = sload(at, 0);
        count = sload(at, 1);
        bits = sload(at, 2);
    }
    __device__ __forceinline__ Walk(const PagedRun* runs, const PagedItem& it, int start) : at((const int*)(runs + it.first)), kt(0), count(0), bits(0), off(0), tiles(it.tiles) {
        if (tiles > 0) load();
        step(start);
    }
    __device__ __forceinline__ bool more() const { return tiles > 0; }
    __device__ __forceinline__ int tile() const { return kt + off; }
    __device__ __forceinline__ void step(int n) {
        tiles -= n;
        if (tiles <= 0) return;
        off += n;
        while (off >= count) {   // (tiles are left, so there is a run behind this one)
            off -= count;
            at += 4;
            load();
        }
    }
};

// The pages of a tile's two halves.  Asked for a tile ahead (the scalar loads are on their way while the tile before is computed); pages of a multiple of
// 32 keys hold both halves, so one is asked for.
struct Pages {
    int n, row0, row1, id0, id1;   // the tile's first 16-key piece; rows of the halves inside their pages; the pages
    __device__ __forceinline__ void ask(const Params& p, const PagedItem& it, int kt) {
        n = 2 * kt;
        const int a = p.page.of(n);
        id0 = sload(p.table, it.tab + a);
        row0 = (n - a * p.page.d) * 16;
        if (p.page.d & 1) {
            const int end = (it.L - 1) >> 4, n1 = n + 1 < end ? n + 1 : end, b = p.page.of(n1);
            id1 = sload(p.table, it.tab + b);
            row1 = (n1 - b * p.page.d) * 16;
        }
    }
};

// Where a tile lies: byte addresses of row 0 and row 16 of the key / value head's keys and values, and the tile's last stored row
struct Place {
    const char *k0, *k1, *v0, *v1;
    int last;
    // kb, vb: the cache's keys and values of the key / value head
    __device__ __forceinline__ Place(const Params& p, const char* kb, const char* vb, int L, const Pages& g) {
        last = L - 1 - g.n * 16 < TK - 1 ? L - 1 - g.n * 16 : TK - 1;
        const unsigned long long ko = (unsigned long long)(unsigned)g.id0 * p.k_page + (unsigned long long)(unsigned)g.row0 * p.k_row;
        k0 = kb + ko;
        v0 = vb + (p.same ? ko : (unsigned long long)(unsigned)g.id0 * p.v_page + (unsigned long long)(unsigned)g.row0 * p.v_row);
        if (p.page.d & 1) {
            const unsigned long long k2 = (unsigned long long)(unsigned)g.id1 * p.k_page + (unsigned long long)(unsigned)g.row1 * p.k_row;
            k1 = kb + k2;
            v1 = vb + (p.same ? k2 : (unsigned long long)(unsigned)g.id1 * p.v_page + (unsigned long long)(unsigned)g.row1 * p.v_row);
        } else {
            k1 = k0 + 16 * (unsigned long long)p.k_row;
            v1 = v0 + 16 * (unsigned long long)p.v_row;
        }
    }
};

// subtree ends and positions of a tile's new tokens into 2 x 256 bytes of LDS (the 32 keys twice)
__device__ __forceinline__ void fetch_meta(const Params& p, const PagedItem& it, int kt, unsigned lds, int lane) {
    int u = kt * TK + (lane & (TK - 1)) - (it.L - it.T);
    u = u < 0 ? 0 : u < it.T ? u : it.T - 1;
    dma4_lane(p.end + it.cu + u, lds);
    dma4_lane(p.pos + it.cu + u, lds + 256);
}

constexpr int LGKM0 = 0xc07f;                                                     // waits for every LDS operation

// A wave's 32 rows: queries, output accumulators, softmax state
template <int D, int DV, bool CAP>
struct Rows {
    using GK = Geo<D, TK>;
    using GV = Geo<DV, TK>;
    static constexpr int NS = D / 16, NDT = DV / 32;
    static constexpr int KAHEAD = D >= 256 ? 3 : 4, VAHEAD = D >= 256 ? 3 : 4;   // fragments read ahead of the products
    bf16x8 qf[NS];
    f32x16 o[NDT];
    float M, l, over;   // reference (0 before a row's first key), sum, score above which the reference is raised (-inf: no key so far)
    int lane, m, g, tok, qpos;

    // queries of rows row0 + m, dims col ..
    __device__ __forceinline__ void load(const Params& p, const PagedItem& it, int row0, int col = 0) {
        lane = threadIdx.x & 63;
        m = lane & 31;
        g = lane >> 5;
        const int N = it.T * p.group, row = row0 + m;
        const int r = row < N ? row : N - 1;
        tok = r / p.group;
        const int head = it.kvh * p.group + (r - tok * p.group);
        const __bf16* qp = p.q + (long)(it.cu + tok) * p.q_tok + (long)head * p.q_head + col + 8 * g;
#pragma unroll
        for (int s = 0; s < NS; s++) qf[s] = *(const bf16x8*)(qp + 16 * s);
        qpos = it.L - it.T + tok;
        if (p.window && p.pos) qpos = p.pos[it.cu + tok];
        // (waited for here: left to the compiler, the wait would sit at the first use inside the tile loop, behind the DMAs in flight)
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
#pragma unroll
        for (int s = 0; s < NS; s++) asm volatile("" : "+v"(qf[s]));
        asm volatile("" : "+v"(qpos));
    }
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
    // (four keys at a time, a scheduling barrier in between: requested all at once, the keys' ends and positions would cost the tile loop its registers)
    __device__ __forceinline__ void mask(const Params& p, const PagedItem& it, int kt, const int* meta, bool tree, f32x16& s) {
        const int u0 = kt * TK - (it.L - it.T) + 4 * g;   // key 8 i4 + j of this lane is new token u0 + 8 i4 + j of the request (below 0: stored before)
        const int sees = p.window ? p.window : INT_MAX, far = p.window ? qpos - (kt * TK + 4 * g) : 0;   // distance to the lane's first key
        if (!tree) {
            // keys first .. last of the lane's: the rows' own key last, the window's first
            const int last = tok - u0, first = far - sees;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int k = 8 * (i >> 2) + (i & 3);
                s[i] = (k <= last) & (k > first) ? s[i] : -INFINITY;
            }
        } else {
            const int row = it.cu + tok;
#pragma unroll
            for (int i4 = 0; i4 < 4; i4++) {
                __builtin_amdgcn_sched_barrier(0);
                const int4 e = *(const int4*)(meta + 8 * i4 + 4 * g), ps = *(const int4*)(meta + 64 + 8 * i4 + 4 * g);
                const int ev[4] = {e.x, e.y, e.z, e.w}, pv[4] = {ps.x, ps.y, ps.z, ps.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int k = 8 * i4 + j;
                    const bool fresh = u0 + k >= 0;
                    bool vis = (u0 + k <= tok) & (!fresh | (row < ev[j]));
                    if (p.window) vis = vis & ((fresh ? qpos - pv[j] : far - k) < sees);
                    s[4 * i4 + j] = vis ? s[4 * i4 + j] : -INFINITY;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // scores (with a cap: their tanh) -> probabilities.  The reference stays while no score lies more than TAU above it, which one comparison per lane with `over` (the score that
    // far above, in the scores' own units) tells; where one does, or a row meets its first keys, it is raised and what was summed is rescaled.
    __device__ __forceinline__ void softmax(const Params& p, f32x16& s, bf16x8 (&pb)[2]) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; i++) mx = fmaxf(mx, s[i]);
        if (__builtin_amdgcn_ballot_w64(mx > over) != 0) {
            mx = lane32_max(mx);
            const float t = mx * p.cap.unit;
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
            over = up ? (M + TAU) / p.cap.unit : over;
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], p.cap.unit, -M));
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

// place of a row in lse
__device__ __forceinline__ long row_head(const Params& p, const PagedItem& it, int row) {
    const int tok = row / p.group;
    return (long)(it.cu + tok) * p.hq + it.kvh * p.group + (row - tok * p.group);
}
// 1 / sum; rows that saw nothing come out as zeros
__device__ __forceinline__ float inverse(float sum) { return sum == 0.f ? 0.f : 1.0f / sum; }
__device__ __forceinline__ float log_sum(float M, float sum) { return sum == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(sum)) * LN2; }

// Do partly masked tiles of an item hold values that are not finite?  (If not, a result that is not finite came from keys the row sees.)  Every wave looks at its
// share of the tiles; groups: row groups of the item.
template <int DV>
__device__ bool rubbish(const Params& p, const PagedItem& it, int vcol, int w, int nw, int groups) {
    constexpr int PIECES = DV / 8;
    const int all = (1 << groups) - 1;
    const int lane = threadIdx.x & 63;
    bool found = false;
#pragma unroll 1
    for (Walk at(p.runs, it, w); at.more(); at.step(nw)) {
        if ((at.bits & all) == all && !((at.bits >> 4) & all)) continue;
        Pages pages;
        pages.ask(p, it, at.tile());
        const Place pl(p, p.k + it.kvh * p.k_head, p.v + it.kvh * p.v_head + vcol * 2, it.L, pages);
#pragma unroll 1
        for (int i = lane; i < TK * PIECES; i += 64) {
            int r = i / PIECES;
            r = r < pl.last ? r : pl.last;
            const s16x8 x = *(const s16x8*)((r >= 16 ? pl.v1 : pl.v0) + (r & 15) * (unsigned long long)p.v_row + (i % PIECES) * 16);
#pragma unroll
            for (int k = 0; k < 8; k++) found |= (x[k] & 0x7f80) == 0x7f80;
        }
    }
    return __builtin_amdgcn_ballot_w64(found) != 0;
}

// One row of an item by a whole wave, from memory: what a workgroup falls back to for all its rows where a result is not finite.  A key's values are
// touched only where the row sees the key.  ml: the row's reference and sum as the workgroup of the output's other dims has them, which need not fall back (its
// values may be finite): a piece of a row has one reference for all dims.  (Values do not go into either: this workgroup's tile loop found the same.)
template <int D, int DV, bool CAP>
__device__ void slow_row(const Params& p, const PagedItem& it, int j, int vcol, const float2* ml = nullptr) {
    constexpr int VEC = DV / 64;   // output dims per lane
    const int lane = threadIdx.x & 63, m = lane & 31, g = lane >> 5;
    const int c = it.L - it.T, tok = (it.row0 + j) / p.group, head = it.kvh * p.group + (it.row0 + j - tok * p.group);
    const __bf16* q = p.q + (long)(it.cu + tok) * p.q_tok + (long)head * p.q_head + g * (D / 2);
    const int qpos = p.window && p.pos ? p.pos[it.cu + tok] : c + tok;
    float o[VEC], M = -INFINITY, l = 0.f;
#pragma unroll
    for (int x = 0; x < VEC; x++) o[x] = 0.f;
#pragma unroll 1
    for (Walk at(p.runs, it, 0); at.more(); at.step(1)) {
        Pages pages;
        pages.ask(p, it, at.tile());
        const Place pl(p, p.k + it.kvh * p.k_head, p.v + it.kvh * p.v_head, it.L, pages);
        const int r = m < pl.last ? m : pl.last, u = at.tile() * TK + m - c;
        const bool fresh = p.end && u >= 0 && u < it.T;
        bool vis = u <= tok && m <= pl.last;
        if (fresh) vis = vis && it.cu + tok < p.end[it.cu + u];
        if (p.window) vis = vis && qpos - (fresh ? p.pos[it.cu + u] : at.tile() * TK + m) < p.window;
        // lane (m, g): half g of the dims of key m
        const __bf16* kr = (const __bf16*)((r >= 16 ? pl.k1 : pl.k0) + (r & 15) * p.k_row) + g * (D / 2);
        float s = 0.f;
#pragma unroll 1
        for (int d = 0; d < D / 2; d += 8) {
            const bf16x8 a = *(const bf16x8*)(q + d), b = *(const bf16x8*)(kr + d);
#pragma unroll
            for (int x = 0; x < 8; x++) s = __builtin_fmaf((float)a[x], (float)b[x], s);
        }
        s = lane32_sum(s);
        const float t = vis ? (CAP ? p.cap.of(s) : s) * p.cap.unit : -INFINITY;
        float mx = t;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
        const float mn = fmaxf(M, mx), ms = mn == -INFINITY ? 0.f : mn, alpha = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(M - ms);
        const float pr = __builtin_amdgcn_exp2f(t - ms);
        M = mn;
        float sum = pr;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor(sum, d);
        l = l * alpha + sum;
#pragma unroll
        for (int x = 0; x < VEC; x++) o[x] *= alpha;
        unsigned see = (unsigned)__builtin_amdgcn_ballot_w64(vis);
#pragma unroll 1
        while (see) {
            const int key = __builtin_ctz(see);
            see &= see - 1;
            const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pr), key));
            const __bf16* vr = (const __bf16*)((key >= 16 ? pl.v1 : pl.v0) + (key & 15) * p.v_row) + vcol + VEC * lane;
#pragma unroll
            for (int x = 0; x < VEC; x++) o[x] = __builtin_fmaf(w, (float)vr[x], o[x]);
        }
    }
    if (it.part >= 0) {
        float* dst = p.part_o + (long)(it.part + j) * D + vcol + VEC * lane;
        const float2 piece = ml ? *ml : make_float2(M, l);
        const float f = M == -INFINITY || piece.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(M - piece.x);
#pragma unroll
        for (int x = 0; x < VEC; x++) dst[x] = o[x] * f;
        if (lane == 0 && vcol == 0) p.part_ml[it.part + j] = piece;
    } else {
        __bf16* dst = p.out + (long)(it.cu + tok) * p.o_tok + (long)head * p.o_head + vcol + VEC * lane;
        const float inv = inverse(l);
#pragma unroll
        for (int x = 0; x < VEC; x++) dst[x] = (__bf16)(o[x] * inv);
        if (p.lse && lane == 0 && vcol == 0) p.lse[(long)(it.cu + tok) * p.hq + head] = log_sum(M, l);
    }
}

// ------------------------------------------------------------------------------------------------ waves that share rows and divide the keys
template <int D, int DV, int NW, bool CAP>
__global__ __launch_bounds__(64 * NW, D >= 256 ? 1 : 2) void paged_wave_kernel(const Params p) {
    using R = Rows<D, DV, CAP>;
    using GK = typename R::GK;
    using GV = typename R::GV;
    constexpr int TILE = GK::KTILEB + GV::VTILEB + 512;
    constexpr int OROW = DV + 4;   // floats of a row of the exchange (16 bytes of padding: rows of neighbouring lanes fall on other banks)
    constexpr int LDS = NW * TILE > NW * 32 * OROW * 4 ? NW * TILE : NW * 32 * OROW * 4;
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    __shared__ float2 ml[NW][32];
    int b = blockIdx.x;
    int vcol = 0;
    if (DV < D) {   // (the workgroups of the two halves run on one XCD, close in time, and read the keys through one L2)
        vcol = ((b >> 3) & 1) * DV;
        b = (b >> 4) * 8 + (b & 7);
        if (b >= p.n_items) return;
    }
    const PagedItem it = load_item(p.items, b);
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = it.L - it.T;
    char* const kb = lds + w * TILE;
    char* const vb = kb + GK::KTILEB;
    int* const meta = (int*)(vb + GV::VTILEB);
    const unsigned k_at = lds_addr(kb), v_at = lds_addr(vb), m_at = lds_addr(meta);
    constexpr int NK = GK::NREG, NV = GV::NREG;
    const char* const k_base = p.k + it.kvh * p.k_head;
    const char* const v_base = p.v + it.kvh * p.v_head + vcol * 2;

    R rows;
    bool tree = false, seen_mask = false;
    {
        Walk at(p.runs, it, w);
        const auto is_tree = [&](const Walk& x) { return p.end != nullptr && (x.bits & 16) && x.tile() * TK + TK > c; };
        Pages pages;
        if (at.more()) {   // (the first tile is asked for ahead of the queries: their latencies pass together)
            pages.ask(p, it, at.tile());
            const Place pl(p, k_base, v_base, it.L, pages);
            const int lane = lane_now();
            tree = is_tree(at);
            if (tree) fetch_meta(p, it, at.tile(), m_at, lane);
            fetch<D, NK, GK::KRS>(pl.k0, pl.k1, p.k_row, pl.last, 0, k_at, lane);
            fetch<DV, NV, GV::VRS>(pl.v0, pl.v1, p.v_row, pl.last, 0, v_at, lane);
        }
        rows.load(p, it, it.row0);
        rows.reset();
        while (at.more()) {
            const int kt = at.tile();
            const bool masked = at.bits & 16;
            seen_mask |= masked;
            at.step(NW);
            const bool next = at.more();
            if (next) pages.ask(p, it, at.tile());
            const bool next_tree = next && is_tree(at);
            f32x16 s;
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(NV));   // the keys (and ends, positions) are there; the values may still be on their way
            __builtin_amdgcn_sched_barrier(0);
            rows.scores(kb, s);
            if (CAP) p.cap.of(s);
            if (masked) rows.mask(p, it, kt, meta, tree, s);
            __builtin_amdgcn_s_waitcnt(LGKM0);           // nothing reads the tile's keys any more
            __builtin_amdgcn_sched_barrier(0);
            const Place pl(p, k_base, v_base, it.L, pages);
            if (next) {
                if (next_tree) fetch_meta(p, it, at.tile(), m_at, rows.lane);
                fetch<D, NK, GK::KRS>(pl.k0, pl.k1, p.k_row, pl.last, 0, k_at, rows.lane);
            }
            bf16x8 pb[2];
            rows.softmax(p, s, pb);
            if (!next) __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            else if (next_tree) __builtin_amdgcn_s_waitcnt(vmcnt_imm(NK + 2));
            else __builtin_amdgcn_s_waitcnt(vmcnt_imm(NK));
            __builtin_amdgcn_sched_barrier(0);
            rows.values(vb, pb);
            __builtin_amdgcn_s_waitcnt(LGKM0);
            __builtin_amdgcn_sched_barrier(0);
            if (next) fetch<DV, NV, GV::VRS>(pl.v0, pl.v1, p.v_row, pl.last, 0, v_at, rows.lane);
            tree = next_tree;
        }
    }
    // ---- join the waves: every wave leaves its references and sums, then its accumulators scaled to the largest reference
    const int left = it.T * p.group - it.row0;   // rows from this group's first on
    const float sum = lane32_sum(rows.l);
    if (sum == 0.f) rows.M = -INFINITY;   // no key seen
    if (rows.g == 0) ml[w][rows.m] = make_float2(rows.M, sum);
    const bool again = __syncthreads_or(seen_mask && rows.spoilt(left)) && __syncthreads_or(rubbish<DV>(p, it, vcol, w, NW, 1));
    __syncthreads();   // (and every wave is done with its tiles)
    const auto joined = [&](int row) __attribute__((always_inline)) {   // a row's reference and sum
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int x = 0; x < NW; x++) top = fmaxf(top, ml[x][row].x);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int x = 0; x < NW; x++) total += ml[x][row].y * (NW == 1 || ml[x][row].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[x][row].x - ref));
        return make_float2(top, total);
    };
    if (again) {
        for (int j = w; j < 32 && j < left; j += NW) {
            const float2 state = joined(j);
            slow_row<D, DV, CAP>(p, it, j, vcol, &state);
        }
        return;
    }
    const float2 state = joined(rows.m);
    const float top = state.x, total = state.y, ref = top == -INFINITY ? 0.f : top;
    const float mine = NW == 1 || rows.M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(rows.M - ref);
    const float f = it.part < 0 ? mine * inverse(total) : mine;
    float* const stage = (float*)lds;
#pragma unroll
    for (int dt = 0; dt < R::NDT; dt++)
#pragma unroll
        for (int i4 = 0; i4 < 4; i4++)
            *(float4*)(stage + (w * 32 + rows.m) * OROW + 32 * dt + 8 * i4 + 4 * rows.g) =
                make_float4(rows.o[dt][4 * i4] * f, rows.o[dt][4 * i4 + 1] * f, rows.o[dt][4 * i4 + 2] * f, rows.o[dt][4 * i4 + 3] * f);
    if (w == 0 && rows.g == 0 && rows.m < left && vcol == 0) {
        if (it.part >= 0) p.part_ml[it.part + rows.m] = make_float2(top, total);
        else if (p.lse) p.lse[row_head(p, it, it.row0 + rows.m)] = log_sum(top, total);
    }
    __syncthreads();
    const int here = left < 32 ? left : 32;
    constexpr int PIECES = DV / 8;
    for (int i = threadIdx.x; i < here * PIECES; i += 64 * NW) {
        const int j = i / PIECES, d = (i - j * PIECES) * 8;
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = stage[j * OROW + d + k];
#pragma unroll
        for (int y = 1; y < NW; y++)
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] += stage[(y * 32 + j) * OROW + d + k];
        if (it.part >= 0) {
            float* dst = p.part_o + (long)(it.part + j) * D + vcol + d;
            *(float4*)dst = make_float4(x[0], x[1], x[2], x[3]);
            *(float4*)(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            const int row = it.row0 + j, tok = row / p.group, head = it.kvh * p.group + (row - tok * p.group);
            bf16x8 y;
#pragma unroll
            for (int k = 0; k < 8; k++) y[k] = (__bf16)x[k];
            *(bf16x8*)(p.out + (long)(it.cu + tok) * p.o_tok + (long)head * p.o_head + vcol + d) = y;
        }
    }
}

// ------------------------------------------------------------------------------------------------ waves with rows of their own on the same tiles
// What the tile loop needs of WIN tiles of an item, found by a thread per tile: where their halves lie, which tile it is and its bits.  Found tile by tile
// with scalar arithmetic, this was 75 of the 110 scalar instructions of a tile, most of them in one wave's way (two documents of 8k new on 8k stored tokens,
// 32 / 16 x 128: 3,554 us).
template <int WIN>
struct Window {
    unsigned long long k[WIN][2], v[WIN][2];
    int2 tile[WIN];   // tile, bits
};
template <int WIN>
__device__ __forceinline__ void fill(Window<WIN>& win, const Params& p, const PagedItem& it, int from, const char* kb, const char* vb) {
    const int i = from + (int)threadIdx.x;
    int kt = 0, bits = 0;
    for (int r = 0; r < it.runs; r++) {
        const int* run = (const int*)(p.runs + it.first + r);
        const int start = sload(run, 3);
        if (i >= start) {
            kt = sload(run, 0) + i - start;
            bits = sload(run, 2);
        }
    }
    if ((int)threadIdx.x < WIN && i < it.tiles) {
        const int n = 2 * kt, end = (it.L - 1) >> 4, n1 = n + 1 < end ? n + 1 : end, a = p.page.of(n), b = p.page.of(n1);
        const unsigned ia = p.table[it.tab + a], ib = p.table[it.tab + b], ra = (n - a * p.page.d) * 16, rb = (n1 - b * p.page.d) * 16;
        const int t = threadIdx.x;
        win.k[t][0] = (unsigned long long)kb + (unsigned long long)ia * p.k_page + (unsigned long long)ra * p.k_row;
        win.k[t][1] = (unsigned long long)kb + (unsigned long long)ib * p.k_page + (unsigned long long)rb * p.k_row;
        win.v[t][0] = (unsigned long long)vb + (unsigned long long)ia * p.v_page + (unsigned long long)ra * p.v_row;
        win.v[t][1] = (unsigned long long)vb + (unsigned long long)ib * p.v_page + (unsigned long long)rb * p.v_row;
        win.tile[t] = make_int2(kt, bits);
    }
}

//
// 512 dims: two waves share 32 rows, each with one half of the dims (H = 2) of queries, keys, values and outputs, as a wave of 256 dims has them.  Their
// scores are exchanged through the place of the tile's keys, which nobody reads any more, and added: both then hold the same bits and the same softmax.
// (Two documents of 8,192 new on 8,192 stored, 16 heads on 1: 8.26 ms, 798 TFLOP/s; with all scores in both halves, each a workgroup of its own, 12.99 ms.)
template <int D, int DV, bool CAP>
__global__ __launch_bounds__(256 * (D / DV), DV == 256 ? 2 : 3) void paged_block_kernel(const Params p) {
    constexpr int H = D / DV;
    using R = Rows<DV, DV, CAP>;
    using GK = typename R::GK;
    using GV = typename R::GV;
    constexpr int HALF = GK::KTILEB + GV::VTILEB + 512, BUF = H * HALF;
    constexpr int OROW = DV * 2 + 16;   // bytes of an output row in LDS
    constexpr int LDS = 2 * BUF > H * 4 * 32 * OROW ? 2 * BUF : H * 4 * 32 * OROW;
    constexpr int NK = GK::NREG / 4, NV = GV::NREG / 4;
    constexpr int WIN = 128;
    static_assert(NK * 4 == GK::NREG && NV * 4 == GV::NREG, "a tile's regions must divide among the four waves");
    static_assert((D == 256 ? 2 : 1) * (LDS + sizeof(Window<WIN>)) <= 160 * 1024, "LDS budget");
    static_assert(H == 1 || 4 * 4096 <= GK::KTILEB, "four waves' scores take the place of a half's keys");
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    __shared__ Window<WIN> win;
    const PagedItem it = load_item(p.items, blockIdx.x);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w = H == 1 ? wave : wave & 3, half = H == 1 ? 0 : wave >> 2, vcol = half * DV;
    const int c = it.L - it.T;
    const char* const k_base = p.k + it.kvh * p.k_head;
    const char* const v_base = p.v + it.kvh * p.v_head;
    fill<WIN>(win, p, it, 0, k_base, v_base);
    R rows;
    const unsigned base = lds_addr(lds) + half * HALF;

    // This lane's place in the regions that its wave copies: rows r + x (x < NK, NV) of the tile, which lie in one half of it
    const auto k_row = [&](int lane) { return w * NK + GK::NREG * (lane / GK::CPR); };
    const auto v_row = [&](int lane) { return w * NV + GV::NREG * (lane / GV::CPR); };
    const auto issue = [&](int i, int kt, int bits, int buf) __attribute__((always_inline)) {
        const unsigned at = base + buf * BUF;
        if (kt * TK + TK <= it.L) {
            const int lane = D >= 256 ? lane_now() : threadIdx.x & 63;   // (256 dims: what depends on the lane alone would be spilled, and reloaded in front of every request)
            const char* ka = (const char*)win.k[i][k_row(lane) >> 4] + ((unsigned)(k_row(lane) & 15) * p.k_row + lane % GK::CPR * 16 + vcol * 2);
            const char* va = (const char*)win.v[i][v_row(lane) >> 4] + ((unsigned)(v_row(lane) & 15) * p.v_row + lane % GV::CPR * 16 + vcol * 2);
#pragma unroll
            for (int x = 0; x < NK; x++, ka += p.k_row) dma16_lane(ka, at + (w * NK + x) * GK::KRS);
#pragma unroll
            for (int x = 0; x < NV; x++, va += p.v_row) dma16_lane(va, at + GK::KTILEB + (w * NV + x) * GV::VRS);
        } else {   // the request's last tile: rows behind the stored keys are the last key's
            const int last = it.L - 1 - kt * TK, lane = lane_now();
#pragma unroll
            for (int x = 0; x < NK; x++) {
                const int r = k_row(lane) + x < last ? k_row(lane) + x : last;
                dma16_lane((const char*)win.k[i][r >> 4] + (r & 15) * (unsigned long long)p.k_row + lane % GK::CPR * 16 + vcol * 2, at + (w * NK + x) * GK::KRS);
            }
#pragma unroll
            for (int x = 0; x < NV; x++) {
                const int r = v_row(lane) + x < last ? v_row(lane) + x : last;
                dma16_lane((const char*)win.v[i][r >> 4] + (r & 15) * (unsigned long long)p.v_row + lane % GV::CPR * 16 + vcol * 2, at + GK::KTILEB + (w * NV + x) * GV::VRS);
            }
        }
        if (wave == 0 && p.end && (bits & 0xf0) && kt * TK + TK > c) fetch_meta(p, it, kt, at + GK::KTILEB + GV::VTILEB, lane_now());
    };

    bool seen_mask = false;
    __syncthreads();
    int kt = 0, bits = 0;
    if (it.tiles > 0) {
        const int2 t = win.tile[0];
        kt = __builtin_amdgcn_readfirstlane(t.x);
        bits = __builtin_amdgcn_readfirstlane(t.y);
        issue(0, kt, bits, 0);   // (ahead of the queries: their latencies pass together)
    }
    rows.load(p, it, it.row0 + 32 * w, vcol);
    rows.reset();
    for (int i = 0, j = 0, buf = 0; i < it.tiles; i++, buf ^= 1) {   // j: tile i's place in the window
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));   // this wave's share of the tile has landed
        __syncthreads();                            // ... and everybody's; the other buffer is free
        if (++j == WIN) {                           // (the window's last tile has been requested)
            j = 0;
            fill<WIN>(win, p, it, i + 1, k_base, v_base);
            __syncthreads();
        }
        int kt_next = 0, bits_next = 0;
        if (i + 1 < it.tiles) {
            const int2 t = win.tile[j];
            kt_next = __builtin_amdgcn_readfirstlane(t.x);
            bits_next = __builtin_amdgcn_readfirstlane(t.y);
            issue(j, kt_next, bits_next, buf ^ 1);
        }
        // A row group that sees nothing of the tile is computed all the same (masked): its wave would wait for the others at the barrier anyway,
        // and a branch around the products makes the compiler keep the accumulators twice (256 dims: 205 registers spilled).
        const bool masked = ((bits >> w) & 17) != 1;
        const bool tree = p.end && (bits & 0xf0) && kt * TK + TK > c;
        seen_mask |= masked;
        char* kb = lds + buf * BUF + half * HALF;
        f32x16 s;
        rows.scores(kb, s);
        if (H == 2) {
            char* const mine = kb + w * 4096 + lane_now() * 16;
            const char* const other = mine + (half ? -HALF : HALF);
            __syncthreads();   // every wave is done with the keys
#pragma unroll
            for (int i4 = 0; i4 < 4; i4++) *(float4*)(mine + i4 * 1024) = make_float4(s[4 * i4], s[4 * i4 + 1], s[4 * i4 + 2], s[4 * i4 + 3]);
            __syncthreads();
#pragma unroll
            for (int i4 = 0; i4 < 4; i4++) {
                const float4 x = *(const float4*)(other + i4 * 1024);
                s[4 * i4] += x.x;
                s[4 * i4 + 1] += x.y;
                s[4 * i4 + 2] += x.z;
                s[4 * i4 + 3] += x.w;
            }
        }
        if (CAP) p.cap.of(s);
        if (masked) rows.mask(p, it, kt, (const int*)(lds + buf * BUF + GK::KTILEB + GV::VTILEB), tree, s);
        bf16x8 pb[2];
        rows.softmax(p, s, pb);
        rows.values(kb + GK::KTILEB, pb);
        kt = kt_next;
        bits = bits_next;
    }
    const int left = it.T * p.group - it.row0 - 32 * w;   // rows from this wave's first on
    // (also the barrier behind which the tile buffers are free)
    if (__syncthreads_or(seen_mask && rows.spoilt(left)) && __syncthreads_or(rubbish<DV>(p, it, vcol, w, 4, left + 32 * w < 128 ? (left + 32 * w + 31) / 32 : 4))) {
        for (int j = w; j < 128 && it.row0 + j < it.T * p.group; j += 4) slow_row<D, DV, CAP>(p, it, j, vcol);
        return;
    }

    const float sum = lane32_sum(rows.l);
    if (sum == 0.f) rows.M = -INFINITY;   // no key seen
    const float f = it.part < 0 ? inverse(sum) : 1.f;
    const int lane = lane_now(), m = lane & 31, g = lane >> 5;
    if (it.part >= 0) {
        if (m >= left) return;
        const long prow = it.part + 32 * w + m;
        if (g == 0 && vcol == 0) p.part_ml[prow] = make_float2(rows.M, sum);
        float* po = p.part_o + prow * D + vcol;
#pragma unroll
        for (int dt = 0; dt < R::NDT; dt++)
#pragma unroll
            for (int i4 = 0; i4 < 4; i4++)
                *(float4*)(po + 32 * dt + 8 * i4 + 4 * g) = make_float4(rows.o[dt][4 * i4], rows.o[dt][4 * i4 + 1], rows.o[dt][4 * i4 + 2], rows.o[dt][4 * i4 + 3]);
        return;
    }
    if (p.lse && g == 0 && m < left && vcol == 0) p.lse[row_head(p, it, it.row0 + 32 * w + m)] = log_sum(rows.M, sum);
    // rows through the wave's own slice of LDS, stored as 16-byte pieces
    char* const stage = lds + wave * 32 * OROW;
#pragma unroll
    for (int dt = 0; dt < R::NDT; dt++)
#pragma unroll
        for (int i4 = 0; i4 < 4; i4++) {
            bf16x4 x;
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = (__bf16)(rows.o[dt][4 * i4 + j] * f);
            *(bf16x4*)(stage + m * OROW + (32 * dt + 8 * i4 + 4 * g) * 2) = x;
        }
    constexpr int PIECES = DV / 8;
#pragma unroll
    for (int k = 0; k < 32 * PIECES / 64; k++) {
        const int i = k * 64 + lane, j = i / PIECES, d = (i - j * PIECES) * 8;
        if (j < left) {
            const int row = it.row0 + 32 * w + j, tok = row / p.group, head = it.kvh * p.group + (row - tok * p.group);
            *(bf16x8*)(p.out + (long)(it.cu + tok) * p.o_tok + (long)head * p.o_head + vcol + d) = *(const bf16x8*)(stage + j * OROW + d * 2);
        }
    }
}

// out = sum_s 2^(M_s - M*) O_s / sum_s 2^(M_s - M*) l_s over a row's pieces.  A workgroup per join and 64 head dims; 16 lanes hold a piece, `share` such groups
// take a row's pieces in turn, each with a reference of its own, and are added up in one fixed order.  Rows of few pieces share a workgroup, a long document's row has
// one for itself.  Bound by the pieces' bytes where rows are many, by one round trip to memory where they are few.
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const Params p) {
    constexpr int SLICES = D / 64, GROUPS = 16;
    __shared__ __attribute__((aligned(16))) float part_sum[GROUPS][64];
    __shared__ float2 part_ml[GROUPS];
    const int slice = blockIdx.x % SLICES;
    const int* jp = (const int*)(p.joins + blockIdx.x / SLICES);
    const int cu = sload(jp, 0), kvh = sload(jp, 1), rows = sload(jp, 3), n = sload(jp, 5), stride = sload(jp, 6), share = sload(jp, 7);
    const int row0 = sload(jp, 2);
    const long part = sload(jp, 4);
    const int group = threadIdx.x >> 4, d = (threadIdx.x & 15) * 4;
    const int j = group / share, piece = group - j * share;
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, top = -INFINITY, total = 0.f;
    // (a piece without a visible key holds zeros, or NaN that stays)
    auto add = [&](const float4& x, float m, float l, float ref) {
        const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - ref);
        acc[0] = __builtin_fmaf(f, x.x, acc[0]);
        acc[1] = __builtin_fmaf(f, x.y, acc[1]);
        acc[2] = __builtin_fmaf(f, x.z, acc[2]);
        acc[3] = __builtin_fmaf(f, x.w, acc[3]);
        total = __builtin_fmaf(f, l, total);
    };
    if (j < rows)
        for (int s0 = piece; s0 < n; s0 += 4 * share) {   // four pieces requested at a time
            float4 x[4];
            float2 ml[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int s = s0 + k * share;
                const long at = part + j + (long)(s < n ? s : s0) * stride;
                x[k] = *(const float4*)(p.part_o + at * D + slice * 64 + d);
                ml[k] = p.part_ml[at];
            }
            float ref = top;
#pragma unroll
            for (int k = 0; k < 4; k++) ref = fmaxf(ref, ml[k].x);   // (a piece asked for twice changes no maximum)
            if (top != -INFINITY) {
                const float f = __builtin_amdgcn_exp2f(top - ref);
                total *= f;
#pragma unroll
                for (int k = 0; k < 4; k++) acc[k] *= f;
            }
            top = ref;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (s0 + k * share < n) add(x[k], ml[k].x, ml[k].y, ref);
        }
    if (share > 1) {
        *(float4*)&part_sum[group][d] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) part_ml[group] = make_float2(top, total);
        __syncthreads();
        if (piece) return;
        const int used = n < share ? n : share;
        const float m0 = top, l0 = total;
        for (int s = 1; s < used; s++) top = fmaxf(top, part_ml[group + s].x);
        total = 0.f;
        const float4 own = make_float4(acc[0], acc[1], acc[2], acc[3]);
        acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
        add(own, m0, l0, top);
        for (int s = 1; s < used; s++) {
            const float2 ml = part_ml[group + s];
            add(*(const float4*)&part_sum[group + s][d], ml.x, ml.y, top);
        }
    }
    if (j >= rows) return;
    const int row = row0 + j, tok = row / p.group, head = kvh * p.group + (row - tok * p.group);
    const float f = inverse(total);
    bf16x4 y;
#pragma unroll
    for (int k = 0; k < 4; k++) y[k] = (__bf16)(acc[k] * f);
    *(bf16x4*)(p.out + (long)(cu + tok) * p.o_tok + (long)head * p.o_head + slice * 64 + d) = y;
    if (p.lse && slice == 0 && d == 0) p.lse[(long)(cu + tok) * p.hq + head] = log_sum(top, total);
}

template <int D, int DV, int NW, bool CAP>
int launch(Params p, const spinf_paged_args* a, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (a->n_block) {
        p.items = (const PagedItem*)a->block;
        p.n_items = (int)a->n_block;
        hipLaunchKernelGGL((paged_block_kernel<D, DV, CAP>), dim3((unsigned)a->n_block), dim3(256 * (D / DV)), 0, s, p);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a->n_wave) {
        p.items = (const PagedItem*)a->wave;
        p.n_items = (int)a->n_wave;
        const int64_t n = D / DV == 2 ? (a->n_wave + 7) / 8 * 16 : a->n_wave;
        hipLaunchKernelGGL((paged_wave_kernel<D, DV, NW, CAP>), dim3((unsigned)n), dim3(64 * NW), 0, s, p);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a->n_joins) {
        hipLaunchKernelGGL((paged_join_kernel<D>), dim3((unsigned)(a->n_joins * (D / 64))), dim3(256), 0, s, p);
        e = hipGetLastError();
    }
    return e == hipSuccess ? SPINF_OK : spinf_fail(SPINF_E_HIP, "paged_attn: launch: %s", hipGetErrorString(e));
}

template <int D, int DV, int NW>
int launch_cap(const Params& p, const spinf_paged_args* a, hipStream_t s) {
    return p.cap.on ? launch<D, DV, NW, true>(p, a, s) : launch<D, DV, NW, false>(p, a, s);
}

}  // namespace

extern "C" int spinf_paged_attn_fwd(const spinf_paged_args* a, void* stream) {
    if (!a) return spinf_fail(SPINF_E_ARG, "paged_attn: null args");
    if (a->n_wave < 0 || a->n_block < 0 || a->n_joins < 0 || a->part_rows < 0 || a->n_wave > (1 << 26) || a->n_block > (1 << 26) || a->n_joins > (1 << 24))
        return spinf_fail(SPINF_E_ARG, "paged_attn: bad item counts");
    if (a->n_wave + a->n_block == 0) return SPINF_OK;
    if (a->hq <= 0 || a->hkv <= 0 || a->hq % a->hkv) return spinf_fail(SPINF_E_ARG, "paged_attn: %d query heads do not group over %d key / value heads", a->hq, a->hkv);
    if (a->page < 16 || a->page % 16 || a->page > (1 << 20)) return spinf_fail(SPINF_E_ARG, "paged_attn: pages of %d keys (a multiple of 16)", a->page);
    if (a->window < 0) return spinf_fail(SPINF_E_ARG, "paged_attn: window %d", a->window);
    if (!(a->scale > 0.f) || !(a->scale < INFINITY) || !(a->softcap >= 0.f) || !(a->softcap < INFINITY))
        return spinf_fail(SPINF_E_ARG, "paged_attn: scale %g must be positive and finite, softcap %g not negative", (double)a->scale, (double)a->softcap);
    if (!a->q || !a->out || !a->k || !a->v || !a->table || !a->runs || (a->n_wave && !a->wave) || (a->n_block && !a->block) || (a->n_joins && !a->joins))
        return spinf_fail(SPINF_E_ARG, "paged_attn: null pointer");
    if ((a->end == nullptr) != (a->pos == nullptr)) return spinf_fail(SPINF_E_ARG, "paged_attn: a tree needs both end and pos");
    for (const void* ptr : {a->q, (const void*)a->out, a->k, a->v, (const void*)a->wave, (const void*)a->block, (const void*)a->runs, (const void*)a->joins})
        if ((uintptr_t)ptr % 16) return spinf_fail(SPINF_E_ARG, "paged_attn: tensors and lists must be 16-byte aligned");
    for (int64_t st : {a->q_tok, a->q_head, a->o_tok, a->o_head, a->k_page, a->k_row, a->k_head, a->v_page, a->v_row, a->v_head})
        if (st % 8) return spinf_fail(SPINF_E_ARG, "paged_attn: strides must be multiples of 8 elements");
    if (a->k_row < 0 || a->v_row < 0 || a->k_row > (1 << 24) || a->v_row > (1 << 24) || a->k_page < 0 || a->v_page < 0 || a->k_page > (1u << 30) || a->v_page > (1u << 30))
        return spinf_fail(SPINF_E_ARG, "paged_attn: strides of the cache must lie in 0 .. 2^24 elements (rows) and 0 .. 2^30 (pages)");   // (32-bit byte counts; 32 rows by 32-bit offsets)
    const int64_t need = a->part_rows * (a->d + 2) * 4;
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || (uintptr_t)a->workspace % 16))
        return spinf_fail(SPINF_E_ARG, "paged_attn: split rows need a 16-byte aligned workspace of %lld bytes", (long long)need);
    Params p = {};
    p.q = (const __bf16*)a->q; p.out = (__bf16*)a->out; p.lse = a->lse;
    p.q_tok = a->q_tok; p.q_head = a->q_head; p.o_tok = a->o_tok; p.o_head = a->o_head;
    p.k = (const char*)a->k; p.v = (const char*)a->v;
    p.k_page = (unsigned)(2 * a->k_page); p.k_row = (unsigned)(2 * a->k_row); p.k_head = 2 * a->k_head;
    p.v_page = (unsigned)(2 * a->v_page); p.v_row = (unsigned)(2 * a->v_row); p.v_head = 2 * a->v_head;
    p.same = a->k_page == a->v_page && a->k_row == a->v_row;
    p.table = a->table; p.end = a->end; p.pos = a->pos;
    p.runs = (const PagedRun*)a->runs; p.joins = (const PagedJoin*)a->joins;
    p.part_o = (float*)a->workspace;
    p.part_ml = (float2*)(p.part_o + a->part_rows * a->d);
    p.hq = a->hq; p.group = a->hq / a->hkv;
    p.window = a->window < 1 << 30 ? a->window : 1 << 30;   // (no request is longer; a wider one would leave 32 bits where a tile's first key is subtracted)
    p.page = PageDiv::of_page(a->page);
    if (!SoftCap::of(a->scale, a->softcap, p.cap)) return spinf_fail(SPINF_E_ARG, "paged_attn: scale %g and softcap %g leave fp32's range", (double)a->scale, (double)a->softcap);
    hipStream_t s = (hipStream_t)stream;
    switch (a->d) {
        case 64: return launch_cap<64, 64, 4>(p, a, s);
        case 128: return launch_cap<128, 128, 4>(p, a, s);
        case 256: return launch_cap<256, 256, 4>(p, a, s);   // (as many waves as have tile buffers in 160 KB of LDS; two waves: a request's questions 21.7 us for 15.5)
        case 512: return launch_cap<512, 256, 3>(p, a, s);
        default: return spinf_fail(SPINF_E_ARG, "paged_attn: head dim %d not supported (64, 128, 256, 512)", a->d);
    }
}
