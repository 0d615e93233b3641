// Attention of a decoding step over contents that seats share and over their own keys, for gfx950 (MI355X), from work lists that seats_step.hip leaves in device memory.  No
// counterpart in the reference, whose contents are read anew with every request.
//
// Mathematics.  Row = new token x query head; it sees its content's P stored keys and its seat's own up to its own place: out = (sum_A p v + sum_B p v) / (sum_A p + sum_B p), p =
// exp(t - ref).  The sums over a content's keys are one product per key / value head for all rows that go on below it, so its keys are read once per 128 rows and not once
// per seat; the sums over own keys are made seat by seat; a piece leaves its reference, its sum and its weighted values in 32 bits, and a row's pieces are put together at the end.
// Tiles, products and the softmax of a tile are those of paged_rows.h; a row sees one interval of a span's keys, so a mask is two comparisons.
//
// Kernels (lists of csrc/seats.h):
//   wave    few rows (up to 64 below one content, up to 32 of a seat): four waves (three at 512 dims) divide the tiles, or, where a seat's keys are few, take an item each.
//   block   many rows: four waves with 32 rows each on shared double-buffered tiles.
//   finish  in steps of many such: one token on few keys of its own, which then adds what its content's pieces left; the pieces of all other rows; rows behind the step's last become zeros.
// The lists' lengths are known on the GPU alone: grids have a bounded size and walk the lists.  A list without items costs 3 to 5 us of a launch.
//
// What bounds it.  24 answers below 301 tokens, 18 us: latency, three launches of one short item to a place each.  24 x 56 branches of one token on 470 + 9 keys, 77 us: the keys
// alone would be 40 us, pieces written and read again are half as much.  48 answers below 65,536 tokens, 161 us (0.48 PFLOP/s), and 35 questions of 150 tokens in a window of 1,024, 170 us (0.52): a
// set's last block is mostly empty (288 and 300 rows are three blocks of 128: a third of all tiles are computed for 11 and 15 % of the rows), and a workgroup whose waves have no rows takes as long over a tile as a full one;
// then the turns of a tile's products and its softmax.  The matrix unit is busy 30 % of the time; the same tiles and registers in paged_attn.hip's blocks, all of them full, keep it busy for 54 %.
// At 256 dims two waves to a SIMD are all that fit: with 64 rows to a wave the accumulators spill, and eight waves
// on the same tiles (four buffers) go in step, with nothing beside the softmax to feed the matrix unit: 146 for 129 us of the block kernel, 279 for 191.
//
// Keys that a row does not see leave no trace: as in paged_attn.hip, a workgroup that masked some tile and holds a result that is not finite looks whether masked tiles hold such
// values, and if so computes its rows one by one over the keys they see.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "spinf_tree.h"
#include "common.h"
#include "seats.h"
#include "attn_tiles.h"
#include "paged_dev.h"
#include "paged_rows.h"
#include "lanes.h"

namespace {

struct Params {
    const __bf16* q; __bf16* out; float* lse;
    long q_tok, q_head, o_tok, o_head;
    const char* k; const char* v;
    unsigned k_page, k_row, v_page, v_row; long k_head, v_head;   // bytes
    bool same;                                                    // keys and values have the same strides
    const int* lists; const int* first; const int* pos; const int* counts; const int* parts;
    const SeatItem* wave; const SeatItem* single; const SeatItem* block; const SeatLast* last;
    float* part_o; float2* part_ml;
    int hq, hkv, group, window, rows, seats, last_blocks, join_x, join_y;
    int room[4];   // (the lists hold no more than they have room for, whatever their counts say)
    PageDiv page;
    Div by_group, by_heads;
    SoftCap cap;
};

struct Item { int tok0, T, row0, piece, only; };
struct Span { int tab, L, kt0, tiles, flo, fhi, own; };
__device__ __forceinline__ Item load_item(const SeatItem* items, int i) {
    const int* p = (const int*)(items + i);
    return {sload(p, 0), sload(p, 1), sload(p, 2), sload(p, 3), sload(p, 4)};
}
// (a step of more rows than the call's tensors have does not go with them: its lists are not walked, and all rows become NaN)
__device__ __forceinline__ int tokens_of(const Params& p) { return sload(p.first, p.seats); }
__device__ __forceinline__ Span load_span(const SeatItem* items, int i, int which) {
    const int* p = (const int*)(items + i) + 8 + 8 * which;
    return {sload(p, 0), sload(p, 1), sload(p, 2), sload(p, 3), sload(p, 4), sload(p, 5), sload(p, 6)};
}
// (pins an item's loads where they are asked for: beside the list's count and not behind it.  There is room for an item of that index, whatever it holds.)
__device__ __forceinline__ void asked(int count, int tokens, const Item& a, const Span& b) {
    asm volatile("" ::"s"(count), "s"(tokens), "s"(a.tok0), "s"(a.T), "s"(a.row0), "s"(a.piece), "s"(a.only), "s"(b.tab), "s"(b.L), "s"(b.kt0), "s"(b.tiles), "s"(b.flo), "s"(b.fhi), "s"(b.own));
}
__device__ __forceinline__ bool is_masked(const Span& s, int kt) { return kt * TK < s.flo || kt * TK + TK - 1 > s.fhi; }

// Where a tile lies: byte addresses of row 0 and row 16 of the key / value head's keys and values, and the tile's last stored row.  The pages are asked for a tile ahead.
struct Pages {
    int n, row0, row1, id0, id1;
    __device__ __forceinline__ void ask(const Params& p, const Span& s, int kt) {
        n = 2 * kt;
        const int a = p.page.of(n);
        id0 = sload(p.lists, s.tab + a);
        row0 = (n - a * p.page.d) * 16;
        if (p.page.d & 1) {
            const int end = (s.L - 1) >> 4, n1 = n + 1 < end ? n + 1 : end, b = p.page.of(n1);
            id1 = sload(p.lists, s.tab + b);
            row1 = (n1 - b * p.page.d) * 16;
        }
    }
};
struct Place {
    const char *k0, *k1, *v0, *v1;
    int last;
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

// the keys lo .. hi of the span that token t of the item's set sees
__device__ __forceinline__ void interval(const Params& p, const Item& it, const Span& s, int t, int& lo, int& hi) {
    const int at = s.L - it.T + t;   // its own place (of a seat's own keys)
    hi = s.own ? at : s.L - 1;
    lo = p.window ? (s.own ? at : p.pos[it.tok0 + t]) - p.window + 1 : INT_MIN;
}

// A wave's 32 rows, and the keys that they see
template <int D, int DV, bool CAP>
struct Rows : RowTile<D, DV, CAP> {
    using B = RowTile<D, DV, CAP>;
    using B::qf, B::lane, B::m, B::g, B::NS;
    int lo, hi;

    __device__ __forceinline__ void see(const Params& p, const Item& it, const Span& s, int row0) {
        const int N = it.T * p.group, row = row0 + (lane_now() & 31), r = row < N ? row : N - 1;
        interval(p, it, s, p.by_group.of(r), lo, hi);
    }
    // queries of rows row0 + m, dims col ..
    __device__ __forceinline__ void load(const Params& p, const Item& it, const Span& s, int kvh, int row0, int col = 0) {
        lane = threadIdx.x & 63;
        m = lane & 31;
        g = lane >> 5;
        const int N = it.T * p.group, row = row0 + m, r = row < N ? row : N - 1;
        const int tok = p.by_group.of(r), head = kvh * p.group + (r - tok * p.group);
        const __bf16* qp = p.q + (long)(it.tok0 + tok) * p.q_tok + (long)head * p.q_head + col + 8 * g;
#pragma unroll
        for (int s = 0; s < NS; s++) qf[s] = *(const bf16x8*)(qp + 16 * s);
        interval(p, it, s, tok, lo, hi);
        // (waited for here: left to the compiler, the wait would sit at the first use inside the tile loop, behind the DMAs in flight)
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
#pragma unroll
        for (int s = 0; s < NS; s++) asm volatile("" : "+v"(qf[s]));
        asm volatile("" : "+v"(lo), "+v"(hi));
    }
    __device__ __forceinline__ void mask(int kt, f32x16& s) {
        const int key = kt * TK + 4 * g;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int x = key + 8 * (i >> 2) + (i & 3);
            s[i] = ((x >= lo) & (x <= hi)) ? s[i] : -INFINITY;
        }
    }
};

__device__ __forceinline__ void token_head(const Params& p, const Item& it, int kvh, int row, int& tok, int& head) {
    const int t = p.by_group.of(row);
    tok = it.tok0 + t;
    head = kvh * p.group + (row - t * p.group);
}
__device__ __forceinline__ long part_of(const Params& p, const Item& it, int tok, int head) { return (long)((p.parts[tok] & INT_MAX) + it.piece) * p.hq + head; }

// Do masked tiles of an item hold values that are not finite?  A wave looks at tiles w, w + nw ..
template <int DV>
__device__ bool rubbish(const Params& p, const Span& it, int kvh, int vcol, int w, int nw) {
    constexpr int PIECES = DV / 8;
    const int lane = threadIdx.x & 63;
    bool found = false;
#pragma unroll 1
    for (int i = w; i < it.tiles; i += nw) {
        if (!is_masked(it, it.kt0 + i)) continue;
        Pages pages;
        pages.ask(p, it, it.kt0 + i);
        const Place pl(p, p.k + kvh * p.k_head, p.v + kvh * p.v_head + vcol * 2, it.L, pages);
#pragma unroll 1
        for (int j = lane; j < TK * PIECES; j += 64) {
            int r = j / PIECES;
            r = r < pl.last ? r : pl.last;
            const s16x8 x = *(const s16x8*)((r >= 16 ? pl.v1 : pl.v0) + (r & 15) * (unsigned long long)p.v_row + (j % PIECES) * 16);
#pragma unroll
            for (int k = 0; k < 8; k++) found |= (x[k] & 0x7f80) == 0x7f80;
        }
    }
    return __builtin_amdgcn_ballot_w64(found) != 0;
}

// One row of an item by a whole wave, from memory, values touched only where the row sees the key.  state: the row's reference and sum as the tile loop found them: a
// piece has one reference for all dims, also where the workgroup of the others does not come here (its values may be finite).
template <int D, int DV, bool CAP>
__device__ void slow_row(const Params& p, const Item& it, const Span* spans, int n_spans, int kvh, int j, int vcol, const float2 state) {
    constexpr int VEC = DV / 64;   // output dims per lane
    const int lane = threadIdx.x & 63, m = lane & 31, g = lane >> 5;
    int tok, head, lo, hi;
    token_head(p, it, kvh, it.row0 + j, tok, head);
    const __bf16* q = p.q + (long)tok * p.q_tok + (long)head * p.q_head + g * (D / 2);
    const float ref = state.x == -INFINITY ? 0.f : state.x;
    float o[VEC];
#pragma unroll
    for (int x = 0; x < VEC; x++) o[x] = 0.f;
#pragma unroll 1
    for (int x = 0; x < n_spans; x++) {
    const Span& sp = spans[x];
    interval(p, it, sp, tok - it.tok0, lo, hi);
#pragma unroll 1
    for (int i = 0; i < sp.tiles; i++) {
        const int kt = sp.kt0 + i;
        Pages pages;
        pages.ask(p, sp, kt);
        const Place pl(p, p.k + kvh * p.k_head, p.v + kvh * p.v_head, sp.L, pages);
        const int r = m < pl.last ? m : pl.last;
        const bool vis = kt * TK + m >= lo && kt * TK + m <= hi;
        // lane (m, g): half g of the dims of key m
        const __bf16* kr = (const __bf16*)((r >= 16 ? pl.k1 : pl.k0) + (r & 15) * (unsigned long long)p.k_row) + g * (D / 2);
        float s = 0.f;
#pragma unroll 1
        for (int d = 0; d < D / 2; d += 8) {
            const bf16x8 a = *(const bf16x8*)(q + d), b = *(const bf16x8*)(kr + d);
#pragma unroll
            for (int x = 0; x < 8; x++) s = __builtin_fmaf((float)a[x], (float)b[x], s);
        }
        s = lane32_sum(s);
        const float pr = vis ? __builtin_amdgcn_exp2f(__builtin_fmaf(CAP ? p.cap.of(s) : s, p.cap.unit, -ref)) : 0.f;
        unsigned see = (unsigned)__builtin_amdgcn_ballot_w64(vis);
#pragma unroll 1
        while (see) {
            const int key = __builtin_ctz(see);
            see &= see - 1;
            const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pr), key));
            const __bf16* vr = (const __bf16*)((key >= 16 ? pl.v1 : pl.v0) + (key & 15) * (unsigned long long)p.v_row) + vcol + VEC * lane;
#pragma unroll
            for (int x = 0; x < VEC; x++) o[x] = __builtin_fmaf(w, (float)vr[x], o[x]);
        }
    }
    }
    if (it.only) {
        __bf16* dst = p.out + (long)tok * p.o_tok + (long)head * p.o_head + vcol + VEC * lane;
        const float inv = inverse(state.y);
#pragma unroll
        for (int x = 0; x < VEC; x++) dst[x] = (__bf16)(o[x] * inv);
        if (p.lse && lane == 0 && vcol == 0) p.lse[(long)tok * p.hq + head] = log_sum(state.x, state.y);
    } else {
        const long part = part_of(p, it, tok, head);
        float* dst = p.part_o + part * D + vcol + VEC * lane;
#pragma unroll
        for (int x = 0; x < VEC; x++) dst[x] = o[x];
        if (lane == 0 && vcol == 0) p.part_ml[part] = state;
    }
}

// eight dims of a row, as the last word or as a piece
template <int D>
__device__ __forceinline__ void put8(const Params& p, const Item& it, int tok, int head, int begin, int d, const float (&x)[8]) {
    if (it.only) {
        bf16x8 y;
#pragma unroll
        for (int k = 0; k < 8; k++) y[k] = (__bf16)x[k];
        *(bf16x8*)(p.out + (long)tok * p.o_tok + (long)head * p.o_head + d) = y;
    } else {
        float* dst = p.part_o + ((long)(begin + it.piece) * p.hq + head) * D + d;
        *(float4*)dst = make_float4(x[0], x[1], x[2], x[3]);
        *(float4*)(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
}
__device__ __forceinline__ void put_sum(const Params& p, const Item& it, int tok, int head, int begin, float M, float sum) {
    if (!it.only) p.part_ml[(long)(begin + it.piece) * p.hq + head] = make_float2(M, sum);
    else if (p.lse) p.lse[(long)tok * p.hq + head] = log_sum(M, sum);
}

// ------------------------------------------------------------------------------------------------ a seat's own keys
template <int D, int DV, int NW, bool CAP>
__global__ __launch_bounds__(64 * NW, D >= 256 ? 1 : 2) void seats_wave_kernel(const Params p) {
    using R = Rows<D, DV, CAP>;
    using GK = typename R::GK;
    using GV = typename R::GV;
    constexpr int OROW = DV + 4;   // floats of a row of the exchange (16 bytes of padding: rows of neighbouring lanes fall on other banks)
    constexpr int TILE = GK::KTILEB + GV::VTILEB > 32 * OROW * 4 ? GK::KTILEB + GV::VTILEB : 32 * OROW * 4;   // a wave's rows take the place of its tile
    __shared__ __attribute__((aligned(16))) char lds[NW * TILE];
    __shared__ float2 ml[NW][32];
    __shared__ int part_of_row[NW][32];   // where the rows' pieces begin
    constexpr int NK = GK::NREG, NV = GV::NREG;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char* const kb = lds + w * TILE;
    char* const vb = kb + GK::KTILEB;
    const unsigned k_at = lds_addr(kb), v_at = lds_addr(vb);
    // (the first item, if it is one for all waves)
    const int first_unit = DV < D ? (blockIdx.x >> 4) * 8 + (blockIdx.x & 7) : blockIdx.x, first_item = seats_least(p.by_heads.of(first_unit), p.room[0] - 1);
    const int count = sload(p.counts, 0), singles = sload(p.counts, 1), tokens = tokens_of(p);
    const Item item0 = load_item(p.wave, first_item);
    const Span span0 = load_span(p.wave, first_item, 0);
    asked(count, tokens, item0, span0);
    const bool right = tokens <= p.rows;
    const int shared = right ? seats_least(count, p.room[0]) * p.hkv : 0, alone = right ? seats_least(singles, p.room[1]) * p.hkv : 0;
    const int units = shared + (alone + NW - 1) / NW;
    const int last_unit = DV < D ? (units + 7) / 8 * 16 : units;
    for (int u = blockIdx.x; u < last_unit; u += gridDim.x) {
        int unit = u, vcol = 0;
        if (DV < D) {   // (the workgroups of the two halves run on one XCD, close in time, and read the keys through one L2)
            vcol = ((u >> 3) & 1) * DV;
            unit = (u >> 4) * 8 + (u & 7);
            if (unit >= units) continue;
        }
        const bool single = unit >= shared;
        const int x = single ? (unit - shared) * NW + w : unit;
        if (single && x >= alone) continue;   // (waves of these items meet nowhere: only the last unit of a workgroup's walk has idle ones)
        const int item = p.by_heads.of(x), kvh = x - item * p.hkv;
        const SeatItem* const list = single ? p.single : p.wave;
        const bool known = !single && u == (int)blockIdx.x;
        const Item it = known ? item0 : load_item(list, item);
        const Span span = known ? span0 : load_span(list, item, 0);
        const char* const k_base = p.k + kvh * p.k_head;
        const char* const v_base = p.v + kvh * p.v_head + vcol * 2;
        const int step = single ? 1 : NW;
        R rows;
        bool seen_mask = false;
        int kt = span.kt0 + (single ? 0 : w);
        const int end = span.kt0 + span.tiles;
        {
            Pages pages;
            if (kt < end) {   // (the first tile is asked for ahead of the queries: their latencies pass together)
                pages.ask(p, span, kt);
                const Place pl(p, k_base, v_base, span.L, pages);
                const int lane = lane_now();
                fetch<D, NK, GK::KRS>(pl.k0, pl.k1, p.k_row, pl.last, 0, k_at, lane);
                fetch<DV, NV, GV::VRS>(pl.v0, pl.v1, p.v_row, pl.last, 0, v_at, lane);
            }
            rows.load(p, it, span, kvh, it.row0);
            rows.reset();
            if (rows.g == 0 && !it.only) {   // (asked for here: at the end they would be one more wait for memory)
                const int N = it.T * p.group, row = it.row0 + rows.m;
                part_of_row[w][rows.m] = p.parts[it.tok0 + p.by_group.of(row < N ? row : N - 1)] & INT_MAX;
            }
            while (kt < end) {
                const bool masked = is_masked(span, kt), next = kt + step < end;
                seen_mask |= masked;
                if (next) pages.ask(p, span, kt + step);
                f32x16 s;
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(NV));   // the keys are there; the values may still be on their way
                __builtin_amdgcn_sched_barrier(0);
                rows.scores(kb, s);
                if (CAP) p.cap.of(s);
                if (masked) rows.mask(kt, s);
                __builtin_amdgcn_s_waitcnt(LGKM0);           // nothing reads the tile's keys any more
                __builtin_amdgcn_sched_barrier(0);
                const Place pl(p, k_base, v_base, span.L, pages);
                if (next) fetch<D, NK, GK::KRS>(pl.k0, pl.k1, p.k_row, pl.last, 0, k_at, rows.lane);
                bf16x8 pb[2];
                rows.softmax(p.cap, s, pb);
                if (!next) __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
                else __builtin_amdgcn_s_waitcnt(vmcnt_imm(NK));
                __builtin_amdgcn_sched_barrier(0);
                rows.values(vb, pb);
                __builtin_amdgcn_s_waitcnt(LGKM0);
                __builtin_amdgcn_sched_barrier(0);
                if (next) fetch<DV, NV, GV::VRS>(pl.v0, pl.v1, p.v_row, pl.last, 0, v_at, rows.lane);
                kt += step;
            }
        }
        const int left = it.T * p.group - it.row0, here = left < 32 ? left : 32;
        const float sum = lane32_sum(rows.l);
        if (sum == 0.f) rows.M = -INFINITY;   // no key seen
        constexpr int PIECES = DV / 8;
        float* const stage = (float*)lds;
        if (single) {
            if (seen_mask && rows.spoilt(left) && rubbish<DV>(p, span, kvh, vcol, 0, 1)) {
                for (int j = 0; j < here; j++) {
                    const float2 state = make_float2(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(rows.M), j)), __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sum), j)));
                    slow_row<D, DV, CAP>(p, it, &span, 1, kvh, j, vcol, state);
                }
                continue;
            }
            const float f = it.only ? inverse(sum) : 1.f;
            float* const mine = (float*)kb;
            if (rows.m < left) {
#pragma unroll
                for (int dt = 0; dt < R::NDT; dt++)
#pragma unroll
                    for (int i4 = 0; i4 < 4; i4++)
                        *(float4*)(mine + rows.m * OROW + 32 * dt + 8 * i4 + 4 * rows.g) =
                            make_float4(rows.o[dt][4 * i4] * f, rows.o[dt][4 * i4 + 1] * f, rows.o[dt][4 * i4 + 2] * f, rows.o[dt][4 * i4 + 3] * f);
                if (rows.g == 0 && vcol == 0) {
                    int tok, head;
                    token_head(p, it, kvh, it.row0 + rows.m, tok, head);
                    put_sum(p, it, tok, head, part_of_row[w][rows.m], rows.M, sum);
                }
            }
            __builtin_amdgcn_wave_barrier();   // (LDS operations of a wave are done in order)
            for (int i = rows.lane; i < here * PIECES; i += 64) {
                const int j = i / PIECES, d = (i - j * PIECES) * 8;
                int tok, head;
                token_head(p, it, kvh, it.row0 + j, tok, head);
                float y[8];
#pragma unroll
                for (int k = 0; k < 8; k++) y[k] = mine[j * OROW + d + k];
                put8<D>(p, it, tok, head, part_of_row[w][j], vcol + d, y);
            }
            __builtin_amdgcn_s_waitcnt(LGKM0);   // (the next item's tile comes here)
            __builtin_amdgcn_sched_barrier(0);
            continue;
        }
        // ---- join the waves: every wave leaves its references and sums, then its accumulators scaled to the largest reference
        if (rows.g == 0) ml[w][rows.m] = make_float2(rows.M, sum);
        const bool again = __syncthreads_or(seen_mask && rows.spoilt(left)) && __syncthreads_or(rubbish<DV>(p, span, kvh, vcol, w, NW));
        __syncthreads();   // (and every wave is done with its tiles)
        const auto joined = [&](int row) __attribute__((always_inline)) {   // a row's reference and sum
            float top = -INFINITY, total = 0.f;
#pragma unroll
            for (int y = 0; y < NW; y++) top = fmaxf(top, ml[y][row].x);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int y = 0; y < NW; y++) total += ml[y][row].y * (ml[y][row].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[y][row].x - ref));
            return make_float2(top, total);
        };
        if (again) {
            for (int j = w; j < here; j += NW) slow_row<D, DV, CAP>(p, it, &span, 1, kvh, j, vcol, joined(j));
            __syncthreads();
            continue;
        }
        const float2 state = joined(rows.m);
        const float ref = state.x == -INFINITY ? 0.f : state.x;
        const float f = (rows.M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(rows.M - ref)) * (it.only ? inverse(state.y) : 1.f);
        if (rows.m < left) {
#pragma unroll
            for (int dt = 0; dt < R::NDT; dt++)
#pragma unroll
                for (int i4 = 0; i4 < 4; i4++)
                    *(float4*)(stage + (w * 32 + rows.m) * OROW + 32 * dt + 8 * i4 + 4 * rows.g) =
                        make_float4(rows.o[dt][4 * i4] * f, rows.o[dt][4 * i4 + 1] * f, rows.o[dt][4 * i4 + 2] * f, rows.o[dt][4 * i4 + 3] * f);
            if (w == 0 && rows.g == 0 && vcol == 0) {
                int tok, head;
                token_head(p, it, kvh, it.row0 + rows.m, tok, head);
                put_sum(p, it, tok, head, part_of_row[w][rows.m], state.x, state.y);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < here * PIECES; i += 64 * NW) {
            const int j = i / PIECES, d = (i - j * PIECES) * 8;
            int tok, head;
            token_head(p, it, kvh, it.row0 + j, tok, head);
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) y[k] = stage[j * OROW + d + k];
#pragma unroll
            for (int z = 1; z < NW; z++)
#pragma unroll
                for (int k = 0; k < 8; k++) y[k] += stage[(z * 32 + j) * OROW + d + k];
            put8<D>(p, it, tok, head, part_of_row[w][j], vcol + d, y);
        }
        __syncthreads();   // (the next item's tiles come here)
    }
}

// ------------------------------------------------------------------------------------------------ contents, and own keys of many new tokens
// A tile's halves, found by a thread per tile, SPAN tiles at a time
template <int SPAN>
struct Halves { unsigned long long k[SPAN][2], v[SPAN][2]; };
template <int SPAN>
__device__ __forceinline__ void fill(Halves<SPAN>& h, const Params& p, const Span (&span)[2], int from, const char* kb, const char* vb) {
    const int t = threadIdx.x, i = from + t;
    if (t < SPAN && i < span[0].tiles + span[1].tiles) {
        const bool second = i >= span[0].tiles;
        const int kt = second ? span[1].kt0 + i - span[0].tiles : span[0].kt0 + i, L = second ? span[1].L : span[0].L, tab = second ? span[1].tab : span[0].tab;
        const int n = 2 * kt, end = (L - 1) >> 4, n1 = n + 1 < end ? n + 1 : end, a = p.page.of(n), b = p.page.of(n1);
        const unsigned ia = p.lists[tab + a], ib = p.lists[tab + b], ra = (n - a * p.page.d) * 16, rb = (n1 - b * p.page.d) * 16;
        h.k[t][0] = (unsigned long long)kb + (unsigned long long)ia * p.k_page + (unsigned long long)ra * p.k_row;
        h.k[t][1] = (unsigned long long)kb + (unsigned long long)ib * p.k_page + (unsigned long long)rb * p.k_row;
        h.v[t][0] = (unsigned long long)vb + (unsigned long long)ia * p.v_page + (unsigned long long)ra * p.v_row;
        h.v[t][1] = (unsigned long long)vb + (unsigned long long)ib * p.v_page + (unsigned long long)rb * p.v_row;
    }
}

// 512 dims: two waves share 32 rows, each with one half of the dims of queries, keys, values and outputs; their scores are exchanged through the place of the tile's keys,
// which nobody reads any more, and added: both then hold the same bits and the same softmax.
template <int D, int DV, bool CAP>
__global__ __launch_bounds__(256 * (D / DV), DV == 256 ? 2 : 3) void seats_block_kernel(const Params p) {
    constexpr int H = D / DV;
    using R = Rows<DV, DV, CAP>;
    using GK = typename R::GK;
    using GV = typename R::GV;
    constexpr int HALF = GK::KTILEB + GV::VTILEB, BUF = H * HALF;
    constexpr int OROW = DV * 2 + 16;   // bytes of an output row in LDS
    constexpr int LDS = 2 * BUF > H * 4 * 32 * OROW ? 2 * BUF : H * 4 * 32 * OROW;
    constexpr int NK = GK::NREG / 4, NV = GV::NREG / 4;
    constexpr int SPAN = 128;
    static_assert(NK * 4 == GK::NREG && NV * 4 == GV::NREG, "a tile's regions must divide among the four waves");
    static_assert((D == 256 ? 2 : 1) * (LDS + sizeof(Halves<SPAN>)) <= 160 * 1024, "LDS budget");
    static_assert(H == 1 || 4 * 4096 <= GK::KTILEB, "four waves' scores take the place of a half's keys");
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    __shared__ Halves<SPAN> at;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w = H == 1 ? wave : wave & 3, half = H == 1 ? 0 : wave >> 2, vcol = half * DV;
    const unsigned base = lds_addr(lds) + half * HALF;
    const int units = tokens_of(p) <= p.rows ? seats_least(sload(p.counts, 2), p.room[2]) * p.hkv : 0;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int item = p.by_heads.of(unit), kvh = unit - item * p.hkv;
        const Item it = load_item(p.block, item);
        const Span span[2] = {load_span(p.block, item, 0), load_span(p.block, item, 1)};
        const int tiles = span[0].tiles + span[1].tiles;
        const char* const k_base = p.k + kvh * p.k_head;
        const char* const v_base = p.v + kvh * p.v_head;
        fill<SPAN>(at, p, span, 0, k_base, v_base);
        R rows;

        // This lane's place in the regions that its wave copies: rows r + x (x < NK, NV) of the tile, which lie in one half of it
        const auto k_row = [&](int lane) { return w * NK + GK::NREG * (lane / GK::CPR); };
        const auto v_row = [&](int lane) { return w * NV + GV::NREG * (lane / GV::CPR); };
        const auto issue = [&](int i, int last, int buf) __attribute__((always_inline)) {
            const unsigned to = base + buf * BUF;
            const int lane = lane_now();
            if (last >= TK - 1) {
                const char* ka = (const char*)at.k[i][k_row(lane) >> 4] + ((unsigned)(k_row(lane) & 15) * p.k_row + lane % GK::CPR * 16 + vcol * 2);
                const char* va = (const char*)at.v[i][v_row(lane) >> 4] + ((unsigned)(v_row(lane) & 15) * p.v_row + lane % GV::CPR * 16 + vcol * 2);
#pragma unroll
                for (int x = 0; x < NK; x++, ka += p.k_row) dma16_lane(ka, to + (w * NK + x) * GK::KRS);
#pragma unroll
                for (int x = 0; x < NV; x++, va += p.v_row) dma16_lane(va, to + GK::KTILEB + (w * NV + x) * GV::VRS);
            } else {   // the span's last tile: rows behind the stored keys are the last key's
#pragma unroll
                for (int x = 0; x < NK; x++) {
                    const int r = k_row(lane) + x < last ? k_row(lane) + x : last;
                    dma16_lane((const char*)at.k[i][r >> 4] + (r & 15) * (unsigned long long)p.k_row + lane % GK::CPR * 16 + vcol * 2, to + (w * NK + x) * GK::KRS);
                }
#pragma unroll
                for (int x = 0; x < NV; x++) {
                    const int r = v_row(lane) + x < last ? v_row(lane) + x : last;
                    dma16_lane((const char*)at.v[i][r >> 4] + (r & 15) * (unsigned long long)p.v_row + lane % GV::CPR * 16 + vcol * 2, to + GK::KTILEB + (w * NV + x) * GV::VRS);
                }
            }
        };

        bool seen_mask = false;
        __syncthreads();
        // keys of tile i behind its first one
        const auto behind = [&](int i) __attribute__((always_inline)) { return i < span[0].tiles ? span[0].L - 1 - (span[0].kt0 + i) * TK : span[1].L - 1 - (span[1].kt0 + i - span[0].tiles) * TK; };
        if (tiles > 0) issue(0, behind(0), 0);   // (ahead of the queries: their latencies pass together)
        if (it.row0 + 32 * w >= it.T * p.group) {   // a wave without rows brings its share of the tiles
            for (int i = 0, j = 0, buf = 0; i < tiles; i++, buf ^= 1) {
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
                __syncthreads();
                if (++j == SPAN) {
                    j = 0;
                    fill<SPAN>(at, p, span, i + 1, k_base, v_base);
                    __syncthreads();
                }
                if (i + 1 < tiles) issue(j, behind(i + 1), buf ^ 1);
                if (H == 2) {
                    __syncthreads();
                    __syncthreads();
                }
            }
            if (__syncthreads_or(0)) __syncthreads_or(0);
            __syncthreads();
            continue;
        }
        rows.load(p, it, span[0], kvh, it.row0 + 32 * w, vcol);
        rows.reset();
        for (int i = 0, j = 0, buf = 0; i < tiles; i++, buf ^= 1) {   // j: tile i's place among the halves
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));   // this wave's share of the tile has landed
            __syncthreads();                            // ... and everybody's; the other buffer is free
            if (++j == SPAN) {                          // (the last tile of the span in hand has been requested)
                j = 0;
                fill<SPAN>(at, p, span, i + 1, k_base, v_base);
                __syncthreads();
            }
            if (i + 1 < tiles) issue(j, behind(i + 1), buf ^ 1);
            if (i == span[0].tiles) rows.see(p, it, span[1], it.row0 + 32 * w);   // (from here on it is the seat's own keys)
            const bool second = i >= span[0].tiles;
            const int kt = second ? span[1].kt0 + i - span[0].tiles : span[0].kt0 + i;
            const bool masked = second ? is_masked(span[1], kt) : is_masked(span[0], kt);
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
            if (masked) rows.mask(kt, s);
            bf16x8 pb[2];
            rows.softmax(p.cap, s, pb);
            rows.values(kb + GK::KTILEB, pb);
        }
        const int left = it.T * p.group - it.row0 - 32 * w;   // rows from this wave's first on
        const int live = seats_least(4, seats_up(left + 32 * w, 32));   // waves that have rows
        const float sum = lane32_sum(rows.l);
        if (sum == 0.f) rows.M = -INFINITY;   // no key seen
        // (also the barrier behind which the tile buffers are free)
        if (__syncthreads_or(seen_mask && rows.spoilt(left)) && __syncthreads_or(rubbish<DV>(p, span[0], kvh, vcol, w, live) | rubbish<DV>(p, span[1], kvh, vcol, w, live))) {
            for (int j = 0; j < 32 && j < left; j++) {
                const float2 state = make_float2(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(rows.M), j)), __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sum), j)));
                slow_row<D, DV, CAP>(p, it, span, 2, kvh, 32 * w + j, vcol, state);
            }
            __syncthreads();
            continue;
        }
        const float f = it.only ? inverse(sum) : 1.f;
        const int lane = lane_now(), m = lane & 31, g = lane >> 5;
        if (it.only) {   // rows through the wave's own slice of LDS, stored as 16-byte pieces
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
            if (p.lse && g == 0 && m < left && vcol == 0) {
                int tok, head;
                token_head(p, it, kvh, it.row0 + 32 * w + m, tok, head);
                p.lse[(long)tok * p.hq + head] = log_sum(rows.M, sum);
            }
            constexpr int PIECES = DV / 8;
#pragma unroll
            for (int k = 0; k < 32 * PIECES / 64; k++) {
                const int i = k * 64 + lane, j = i / PIECES, d = (i - j * PIECES) * 8;
                if (j < left) {
                    int tok, head;
                    token_head(p, it, kvh, it.row0 + 32 * w + j, tok, head);
                    *(bf16x8*)(p.out + (long)tok * p.o_tok + (long)head * p.o_head + vcol + d) = *(const bf16x8*)(stage + j * OROW + d * 2);
                }
            }
        } else if (m < left) {
            int tok, head;
            token_head(p, it, kvh, it.row0 + 32 * w + m, tok, head);
            const long part = part_of(p, it, tok, head);
            if (g == 0 && vcol == 0) p.part_ml[part] = make_float2(rows.M, sum);
            float* po = p.part_o + part * D + vcol;
#pragma unroll
            for (int dt = 0; dt < R::NDT; dt++)
#pragma unroll
                for (int i4 = 0; i4 < 4; i4++)
                    *(float4*)(po + 32 * dt + 8 * i4 + 4 * g) = make_float4(rows.o[dt][4 * i4], rows.o[dt][4 * i4 + 1], rows.o[dt][4 * i4 + 2], rows.o[dt][4 * i4 + 3]);
        }
        __syncthreads();   // (the next item's tiles and halves come here)
    }
}

// ------------------------------------------------------------------------------------------------ one token on few keys of its own: the last word
// A wave per (seat, key / value head), D / 8 lanes to a key, its dot products in the vector unit: as few keys as these would leave the matrix unit's tiles mostly empty, and without LDS
// four times as many waves run at a time, which is what hides the latency of so little (10,752 items of some nine keys of 256 dims: 95 us as tiles, half of it so; csrc/seats.h has both
// sides' times).
// Probabilities stay 32-bit.  Then the pieces that the content's items left are added, and the row is written.
template <int D, bool CAP>
__device__ __forceinline__ void last_words(const Params& p) {
    constexpr int RM = SEAT_LAST_HEADS, LPK = D / 8, G = 64 / LPK, U = 4;   // heads, lanes of a key, keys of a load, loads ahead
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, mine = lane / LPK, col = lane % LPK * 8;
    // (an item is read a round ahead, the first one beside the count: there is room for it, whatever it holds)
    struct Words { int w[12]; };
    const auto load = [&](int unit) __attribute__((always_inline)) {
        const int* ip = (const int*)(p.last + seats_least(p.by_heads.of(unit), p.room[3] - 1));
        Words x;
#pragma unroll
        for (int i = 0; i < 12; i++) x.w[i] = sload(ip, i);
        return x;
    };
    const int count = sload(p.counts, 3), tokens = tokens_of(p);
    Words next = load(blockIdx.x * 4 + w);
    asm volatile("" ::"s"(count), "s"(tokens), "s"(next.w[0]), "s"(next.w[4]), "s"(next.w[8]));
    const int most = tokens <= p.rows ? seats_least(count, p.room[3]) * p.hkv : 0, stride = p.last_blocks * 4;
    for (int unit = blockIdx.x * 4 + w; unit < most; unit += stride) {
        const int item = p.by_heads.of(unit), kvh = unit - item * p.hkv;
        const Words now = next;
        if (unit + stride < most) next = load(unit + stride);
        const int tok = now.w[0], L = now.w[1], lo = now.w[2], tab = now.w[3], part = now.w[4], parts = now.w[5];
        const int page[SEAT_PAGES] = {now.w[6], now.w[7], now.w[8], now.w[9], now.w[10], now.w[11]};
        const int n = L - lo, page0 = p.page.of(lo >> 4), many = p.page.of((L - 1) >> 4) - page0 + 1;
        const char* const kb = p.k + kvh * p.k_head + col * 2;
        const char* const vb = p.v + kvh * p.v_head + col * 2;
        bf16x8 q[RM];
#pragma unroll
        for (int r = 0; r < RM; r++) q[r] = *(const bf16x8*)(p.q + (long)tok * p.q_tok + (long)(kvh * p.group + (r < p.group ? r : p.group - 1)) * p.q_head + col);
        float M[RM], l[RM], o[RM][8];
#pragma unroll
        for (int r = 0; r < RM; r++) {
            M[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int d = 0; d < 8; d++) o[r][d] = 0.f;
        }
        for (int k0 = 0; k0 < n; k0 += U * G) {
            bf16x8 kx[U], vx[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (k0 + u * G >= n) break;
                const int j = k0 + u * G + mine, key = lo + (j < n ? j : n - 1);   // (behind the last key: that one again)
                const int a = p.page.of(key >> 4), x = a - page0;
                int id = page[0];
                if (many <= SEAT_PAGES) {
#pragma unroll
                    for (int y = 1; y < SEAT_PAGES; y++) id = x == y ? page[y] : id;
                } else id = p.lists[tab + a];
                const unsigned row = key - a * p.page.d * 16;
                kx[u] = *(const bf16x8*)(kb + (unsigned long long)(unsigned)id * p.k_page + (unsigned long long)row * p.k_row);
                vx[u] = *(const bf16x8*)(vb + (unsigned long long)(unsigned)id * p.v_page + (unsigned long long)row * p.v_row);
            }
            float s[U][RM];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int r = 0; r < RM; r++) {
                    s[u][r] = -INFINITY;
                    if (k0 + u * G < n) {
                        float x = 0.f;
#pragma unroll
                        for (int d = 0; d < 8; d++) x = __builtin_fmaf((float)q[r][d], (float)kx[u][d], x);
                        x = over_lanes<LPK>(x, [](float a, float b) { return a + b; });
                        if (CAP) x = p.cap.of(x);
                        s[u][r] = k0 + u * G + mine < n ? x * p.cap.unit : -INFINITY;
                    }
                }
#pragma unroll
            for (int r = 0; r < RM; r++) {
                float top = M[r];
#pragma unroll
                for (int u = 0; u < U; u++) top = fmaxf(top, s[u][r]);
                const float ref = top == -INFINITY ? 0.f : top, f = __builtin_amdgcn_exp2f(M[r] - ref);
                M[r] = top;
                l[r] *= f;
#pragma unroll
                for (int d = 0; d < 8; d++) o[r][d] *= f;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (k0 + u * G >= n) break;
                    const float y = __builtin_amdgcn_exp2f(s[u][r] - ref);
                    l[r] += y;
                    if (k0 + u * G + mine < n) {
#pragma unroll
                        for (int d = 0; d < 8; d++) o[r][d] = __builtin_fmaf(y, (float)vx[u][d], o[r][d]);
                    }
                }
            }
        }
        // (rescaled to each other: nothing seen weighs nothing, and leaves NaN where it is)
        const auto add = [&](int r, float m, float sum, const float (&x)[8]) __attribute__((always_inline)) {
            const float top = fmaxf(M[r], m), ref = top == -INFINITY ? 0.f : top;
            const float f = M[r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(M[r] - ref), g = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - ref);
            M[r] = top;
            l[r] = f * l[r] + g * sum;
#pragma unroll
            for (int d = 0; d < 8; d++) o[r][d] = f * o[r][d] + g * x[d];
        };
        for (int s = mine; s < parts; s += G)
#pragma unroll
            for (int r = 0; r < RM; r++) {
                const long at = (long)(part + s) * p.hq + kvh * p.group + (r < p.group ? r : p.group - 1);
                const float4 a = *(const float4*)(p.part_o + at * D + col), b = *(const float4*)(p.part_o + at * D + col + 4);
                const float2 ml = p.part_ml[at];
                const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                add(r, ml.x, ml.y, x);
            }
#pragma unroll
        for (int d = LPK; d < 64; d <<= 1)
#pragma unroll
            for (int r = 0; r < RM; r++) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = __shfl_xor(o[r][i], d);
                const float m = __shfl_xor(M[r], d), sum = __shfl_xor(l[r], d);
                add(r, m, sum, x);
            }
#pragma unroll
        for (int r = 0; r < RM; r++)
            if (mine == 0 && r < p.group) {
                const float f = inverse(l[r]);
                bf16x8 y;
#pragma unroll
                for (int d = 0; d < 8; d++) y[d] = (__bf16)(o[r][d] * f);
                *(bf16x8*)(p.out + (long)tok * p.o_tok + (long)(kvh * p.group + r) * p.o_head + col) = y;
                if (p.lse && lane == 0) p.lse[(long)tok * p.hq + kvh * p.group + r] = log_sum(M[r], l[r]);
            }
    }
}

// ------------------------------------------------------------------------------------------------ pieces joined
// out = sum_s 2^(M_s - M*) O_s / sum_s 2^(M_s - M*) l_s over a row's pieces.  A workgroup per token and 64 dims of its heads (or some of them: y0); 16 lanes hold a piece of
// a head, `share` such groups take a head's pieces in turn, each with a reference of its own, and are added up in one fixed order.
template <int D>
__device__ __forceinline__ void join(const Params& p, int block) {
    constexpr int SLICES = D / 64, GROUPS = 16;
    __shared__ __attribute__((aligned(16))) float part_sum[GROUPS][64];
    __shared__ float2 part_ml[GROUPS];
    const int sets = p.join_x * SLICES, y0 = block / sets, x0 = block - y0 * sets, slice = x0 % SLICES;
    const int group = threadIdx.x >> 4, d = (threadIdx.x & 15) * 4, lane = threadIdx.x & 63, used = tokens_of(p);
    for (int tok0 = x0 / SLICES; tok0 < p.rows; tok0 += 64 * p.join_x) {
    // of 64 tokens of this workgroup: where their pieces begin, and how many there are (0: the last word is spoken).  Behind the step's last token the list may be an older step's, of
    // more rows, whose pieces are not in this call's workspace: nothing there counts
    const int at = tok0 + lane * p.join_x, begins = at < p.rows ? p.parts[at] : 0, ends = at < p.rows ? p.parts[at + 1] : 0;
    const int number = at >= used || used > p.rows || begins < 0 ? 0 : (ends & INT_MAX) - begins;
    unsigned long long left = __builtin_amdgcn_ballot_w64(number > 0 || ((at >= used || used > p.rows) && at < p.rows));
    while (left) {
    const int which = __builtin_ctzll(left), tok = tok0 + which * p.join_x;
    left &= left - 1;
    const int first = __builtin_amdgcn_readlane(begins, which), n = __builtin_amdgcn_readlane(number, which);
    if (n == 0) {
        const unsigned nothing = used > p.rows ? 0x7fc07fc0u : 0;
        for (int h = y0 * GROUPS + group; h < p.hq; h += p.join_y * GROUPS) {
            *(uint2*)(p.out + (long)tok * p.o_tok + (long)h * p.o_head + slice * 64 + d) = make_uint2(nothing, nothing);
            if (p.lse && slice == 0 && d == 0) p.lse[(long)tok * p.hq + h] = nothing ? NAN : -INFINITY;
        }
        continue;
    }
    int share = 1;   // (each group asks for four pieces at a time)
    while (share < GROUPS && share * 4 < n) share *= 2;
    const int heads = GROUPS / share, piece = group % share;
    for (int h0 = y0 * heads; h0 < p.hq; h0 += p.join_y * heads) {
        const int h = h0 + group / share;
        const bool on = h < p.hq;
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
        if (on)
            for (int s0 = piece; s0 < n; s0 += 4 * share) {   // four pieces requested at a time
                float4 x[4];
                float2 ml[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int s = s0 + k * share;
                    const long at = (long)(first + (s < n ? s : s0)) * p.hq + h;
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
            __syncthreads();   // (the room is free)
            *(float4*)&part_sum[group][d] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            if (d == 0) part_ml[group] = make_float2(top, total);
            __syncthreads();
            if (piece == 0) {
                const int shares = n < share ? n : share;
                const float m0 = top, l0 = total;
                for (int s = 1; s < shares; s++) top = fmaxf(top, part_ml[group + s].x);
                total = 0.f;
                const float4 own = make_float4(acc[0], acc[1], acc[2], acc[3]);
                acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
                add(own, m0, l0, top);
                for (int s = 1; s < shares; s++) {
                    const float2 ml = part_ml[group + s];
                    add(*(const float4*)&part_sum[group + s][d], ml.x, ml.y, top);
                }
            }
        }
        if (on && piece == 0) {
            const float f = inverse(total);
            bf16x4 y;
#pragma unroll
            for (int k = 0; k < 4; k++) y[k] = (__bf16)(acc[k] * f);
            *(bf16x4*)(p.out + (long)tok * p.o_tok + (long)h * p.o_head + slice * 64 + d) = y;
            if (p.lse && slice == 0 && d == 0) p.lse[(long)tok * p.hq + h] = log_sum(top, total);
        }
    }
    }
    }
}

// What comes behind the contents' and the own keys' pieces: workgroups ahead of `last_blocks` speak last words (WORDS: there may be some), the others join pieces.
template <int D, bool WORDS, bool CAP>
__global__ __launch_bounds__(256, WORDS ? 4 : 8) void seats_finish_kernel(const Params p) {
    if constexpr (WORDS) {
        if ((int)blockIdx.x < p.last_blocks) {
            last_words<D, CAP>(p);
            return;
        }
    }
    join<D>(p, blockIdx.x - p.last_blocks);
}

// Workgroups that walk a list: two rounds of those that run at a time (one that finds nothing still takes a microsecond of a place)
template <int D, int DV, int NW, bool CAP>
int launch(Params p, const spinf_seats_attn_args* a, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (a->rooms[2]) {
        const int64_t units = std::min<int64_t>(a->rooms[2] * p.hkv, 2 * seats_block_places(D));
        hipLaunchKernelGGL((seats_block_kernel<D, DV, CAP>), dim3((unsigned)units), dim3(256 * (D / DV)), 0, s, p);
        e = hipGetLastError();
    }
    if (e == hipSuccess) {
        const int64_t units = std::min<int64_t>(a->rooms[0] * p.hkv + (a->rooms[1] * p.hkv + NW - 1) / NW, 2 * seats_wave_places(D));
        hipLaunchKernelGGL((seats_wave_kernel<D, DV, NW, CAP>), dim3((unsigned)(DV < D ? (units + 7) / 8 * 16 : units)), dim3(64 * NW), 0, s, p);
        e = hipGetLastError();
    }
    if (e == hipSuccess) {
        p.last_blocks = (int)std::min<int64_t>((a->rooms[3] * p.hkv + 3) / 4, 1024);   // (as many waves as run at a time)
        p.join_x = std::min(p.rows, 4096 / (D / 64));
        const int x = p.join_x * (D / 64);
        p.join_y = x >= 1024 ? 1 : std::min(p.hq, (1024 + x - 1) / x);
        const dim3 grid((unsigned)(p.last_blocks + x * p.join_y));
        if (D >= 128 && p.last_blocks) hipLaunchKernelGGL((seats_finish_kernel<D, D >= 128, CAP>), grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL((seats_finish_kernel<D, false, CAP>), grid, dim3(256), 0, s, p);
        e = hipGetLastError();
    }
    return e == hipSuccess ? SPINF_OK : spinf_fail(SPINF_E_HIP, "seats_attn: launch: %s", hipGetErrorString(e));
}

template <int D, int DV, int NW>
int launch_cap(const Params& p, const spinf_seats_attn_args* a, hipStream_t s) {
    return p.cap.on ? launch<D, DV, NW, true>(p, a, s) : launch<D, DV, NW, false>(p, a, s);
}

}  // namespace

extern "C" int spinf_seats_attn_fwd(const spinf_seats_attn_args* a, void* stream) {
    if (!a) return spinf_fail(SPINF_E_ARG, "seats_attn: null args");
    const spinf_seats_kind& kd = a->kind;
    if (a->rows < 1 || a->rows > (1 << 22) || a->seats < 1 || a->seats > SEATS_MOST) return spinf_fail(SPINF_E_ARG, "seats_attn: %lld rows of %d seats", (long long)a->rows, a->seats);
    if (kd.hq <= 0 || kd.hkv <= 0 || kd.hq % kd.hkv || a->rows * kd.hq > (1 << 30)) return spinf_fail(SPINF_E_ARG, "seats_attn: %d query heads do not group over %d key / value heads", kd.hq, kd.hkv);
    if (a->page < 16 || a->page % 16 || a->page > (1 << 20)) return spinf_fail(SPINF_E_ARG, "seats_attn: pages of %d keys (a multiple of 16)", a->page);
    if (kd.window < 0) return spinf_fail(SPINF_E_ARG, "seats_attn: window %d", kd.window);
    if (!(a->scale > 0.f) || !(a->scale < INFINITY) || !(a->softcap >= 0.f) || !(a->softcap < INFINITY))
        return spinf_fail(SPINF_E_ARG, "seats_attn: scale %g must be positive and finite, softcap %g not negative", (double)a->scale, (double)a->softcap);
    if (!a->q || !a->out || !a->k || !a->v || !a->lists || !a->first || !a->pos || !kd.wave || !kd.single || !kd.block || !kd.last || !kd.counts || !kd.parts)
        return spinf_fail(SPINF_E_ARG, "seats_attn: null pointer");
    for (const void* ptr : {a->q, (const void*)a->out, a->k, a->v, (const void*)kd.wave, (const void*)kd.single, (const void*)kd.block, (const void*)kd.last})
        if ((uintptr_t)ptr % 16) return spinf_fail(SPINF_E_ARG, "seats_attn: tensors and lists must be 16-byte aligned");
    for (int64_t st : {a->q_tok, a->q_head, a->o_tok, a->o_head, a->k_page, a->k_row, a->k_head, a->v_page, a->v_row, a->v_head})
        if (st % 8) return spinf_fail(SPINF_E_ARG, "seats_attn: strides must be multiples of 8 elements");
    if (a->k_row < 0 || a->v_row < 0 || a->k_row > (1 << 24) || a->v_row > (1 << 24) || a->k_page < 0 || a->v_page < 0 || a->k_page > (1u << 30) || a->v_page > (1u << 30))
        return spinf_fail(SPINF_E_ARG, "seats_attn: strides of the cache must lie in 0 .. 2^24 elements (rows) and 0 .. 2^30 (pages)");   // (32-bit byte counts; 32 rows by 32-bit offsets)
    for (int i = 0; i < 5; i++)
        if (a->rooms[i] < (i < 2) || a->rooms[i] > (1 << 26) || (i < 4 && a->rooms[i] * kd.hkv > (1 << 30))) return spinf_fail(SPINF_E_ARG, "seats_attn: bad lengths of lists");
    const int64_t parts = a->rooms[4] * kd.hq, need = parts * (kd.d + 2) * 4;
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || (uintptr_t)a->workspace % 16))
        return spinf_fail(SPINF_E_ARG, "seats_attn: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
    Params p = {};
    p.q = (const __bf16*)a->q; p.out = (__bf16*)a->out; p.lse = a->lse;
    p.q_tok = a->q_tok; p.q_head = a->q_head; p.o_tok = a->o_tok; p.o_head = a->o_head;
    p.k = (const char*)a->k; p.v = (const char*)a->v;
    p.k_page = (unsigned)(2 * a->k_page); p.k_row = (unsigned)(2 * a->k_row); p.k_head = 2 * a->k_head;
    p.v_page = (unsigned)(2 * a->v_page); p.v_row = (unsigned)(2 * a->v_row); p.v_head = 2 * a->v_head;
    p.same = a->k_page == a->v_page && a->k_row == a->v_row;
    p.lists = a->lists; p.first = a->first; p.pos = a->pos; p.counts = kd.counts; p.parts = kd.parts;
    p.wave = (const SeatItem*)kd.wave; p.single = (const SeatItem*)kd.single; p.block = (const SeatItem*)kd.block; p.last = (const SeatLast*)kd.last;
    p.part_o = (float*)a->workspace;
    p.part_ml = (float2*)(p.part_o + parts * kd.d);
    p.hq = kd.hq; p.hkv = kd.hkv; p.group = kd.hq / kd.hkv; p.rows = (int)a->rows; p.seats = a->seats;
    p.window = kd.window < 1 << 30 ? kd.window : 1 << 30;
    for (int i = 0; i < 4; i++) p.room[i] = (int)a->rooms[i];
    p.page = PageDiv::of_page(a->page);
    p.by_group = Div::by(p.group);
    p.by_heads = Div::by(p.hkv);
    if (!SoftCap::of(a->scale, a->softcap, p.cap)) return spinf_fail(SPINF_E_ARG, "seats_attn: scale %g and softcap %g leave fp32's range", (double)a->scale, (double)a->softcap);
    hipStream_t s = (hipStream_t)stream;
    switch (kd.d) {
        case 64: return launch_cap<64, 64, 4>(p, a, s);
        case 128: return launch_cap<128, 128, 4>(p, a, s);
        case 256: return launch_cap<256, 256, 4>(p, a, s);
        case 512: return launch_cap<512, 256, 3>(p, a, s);
        default: return spinf_fail(SPINF_E_ARG, "seats_attn: head dim %d not supported (64, 128, 256, 512)", kd.d);
    }
}
