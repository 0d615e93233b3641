// Eviction from a paged cache by accumulated weight, for gfx950 (MI355X): which of a request's stored keys stay, per key / value head, and their move into
// other pages.  No counterpart in the reference.
//
// Which: all of them where `keep` is enough; else the first `sink`, the last `recent`, and of the others the keep - sink - recent with the largest weight,
// ties to the lowest index.  paged_keep_kernel, a workgroup per (request, head): the weights as unsigned keys of the same order (NaN above
// everything, -0 as +0), the smallest kept key found digit by digit (11, 11 and 10 bits, each digit by a histogram in LDS over the weights, which the L2 holds
// after the first), then one pass in which every wave counts, and one in which it writes, its own stretch in ascending order: no sort, no global atomics.
//
// Bound by the histograms' LDS operations (a weight's exponent falls into few bins) on the one compute unit that a set has: 128 sets of 7,000 .. 17,000 keys 35 us.
//
// Move: paged_move_kernel copies the kept rows of K and V, 16 bytes per lane; bound by HBM (16 requests, 4,096 kept keys on 8 heads of 128 dims: 537 MB read and
// written in 111 us, 4.8 TB/s; a plain copy reaches 5.2).
#include <hip/hip_runtime.h>

#include "spinf_tree.h"
#include "common.h"
#include "paged_dev.h"

namespace {

struct Params {
    const float* acc; long keys;            // [reqs, hkv, keys]
    const int* reqs; const int* new_reqs;   // {row, new tokens, stored keys, first page} of the requests before and behind
    const int* table; const int* new_table;
    int* kept; float* new_acc;              // [reqs, hkv, keep]
    char* k; char* v;
    long k_page, k_row, k_head, v_page, v_row, v_head;   // bytes
    int hkv, keep, sink, recent, chunks;
    PageDiv page;
};

// the weight as an unsigned number of the same order
__device__ __forceinline__ unsigned order(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int KW = 16;          // waves of a workgroup
constexpr int BINS = 2048;

// J: 64-key pieces of a wave's stretch that stay in registers, loaded once and together; 0: any number, loaded anew for every pass, eight at a time.
// (One at a time, anew for every pass, the loads' latency was all the time there was: 128 sets of 12,000 keys 45 us.)
template <int J>
__global__ __launch_bounds__(64 * KW) void paged_keep_kernel(const Params p) {
    __shared__ __attribute__((aligned(16))) int hist[BINS][4];   // four counts a bin, by lane: equal weights queue for one word otherwise
    __shared__ int wave_sum[KW], above[KW], equal[KW];
    __shared__ int found[2];
    const int rh = blockIdx.x, r = rh / p.hkv;
    const int n = sload(p.reqs, 4 * r + 2);
    const float* x = p.acc + (long)rh * p.keys;
    int* kept = p.kept + (long)rh * p.keep;
    float* new_acc = p.new_acc + (long)rh * p.keep;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (n <= p.keep) {
        for (int i = tid; i < p.keep; i += 64 * KW) {
            kept[i] = i < n ? i : -1;
            new_acc[i] = i < n ? x[i] : 0.f;
        }
        return;
    }
    const int c0 = p.sink, c1 = n - p.recent;             // candidates
    const int want = p.keep - p.sink - p.recent;          // of these stay (0 <= want < c1 - c0)
    const int per = ((n + KW - 1) / KW + 63) / 64 * 64, i0 = w * per, i1 = i0 + per < n ? i0 + per : n;   // this wave's stretch of the keys
    float mine[J ? J : 8];
    if (J) {
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int i = i0 + j * 64 + lane;
            mine[j] = j * 64 < per ? x[i < i1 ? i : 0] : 0.f;
        }
    }
    // f(i, weight) for every 64 keys of the stretch, whole waves: i >= i1 is no key
    const auto each = [&](auto f) __attribute__((always_inline)) {
        if (J) {
#pragma unroll
            for (int j = 0; j < J; j++)
                if (i0 + j * 64 < i1) f(i0 + j * 64 + lane, mine[j]);
        } else {
            for (int b = i0; b < i1; b += 8 * 64) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int i = b + j * 64 + lane;
                    mine[j] = x[i < i1 ? i : 0];
                }
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (b + j * 64 < i1) f(b + j * 64 + lane, mine[j]);
            }
        }
    };
    // the smallest key that stays, digit by digit: `floor` holds the digits found, `left` how many of the keys with these digits stay
    unsigned floor = 0;
    int left = want;
    if (want > 0) {
#pragma unroll 1
        for (int d = 0; d < 3; d++) {
            const int sh = d == 0 ? 21 : d == 1 ? 10 : 0, bits = d == 2 ? 10 : 11;
            for (int i = tid; i < BINS; i += 64 * KW) *(int4*)hist[i] = make_int4(0, 0, 0, 0);
            __syncthreads();
            each([&](int i, float xi) __attribute__((always_inline)) {
                const unsigned o = order(xi);
                if (i >= c0 && i < c1 && i < i1 && (d == 0 || (o >> (sh + bits)) == (floor >> (sh + bits)))) atomicAdd(&hist[(o >> sh) & ((1 << bits) - 1)][lane & 3], 1);
            });
            __syncthreads();
            // bins from the highest down, two per thread: a running count over the workgroup, and the bin in which it reaches `left`
            const int b1 = BINS - 1 - 2 * tid;
            const int4 h1 = *(const int4*)hist[b1], h0 = *(const int4*)hist[b1 - 1];
            const int n1 = h1.x + h1.y + h1.z + h1.w, n0 = h0.x + h0.y + h0.z + h0.w;
            int run = n1 + n0;
#pragma unroll
            for (int k = 1; k < 64; k <<= 1) {
                const int o = __shfl_up(run, k);
                if (lane >= k) run += o;
            }
            if (lane == 63) wave_sum[w] = run;
            __syncthreads();
            int before = run - n1 - n0;
            for (int k = 0; k < w; k++) before += wave_sum[k];
            if (before < left && before + n1 >= left) { found[0] = b1; found[1] = left - before; }
            else if (before + n1 < left && before + n1 + n0 >= left) { found[0] = b1 - 1; found[1] = left - before - n1; }
            __syncthreads();
            floor |= (unsigned)found[0] << sh;
            left = found[1];
        }
    }
    // Each wave counts in its stretch the keys above the floor (or kept whatever they weigh), and those equal to it.
    int a = 0, e = 0;
    each([&](int i, float xi) __attribute__((always_inline)) {
        const bool in = i < i1, always = in && (i < c0 || i >= c1);
        const unsigned o = order(xi);
        a += __popcll(__builtin_amdgcn_ballot_w64(always || (in && want > 0 && o > floor)));
        e += __popcll(__builtin_amdgcn_ballot_w64(in && !always && want > 0 && o == floor));
    });
    if (lane == 0) { above[w] = a; equal[w] = e; }
    __syncthreads();
    int at = 0, ties = 0;   // kept keys and ties in front of this wave's stretch
    for (int k = 0; k < w; k++) {
        const int room = left - ties, t = equal[k] < room ? equal[k] : room;
        at += above[k] + (t > 0 ? t : 0);
        ties += equal[k];
    }
    const unsigned long long below = (1ull << lane) - 1;
    each([&](int i, float xi) __attribute__((always_inline)) {
        const bool in = i < i1, always = in && (i < c0 || i >= c1);
        const unsigned o = order(xi);
        const bool tie = in && !always && want > 0 && o == floor;
        const unsigned long long tie_mask = __builtin_amdgcn_ballot_w64(tie);
        const bool stays = always || (in && want > 0 && o > floor) || (tie && ties + __popcll(tie_mask & below) < left);
        const unsigned long long mask = __builtin_amdgcn_ballot_w64(stays);
        if (stays) {
            const int j = at + __popcll(mask & below);
            kept[j] = i;
            new_acc[j] = xi;
        }
        at += __popcll(mask);
        ties += __popcll(tie_mask);
    });
}

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

constexpr int MROWS = 64;   // rows of a workgroup of the move

template <int D>
__global__ __launch_bounds__(256) void paged_move_kernel(const Params p) {
    constexpr int PIECES = D / 8, STEP = 256 / PIECES, U = MROWS / STEP < 4 ? MROWS / STEP : 4;   // rows at a time; of these so many requested together
    const int chunk = blockIdx.x % p.chunks, rh = blockIdx.x / p.chunks, r = rh / p.hkv, h = rh - r * p.hkv;
    const int n = sload(p.reqs, 4 * r + 2), tab = sload(p.reqs, 4 * r + 3), to = sload(p.new_reqs, 4 * r + 3);
    const int m = n < p.keep ? n : p.keep;
    const int piece = threadIdx.x % PIECES, row0 = chunk * MROWS + threadIdx.x / PIECES;
    if (chunk * MROWS >= m) return;
    const int* kept = p.kept + (long)rh * p.keep;
    for (int u0 = 0; u0 < MROWS; u0 += U * STEP) {
        u32x4 xk[U], xv[U];
        long dk[U], dv[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = row0 + u0 + u * STEP, jc = j < m ? j : m - 1;
            const int s = kept[jc];
            const int a = p.page.of(s >> 4), b = p.page.of(jc >> 4);
            const long from = p.table[tab + a], dst = p.new_table[to + b];
            const long es = s - a * p.page.d * 16, ed = jc - b * p.page.d * 16;
            xk[u] = *(const u32x4*)(p.k + from * p.k_page + es * p.k_row + h * p.k_head + piece * 16);
            xv[u] = *(const u32x4*)(p.v + from * p.v_page + es * p.v_row + h * p.v_head + piece * 16);
            dk[u] = dst * p.k_page + ed * p.k_row + h * p.k_head + piece * 16;
            dv[u] = dst * p.v_page + ed * p.v_row + h * p.v_head + piece * 16;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (row0 + u0 + u * STEP < m) {
                *(u32x4*)(p.k + dk[u]) = xk[u];
                *(u32x4*)(p.v + dv[u]) = xv[u];
            }
    }
}

}  // namespace

extern "C" int spinf_cache_evict(const spinf_evict_args* a, void* stream) {
    if (!a) return spinf_fail(SPINF_E_ARG, "cache_evict: null args");
    if (a->n_reqs < 0 || a->n_reqs > (1 << 24) || a->hkv <= 0 || a->hkv > 4096 || a->keys < 0 || a->keys > (1 << 30)) return spinf_fail(SPINF_E_ARG, "cache_evict: bad sizes");
    if (a->sink < 0 || a->recent < 0 || a->keep < 0 || (int64_t)a->sink + a->recent > a->keep) return spinf_fail(SPINF_E_ARG, "cache_evict: keep %d, of these the first %d and the last %d", a->keep, a->sink, a->recent);
    if (a->d != 64 && a->d != 128 && a->d != 256 && a->d != 512) return spinf_fail(SPINF_E_ARG, "cache_evict: head dim %d not supported (64, 128, 256, 512)", a->d);
    if (a->page < 16 || a->page % 16 || a->page > (1 << 20)) return spinf_fail(SPINF_E_ARG, "cache_evict: pages of %d keys (a multiple of 16)", a->page);
    if (a->n_reqs == 0 || a->keep == 0 || a->keys == 0) return SPINF_OK;
    if (!a->acc || !a->reqs || !a->new_reqs || !a->table || !a->new_table || !a->kept || !a->new_acc || !a->k || !a->v) return spinf_fail(SPINF_E_ARG, "cache_evict: null pointer");
    if ((uintptr_t)a->k % 16 || (uintptr_t)a->v % 16) return spinf_fail(SPINF_E_ARG, "cache_evict: the cache must be 16-byte aligned");
    for (int64_t st : {a->k_page, a->k_row, a->k_head, a->v_page, a->v_row, a->v_head})
        if (st % 8) return spinf_fail(SPINF_E_ARG, "cache_evict: strides must be multiples of 8 elements");
    Params p = {};
    p.acc = a->acc; p.keys = a->keys; p.reqs = a->reqs; p.new_reqs = a->new_reqs; p.table = a->table; p.new_table = a->new_table;
    p.kept = a->kept; p.new_acc = a->new_acc; p.k = (char*)a->k; p.v = (char*)a->v;
    p.k_page = 2 * a->k_page; p.k_row = 2 * a->k_row; p.k_head = 2 * a->k_head;
    p.v_page = 2 * a->v_page; p.v_row = 2 * a->v_row; p.v_head = 2 * a->v_head;
    p.hkv = a->hkv; p.keep = a->keep; p.sink = a->sink; p.recent = a->recent;
    const int64_t most = a->keep < a->keys ? a->keep : a->keys;   // rows of the fullest request
    p.chunks = (int)((most + MROWS - 1) / MROWS);
    p.page = PageDiv::of_page(a->page);
    const int64_t grid = a->n_reqs * a->hkv;
    if (grid * p.chunks > INT32_MAX) return spinf_fail(SPINF_E_ARG, "cache_evict: %lld requests of %d kept keys are too many", (long long)a->n_reqs, a->keep);
    hipStream_t s = (hipStream_t)stream;
    // Stretches of up to 4 and 16 pieces of 64 keys: 4,096 and 16,384 keys.  (us with the variant for that many / the next one / the one for any number: 8 sets of 900 keys
    // 8.5 / 15.2 / 12.1, 128 of 4,000 10.8 / - / 13.5, 128 of 12,000 20.3 / 25.3 / 23.8; 32 pieces in registers gained nothing, 128 sets of 30,000 45 / - / 45.)
    if (a->keys <= 4 * 64 * KW) hipLaunchKernelGGL(paged_keep_kernel<4>, dim3((unsigned)grid), dim3(64 * KW), 0, s, p);
    else if (a->keys <= 16 * 64 * KW) hipLaunchKernelGGL(paged_keep_kernel<16>, dim3((unsigned)grid), dim3(64 * KW), 0, s, p);
    else hipLaunchKernelGGL(paged_keep_kernel<0>, dim3((unsigned)grid), dim3(64 * KW), 0, s, p);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) {
        const dim3 g((unsigned)(grid * p.chunks));
        switch (a->d) {
            case 64: hipLaunchKernelGGL((paged_move_kernel<64>), g, dim3(256), 0, s, p); break;
            case 128: hipLaunchKernelGGL((paged_move_kernel<128>), g, dim3(256), 0, s, p); break;
            case 256: hipLaunchKernelGGL((paged_move_kernel<256>), g, dim3(256), 0, s, p); break;
            default: hipLaunchKernelGGL((paged_move_kernel<512>), g, dim3(256), 0, s, p); break;
        }
        e = hipGetLastError();
    }
    return e == hipSuccess ? SPINF_OK : spinf_fail(SPINF_E_HIP, "cache_evict: launch: %s", hipGetErrorString(e));
}
