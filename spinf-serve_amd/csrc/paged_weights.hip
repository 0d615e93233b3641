// The attention weight that every stored key of a paged cache received, for gfx950 (MI355X): what cache_evict (paged_evict.hip) decides by.  No
// counterpart in the reference.
//
// Mathematics: W[r, h, s] = acc[r, h, s] + sum over the request's new tokens that see key s and the query heads of key / value head h of
// exp(cap(scale q.k) - lse), with the log-sums lse that the attention left: the probabilities once more, without their softmax.
//
// S = Q K^T the other way round than in the attention: a lane of v_mfma_f32_32x32x16_bf16's result owns one KEY and 16 of the 32 rows, so a key's
// sum stays in its lane over all rows: no atomics, one order, one lane exchange at the end.  A workgroup's waves take 32 keys each: the keys come once, by
// DMA through LDS, and stay in registers; the rows follow into the same place, a block of 32 per wave at a time.
//
// Bound by HBM where rows are few (16 requests of ~2,500 keys, one token, 16 heads on 8 of 256 dims: 195 MB in 37 us, 5.3 TB/s); by the products, exponentials and
// key bytes one after the other where they are many (4 requests of 16,001 keys, 64 tokens, 32 on 16 of 128: 85 us; 58 for its bytes alone, 28 for its products).
#include <hip/hip_runtime.h>

#include <climits>

#include "spinf_tree.h"
#include "common.h"
#include "paged_dev.h"

namespace {

struct Params {
    const __bf16* q; const float* lse; const float* acc; float* out;
    long q_tok, q_head;
    const char* k;
    long k_page, k_row, k_head;   // bytes
    const int* table; const int* reqs; const int* end; const int* pos;
    long keys;                    // of a row of acc and out
    int blocks, hq, hkv, window;
    Div group;   // query heads per key / value head
    PageDiv page;
    SoftCap cap;
};

// Rows of up to NW blocks of 32 as the products need them: log-sums in units of log 2 (infinite: the row gives no weight), tokens, positions
template <int NW>
struct RowData {
    float lse[NW][32];
    int tok[NW][32], pos[NW][32];
};

// FEW: every request's rows fit one block (a decoding step)
template <int D, int NW, bool CAP, bool FEW>
__global__ __launch_bounds__(64 * NW) void paged_weights_kernel(const Params p) {
    using GK = Geo<D, TK>;
    constexpr int NS = D / 16;
    __shared__ __attribute__((aligned(16))) char lds[NW * GK::KTILEB];   // 32 keys of each wave; behind that NW blocks of 32 queries
    __shared__ __attribute__((aligned(16))) RowData<NW> rd;
    const int lane = threadIdx.x & 63, m = lane & 31, g = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rh = blockIdx.x / p.blocks, r = rh / p.hkv, kvh = rh - r * p.hkv;
    const int kt0 = (int)(blockIdx.x - (unsigned)rh * p.blocks) * NW, kt = kt0 + w;
    const int cu = sload(p.reqs, 4 * r), T = sload(p.reqs, 4 * r + 1), L = sload(p.reqs, 4 * r + 2), tab = sload(p.reqs, 4 * r + 3);
    const int key = kt * TK + m;
    float sum = 0.f;
    if (kt0 * TK < L && T > 0) {   // (uniform over the workgroup)
        const bool on = kt * TK < L;
        const int c = L - T, N = T * p.group.d;
        char* const kb = lds + w * GK::KTILEB;
        if (on) {
            const int n = 2 * kt, last16 = (L - 1) >> 4, n1 = n + 1 < last16 ? n + 1 : last16;
            const int last = L - 1 - kt * TK < TK - 1 ? L - 1 - kt * TK : TK - 1;
            const int a = p.page.of(n), b = p.page.of(n1);
            const long ia = sload(p.table, tab + a), ib = sload(p.table, tab + b);
            const char* k0 = p.k + ia * p.k_page + (long)(n - a * p.page.d) * 16 * p.k_row + kvh * p.k_head;
            const char* k1 = p.k + ib * p.k_page + (long)(n1 - b * p.page.d) * 16 * p.k_row + kvh * p.k_head;
            fetch<D, GK::NREG, GK::KRS>(k0, k1, p.k_row, last, 0, lds_addr(kb), lane);
        }
        const int u = key - c;   // this lane's key as a new token of the request (below 0: stored before)
        const bool fresh = p.end && u >= 0;
        const int uc = u < T ? u : T - 1;
        const int end_k = fresh ? p.end[cu + uc] : INT_MAX;
        const int pos_k = fresh ? p.pos[cu + uc] : key;
        const int u_lo = kt * TK - c, u_hi = u_lo + TK - 1;
        // token and head of this lane's row of a block (rows behind the last: the last one)
        const auto place = [&](int row, int& tok, int& head) __attribute__((always_inline)) {
            const int rc = row < N ? row : N - 1;
            tok = p.group.of(rc);
            head = kvh * p.group.d + (rc - tok * p.group.d);
        };
        // few rows go straight into registers; where no request has more, they are asked for while the keys are on their way (their registers would
        // cost the kernel for many rows a workgroup per compute unit: 91 -> 99 us)
        const bool few = FEW || N <= 32;
        bf16x8 qf[FEW ? NS : 1];
        int tok0 = 0, head0 = 0;
        place(m, tok0, head0);
        const __bf16* qp = p.q + (long)(cu + tok0) * p.q_tok + (long)head0 * p.q_head + 8 * g;
        if (FEW) {
#pragma unroll
            for (int st = 0; st < NS; st++) qf[st] = *(const bf16x8*)(qp + 16 * st);
        }
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        __builtin_amdgcn_sched_barrier(0);
        bf16x8 kf[NS];
#pragma unroll
        for (int s = 0; s < NS; s++) kf[s] = *(const bf16x8*)(kb + GK::k_off(m) + 16 * g + 32 * s);

        const auto note = [&](int slot, int row, int tok, int head) __attribute__((always_inline)) {   // (lanes of either half: the same values)
            const float lse = p.lse[(long)(cu + tok) * p.hq + head];
            rd.lse[slot][m] = row < N && lse != -INFINITY ? lse * LOG2E : INFINITY;
            rd.tok[slot][m] = tok;
            rd.pos[slot][m] = p.window ? (p.end ? p.pos[cu + tok] : c + tok) : 0;
        };
        // weights of a block's rows; s: its scores, register i of which holds row 8 (i / 4) + 4 g + i % 4; first: the block's first token
        const auto add = [&](f32x16& s, int slot, int first) __attribute__((always_inline)) {
            if (CAP) p.cap.of(s);
            const bool masked = u_hi > first || p.window || p.end;
#pragma unroll
            for (int i4 = 0; i4 < 4; i4++) {
                const float4 l4 = *(const float4*)&rd.lse[slot][8 * i4 + 4 * g];
                const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
                int tv[4] = {0, 0, 0, 0}, pv[4] = {0, 0, 0, 0};
                if (masked) {
                    const int4 t4 = *(const int4*)&rd.tok[slot][8 * i4 + 4 * g], p4 = *(const int4*)&rd.pos[slot][8 * i4 + 4 * g];
                    tv[0] = t4.x; tv[1] = t4.y; tv[2] = t4.z; tv[3] = t4.w;
                    pv[0] = p4.x; pv[1] = p4.y; pv[2] = p4.z; pv[3] = p4.w;
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i4 + j], p.cap.unit, -lv[j]));
                    bool vis = true;
                    if (masked) {
                        vis = (u <= tv[j]) & (cu + tv[j] < end_k);
                        if (p.window) vis = vis & (pv[j] - pos_k < p.window);
                    }
                    sum += vis ? x : 0.f;
                }
            }
        };
        if (few) {
            if (on) {
                note(w, m, tok0, head0);
                f32x16 s;
#pragma unroll
                for (int i = 0; i < 16; i++) s[i] = 0.f;
#pragma unroll
                for (int st = 0; st < NS; st++) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(FEW ? qf[FEW ? st : 0] : *(const bf16x8*)(qp + 16 * st), kf[st], s, 0, 0, 0);
                add(s, w, 0);
            }
        } else if (!FEW) {
            // Many rows: the keys' place in LDS is free now; it takes a block of rows per wave at a time, from which all waves compute.  (Each wave
            // loading every row from memory by itself: 4 x 16k keys, 64 tokens, 32 / 16 x 128, 154 us.)
            const int top = kt0 * TK - c;   // first key of the workgroup as a new token: earlier rows see none of its keys
            const int first = top > 0 ? (int)((long)top * p.group.d / 32) : 0;
            long rows = N;
            if (p.window && !p.end) {   // (without a tree a row's position is its place) later tokens are too far from the workgroup's keys
                const long most = ((long)kt0 * TK + NW * TK - 1 - c + p.window) * p.group.d;
                rows = most < rows ? most : rows;
            }
            const int blocks = rows > 0 ? (int)((rows + 31) / 32) : 0;
            for (int b0 = first; b0 < blocks; b0 += NW) {
                __syncthreads();   // every wave has its keys in registers, or is through with the blocks before
                if (b0 + w < blocks) {
                    const int row0 = (b0 + w) * 32;
                    int tok, head;
#pragma unroll
                    for (int i = 0; i < GK::NREG; i++) {
                        place(row0 + i + GK::NREG * (lane / GK::CPR), tok, head);
                        dma16_lane((const char*)(p.q + (long)(cu + tok) * p.q_tok + (long)head * p.q_head) + lane % GK::CPR * 16, lds_addr(kb) + i * GK::KRS);
                    }
                    place(row0 + m, tok, head);
                    note(w, row0 + m, tok, head);
                }
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
                __syncthreads();
                if (!on) continue;
                const int here = blocks - b0 < NW ? blocks - b0 : NW;
                for (int b = 0; b < here; b++) {
                    const int last_tok = __builtin_amdgcn_readfirstlane(rd.tok[b][31]);
                    if (last_tok < u_lo) continue;   // all of the block's tokens lie before the wave's keys
                    const char* qb = lds + b * GK::KTILEB + GK::k_off(m) + 16 * g;
                    f32x16 s;
#pragma unroll
                    for (int i = 0; i < 16; i++) s[i] = 0.f;
#pragma unroll
                    for (int st = 0; st < NS; st++) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(qb + 32 * st), kf[st], s, 0, 0, 0);
                    add(s, b, __builtin_amdgcn_readfirstlane(rd.tok[b][0]));
                }
            }
        }
        sum = lane32_sum(sum);
    }
    if (g == 0 && key < p.keys) {
        const long at = (long)rh * p.keys + key;
        const float before = p.acc ? p.acc[at] : 0.f;
        p.out[at] = key < L ? before + sum : before;
    }
}

template <int D, int NW>
int launch(Params p, const spinf_paged_weights_args* a, hipStream_t s) {
    const int64_t blocks = (p.keys + 32 * NW - 1) / (32 * NW), n = blocks * p.hkv * a->n_reqs;
    if (n > INT32_MAX) return spinf_fail(SPINF_E_ARG, "paged_weights: %lld requests of %ld keys are too many", (long long)a->n_reqs, p.keys);
    p.blocks = (int)blocks;
    const dim3 grid((unsigned)n), threads(64 * NW);
    const bool cap = p.cap.on, few = (int64_t)a->max_q * p.group.d <= 32;
    if (cap && few) hipLaunchKernelGGL((paged_weights_kernel<D, NW, true, true>), grid, threads, 0, s, p);
    else if (cap) hipLaunchKernelGGL((paged_weights_kernel<D, NW, true, false>), grid, threads, 0, s, p);
    else if (few) hipLaunchKernelGGL((paged_weights_kernel<D, NW, false, true>), grid, threads, 0, s, p);
    else hipLaunchKernelGGL((paged_weights_kernel<D, NW, false, false>), grid, threads, 0, s, p);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPINF_OK : spinf_fail(SPINF_E_HIP, "paged_weights: launch: %s", hipGetErrorString(e));
}

}  // namespace

extern "C" int spinf_paged_weights(const spinf_paged_weights_args* a, void* stream) {
    if (!a) return spinf_fail(SPINF_E_ARG, "paged_weights: null args");
    if (a->n_reqs < 0 || a->n_reqs > (1 << 24) || a->keys < 0 || a->keys > (1 << 30)) return spinf_fail(SPINF_E_ARG, "paged_weights: %lld requests, %lld keys", (long long)a->n_reqs, (long long)a->keys);
    if (a->hq <= 0 || a->hkv <= 0 || a->hq % a->hkv) return spinf_fail(SPINF_E_ARG, "paged_weights: %d query heads do not group over %d key / value heads", a->hq, a->hkv);
    if (a->d != 64 && a->d != 128 && a->d != 256 && a->d != 512) return spinf_fail(SPINF_E_ARG, "paged_weights: head dim %d not supported (64, 128, 256, 512)", a->d);
    if (a->page < 16 || a->page % 16 || a->page > (1 << 20)) return spinf_fail(SPINF_E_ARG, "paged_weights: pages of %d keys (a multiple of 16)", a->page);
    if (a->max_q < 0 || a->max_q > a->tokens) return spinf_fail(SPINF_E_ARG, "paged_weights: %d new tokens of a request of %lld", a->max_q, (long long)a->tokens);
    if (a->window < 0) return spinf_fail(SPINF_E_ARG, "paged_weights: window %d", a->window);
    if (!(a->scale > 0.f) || !(a->scale < INFINITY) || !(a->softcap >= 0.f) || !(a->softcap < INFINITY))
        return spinf_fail(SPINF_E_ARG, "paged_weights: scale %g must be positive and finite, softcap %g not negative", (double)a->scale, (double)a->softcap);
    if (a->n_reqs == 0 || a->keys == 0) return SPINF_OK;
    if (!a->reqs || !a->out || !a->k || !a->table || (a->tokens > 0 && (!a->q || !a->lse))) return spinf_fail(SPINF_E_ARG, "paged_weights: null pointer");
    if ((a->end == nullptr) != (a->pos == nullptr)) return spinf_fail(SPINF_E_ARG, "paged_weights: a tree needs both end and pos");
    if ((uintptr_t)a->q % 16 || (uintptr_t)a->k % 16 || (uintptr_t)a->reqs % 16) return spinf_fail(SPINF_E_ARG, "paged_weights: tensors must be 16-byte aligned");
    for (int64_t st : {a->q_tok, a->q_head, a->k_page, a->k_row, a->k_head})
        if (st % 8) return spinf_fail(SPINF_E_ARG, "paged_weights: strides must be multiples of 8 elements");
    if (a->k_row < 0 || a->k_row > (1 << 24)) return spinf_fail(SPINF_E_ARG, "paged_weights: row strides of the cache must lie in 0 .. 2^24");
    Params p = {};
    p.q = (const __bf16*)a->q; p.lse = a->lse; p.acc = a->acc; p.out = a->out;
    p.q_tok = a->q_tok; p.q_head = a->q_head;
    p.k = (const char*)a->k; p.k_page = 2 * a->k_page; p.k_row = 2 * a->k_row; p.k_head = 2 * a->k_head;
    p.table = a->table; p.reqs = a->reqs; p.end = a->end; p.pos = a->pos;
    p.keys = a->keys; p.hq = a->hq; p.hkv = a->hkv; p.group = Div::by(a->hq / a->hkv); p.window = a->window;
    p.page = PageDiv::of_page(a->page);
    if (!SoftCap::of(a->scale, a->softcap, p.cap)) return spinf_fail(SPINF_E_ARG, "paged_weights: scale %g and softcap %g leave fp32's range", (double)a->scale, (double)a->softcap);
    hipStream_t s = (hipStream_t)stream;
    switch (a->d) {
        case 64: return launch<64, 4>(p, a, s);
        case 128: return launch<128, 4>(p, a, s);
        case 256: return launch<256, 4>(p, a, s);
        default: return launch<512, 2>(p, a, s);
    }
}
