// Norms of queries and keys for each head, with the rotation by position in the same pass, and the keys' and values' way into a paged cache, for
// gfx950 (MI355X).  What the reference's attention modules leave to a compiler between the projection and the attention call (the lines in front of
// spinf_serve/models/qwen35/qwen.py:604-623 and spinf_serve/models/gemma4.py:98-119); the cache has no counterpart there.
//
// Mathematics, per token and head of d dims: y = x / sqrt(mean x^2 + eps) * w; then pairs (a, b) of the first `rot` dims become
// (a cos - b sin, b cos + a sin), the pairs being (i, i + rot / 2) or (2 i, 2 i + 1).  All of it in fp32, rounded to bf16 once, when stored.
//
// Bound by HBM: every row is read once and written once.  A lane owns two 8-dim pieces of a row that hold both ends of its pairs, so the rotation needs no
// exchange and the norm's sum a few lane exchanges; a wave owns a token and U x (1,024 / d) of its heads, whose loads all go out before the first is
// used, and its cosines and sines are read once for all of them.  (27,452 tokens x 32 rows of 256 dims: 899 MB in 172 us, 5.2 TB/s, a plain copy's rate.)
#include <hip/hip_runtime.h>

#include "spinf_tree.h"
#include "common.h"

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;

namespace {

struct Params {
    const __bf16 *q, *k, *v; long q_tok, q_head, k_tok, k_head, v_tok, v_head;
    const void *wq, *wk, *cos, *sin; long cos_ld, sin_ld;
    const void* pos; const long* slots;
    __bf16 *q_out, *k_out, *v_out;
    long k_page, k_row, kh_out, v_page, v_row, vh_out;   // of the cache; without one (slots NULL) k_out is dense
    long T, n_pos, capacity;
    int hq, hkv, heads, rot, page, parts;
    int neighbours, plus_one, v_norm, w_f32, cs_f32, pos_i64;
    float eps;
};

// eight values of a table in bf16 or fp32
__device__ __forceinline__ void load8(const void* p, long i, int f32, float (&x)[8]) {
    if (f32) {
        const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const bf16x8 a = *(const bf16x8*)((const __bf16*)p + i);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)a[e];
    }
}

// 1 / sqrt(x); the instruction by itself takes a subnormal x for zero (rows of some 1e-19 with eps 0)
__device__ __forceinline__ float inverse_root(float x) {
    const bool tiny = x < 0x1p-100f;
    const float r = __builtin_amdgcn_rsqf(tiny ? x * 0x1p100f : x);
    return tiny ? r * 0x1p50f : r;
}

template <int D, int U>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const Params p) {
    constexpr int LANES = D / 16;       // lanes of a row
    constexpr int ROWS = 64 / LANES;    // heads of a wave at a time
    const int lane = threadIdx.x & 63, j = lane % LANES;
    const long wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const long t = wave / p.parts;
    if (t >= p.T) return;
    const int h0 = (int)(wave - t * p.parts) * (U * ROWS) + lane / LANES;

    // pieces a and b of this lane: both ends of its pairs, or two neighbours behind the rotated dims
    const int half = p.rot / 2, turning = p.rot / 16;
    const bool turn = j < turning;
    const int a0 = turn && !p.neighbours ? 8 * j : 16 * j, b0 = turn && !p.neighbours ? half + 8 * j : 16 * j + 8;

    bf16x8 xa[U], xb[U];
    int kind[U];   // 0 query, 1 key, 2 value, 3 none
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int h = h0 + u * ROWS;
        kind[u] = h < p.hq ? 0 : h < p.hq + p.hkv ? 1 : h < p.heads ? 2 : 3;
        const __bf16* x = kind[u] == 0 ? p.q + t * p.q_tok + h * p.q_head : kind[u] == 1 ? p.k + t * p.k_tok + (h - p.hq) * p.k_head
                        : kind[u] == 2 ? p.v + t * p.v_tok + (h - p.hq - p.hkv) * p.v_head : p.q + t * p.q_tok;
        xa[u] = *(const bf16x8*)(x + a0);
        xb[u] = *(const bf16x8*)(x + b0);
    }
    const long at = p.pos ? (p.pos_i64 ? ((const long*)p.pos)[t] : (long)((const int*)p.pos)[t]) : t;
    const bool known = at >= 0 && at < p.n_pos;
    const long slot = p.slots ? p.slots[t] : 0;
    float c[8], s[8];
    if (p.rot) {
        const long row = known ? at : 0;
        load8(p.cos, row * p.cos_ld + (turn ? 8 * j : 0), p.cs_f32, c);
        load8(p.sin, row * p.sin_ld + (turn ? 8 * j : 0), p.cs_f32, s);
    }
    const unsigned place = p.slots && slot >= 0 && slot < p.capacity ? (unsigned)slot : 0u;
    const unsigned pg = p.slots ? place / (unsigned)p.page : 0u, entry = place - pg * (unsigned)p.page;

#pragma unroll
    for (int u = 0; u < U; u++) {
        float a[8], b[8], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            a[e] = (float)xa[u][e];
            b[e] = (float)xb[u][e];
            sum = __builtin_fmaf(a[e], a[e], __builtin_fmaf(b[e], b[e], sum));
        }
#pragma unroll
        for (int d = 1; d < LANES; d <<= 1) sum += __shfl_xor(sum, d);
        float r = inverse_root(sum * (1.0f / D) + p.eps);
        if (kind[u] == 2 && !p.v_norm) r = 1.0f;
        if (kind[u] < 2) {
            // A position outside the tables, or a place outside the cache, cannot be refused here: the row says so itself.
            if ((p.rot && !known) || (kind[u] == 0 && slot >= p.capacity && p.slots)) r = __builtin_nanf("");
            const void* w = kind[u] == 0 ? p.wq : p.wk;
            if (w) {
                float wa[8], wb[8];
                load8(w, a0, p.w_f32, wa);
                load8(w, b0, p.w_f32, wb);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    a[e] *= p.plus_one ? 1.0f + wa[e] : wa[e];
                    b[e] *= p.plus_one ? 1.0f + wb[e] : wb[e];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            a[e] *= r;
            b[e] *= r;
        }
        if (turn && kind[u] < 2) {
            if (p.neighbours) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float a1 = a[2 * e], a2 = a[2 * e + 1], b1 = b[2 * e], b2 = b[2 * e + 1];
                    a[2 * e] = a1 * c[e] - a2 * s[e];
                    a[2 * e + 1] = a2 * c[e] + a1 * s[e];
                    b[2 * e] = b1 * c[e + 4] - b2 * s[e + 4];
                    b[2 * e + 1] = b2 * c[e + 4] + b1 * s[e + 4];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = a[e], y = b[e];
                    a[e] = x * c[e] - y * s[e];
                    b[e] = y * c[e] + x * s[e];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            xa[u][e] = (__bf16)a[e];
            xb[u][e] = (__bf16)b[e];
        }
    }
    const bool stored = !p.slots || (slot >= 0 && slot < p.capacity);
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int h = h0 + u * ROWS;
        if (kind[u] == 3 || (kind[u] > 0 && !stored)) continue;
        __bf16* y;
        if (kind[u] == 0) y = p.q_out + (t * p.hq + h) * D;
        else if (!p.slots) y = p.k_out + (t * p.hkv + (h - p.hq)) * D;
        else if (kind[u] == 1) y = p.k_out + pg * p.k_page + entry * p.k_row + (h - p.hq) * p.kh_out;
        else y = p.v_out + pg * p.v_page + entry * p.v_row + (h - p.hq - p.hkv) * p.vh_out;
        *(bf16x8*)(y + a0) = xa[u];
        *(bf16x8*)(y + b0) = xb[u];
    }
}

template <int D>
int launch(Params p, hipStream_t s) {
    constexpr int ROWS = 1024 / D;
    // Few tokens: a wave per (1,024 / d) heads, so that nothing waits in line; many: four times as much per wave, whose loads go out together
    // (us, narrow / wide: 16 + 8 + 8 heads of 256 dims, 300 tokens 5.4 / 7.7, 700 7.6 / 8.8, 2,000 16.3 / 15.8, 8,000 49.4 / 48.8; 32 + 16 + 16 of 128, 16,000 107.5 / 105.1).
    const int units = (p.heads + ROWS - 1) / ROWS;
    const bool wide = p.T * units >= 8192;
    p.parts = wide ? (units + 3) / 4 : units;
    const long waves = p.T * p.parts;
    if (waves > INT32_MAX - 4) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: %ld tokens are too many", p.T);
    const dim3 grid((unsigned)((waves + 3) / 4));
    if (wide) hipLaunchKernelGGL((qk_norm_rope_kernel<D, 4>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<D, 1>), grid, dim3(256), 0, s, p);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPINF_OK : spinf_fail(SPINF_E_HIP, "qk_norm_rope: launch: %s", hipGetErrorString(e));
}

}  // namespace

extern "C" int spinf_qk_norm_rope(const spinf_rope_args* a, void* stream) {
    if (!a) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: null args");
    const bool put = a->slots != nullptr;
    if (a->T < 0 || a->T > (1 << 30) || a->hq <= 0 || a->hkv <= 0 || a->hq > 4096 || a->hkv > 4096) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: bad sizes (%lld tokens, %d / %d heads)", (long long)a->T, a->hq, a->hkv);
    if (a->d != 64 && a->d != 128 && a->d != 256 && a->d != 512) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: head dim %d not supported (64, 128, 256, 512)", a->d);
    if (a->rot < 0 || a->rot > a->d || a->rot % 16) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: %d of %d dims rotated (a multiple of 16)", a->rot, a->d);
    if (!(a->eps >= 0.f) || !(a->eps < INFINITY)) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: eps %g", (double)a->eps);
    if (a->T == 0) return SPINF_OK;
    if (!a->q || !a->k || !a->q_out || !a->k_out || (put && (!a->v || !a->v_out)) || (a->rot && (!a->cos || !a->sin))) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: null pointer");
    if (put && (a->page <= 0 || a->pages <= 0 || a->pages * a->page > INT32_MAX)) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: a cache of %lld pages of %d keys", (long long)a->pages, a->page);
    if (a->rot && a->n_pos <= 0) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: tables of %lld positions", (long long)a->n_pos);
    if (a->rot && !a->pos && a->n_pos < a->T) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: tables of %lld positions for %lld tokens", (long long)a->n_pos, (long long)a->T);
    for (const void* ptr : {a->q, a->k, put ? a->v : nullptr, a->wq, a->wk, a->cos, a->sin, (const void*)a->q_out, (const void*)a->k_out, put ? (const void*)a->v_out : nullptr})
        if ((uintptr_t)ptr % 16) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: tensors must be 16-byte aligned");
    for (int64_t st : {a->q_tok, a->q_head, a->k_tok, a->k_head, put ? a->v_tok : 0, put ? a->v_head : 0, put ? a->k_page : 0, put ? a->k_row : 0, put ? a->kh_out : 0, put ? a->v_page : 0,
                       put ? a->v_row : 0, put ? a->vh_out : 0})
        if (st % 8) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: strides must be multiples of 8 elements");
    const int per16 = a->cs_f32 ? 4 : 8;
    if (a->rot && (a->cos_ld % per16 || a->sin_ld % per16)) return spinf_fail(SPINF_E_ARG, "qk_norm_rope: rows of the tables must be 16-byte aligned");
    Params p = {};
    p.q = (const __bf16*)a->q; p.k = (const __bf16*)a->k; p.v = (const __bf16*)a->v;
    p.q_tok = a->q_tok; p.q_head = a->q_head; p.k_tok = a->k_tok; p.k_head = a->k_head; p.v_tok = a->v_tok; p.v_head = a->v_head;
    p.wq = a->wq; p.wk = a->wk; p.cos = a->cos; p.sin = a->sin; p.cos_ld = a->cos_ld; p.sin_ld = a->sin_ld;
    p.pos = a->pos; p.slots = (const long*)a->slots;
    p.q_out = (__bf16*)a->q_out; p.k_out = (__bf16*)a->k_out; p.v_out = (__bf16*)a->v_out;
    p.k_page = a->k_page; p.k_row = a->k_row; p.kh_out = a->kh_out; p.v_page = a->v_page; p.v_row = a->v_row; p.vh_out = a->vh_out;
    p.T = a->T; p.n_pos = a->n_pos; p.capacity = put ? a->pages * a->page : 0;
    p.hq = a->hq; p.hkv = a->hkv; p.heads = a->hq + a->hkv * (put ? 2 : 1); p.rot = a->rot; p.page = a->page;
    p.neighbours = a->neighbours; p.plus_one = a->plus_one; p.v_norm = a->v_norm; p.w_f32 = a->w_f32; p.cs_f32 = a->cs_f32; p.pos_i64 = a->pos_i64;
    p.eps = a->eps;
    hipStream_t s = (hipStream_t)stream;
    switch (a->d) {
        case 64: return launch<64>(p, s);
        case 128: return launch<128>(p, s);
        case 256: return launch<256>(p, s);
        default: return launch<512>(p, s);
    }
}
