// Tokens drawn from logits by given random numbers, for gfx950 (MI355X): temperature, top-k, top-p and min-p of every row.  The reference reads log-probs of given options
// and takes the best tokens of its extraction decoder (spinf_serve/decode.py:246-300); it draws none.
//
// Mathematics.  Order: larger logits first, of equal ones the lower index: as one number per token (the complement of its ordered bits above its index), ascending.  Weight of a
// token w = exp((x - max) / T).  Kept are the first k of the order, of these the shortest beginning that holds p of their weight, of these the tokens with w >= min_p.  The token
// drawn is the first, by index, up to which the kept weights add up to more than u times their sum.
//
// Where a border falls decides which token comes out, so weights are taken in 64 bits, and sums of them are sums of whole numbers: units of 2^-47 of the largest weight of a chunk
// (8,192 logits), the same in any order; where a border is looked for among listed tokens (8,192 at most), of the row's largest, and 2^-80 of it in a whole row.
//
// Kernels.  chunks: a chunk's largest logit, its weight, and how many logits and how much weight lie in each of 255 bins, a twelfth of T wide, below its largest one (bins at whole
// multiples, so those of chunks fit together).  rows: the bins in which the k-th token and the border of p lie.  gather: weights of what is kept for certain, and the tokens
// of the bins in question.  draw: the borders among those few, then the chunk by the chunks' weights and the token in it.  Rows without a filter need the first and the last.  Where
// bins tell too little (a border far below the largest logit, thousands of equal logits) the draw looks through the row itself: 8 rows of 262,144 equal logits, top-p: 1.3 ms.
// Where rows are many (320 of 262,144: 88 us, 61 at the rate of a copy) the chunks take 27 vector instructions a logit, nine of them of 64 bits, beside its bytes: they issue for 58 % of that kernel's time, the table of steps
// keeps LDS busy for 16 % (half of it lanes that meet in a bank), waves wait for three quarters of theirs: a workgroup loads, then computes, and only others overlap it.  Where rows are few, the four launches'
// latencies (one row: 27 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "spinf_tree.h"
#include "common.h"
#include "lanes.h"

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef unsigned long long u64;

namespace {

constexpr int LANES = 512, WAVES = LANES / 64, EACH = 16, CHUNK = LANES * EACH;
constexpr int BINS = 256;              // the last one: all below
constexpr int SEGMENT = 1024;          // tokens of a chunk that lie in the bins in question
constexpr int LISTED = 8192;           // ... of a row
constexpr int FEW = 4096;              // up to so many the first k are listed whole: their weights are taken one by one and nobody else's
constexpr int MOST_CHUNKS = 512;
constexpr float BINS_PER_UNIT = 12.f;

struct Stat { float top; unsigned at; u64 sum; };       // of a chunk: largest logit (-inf: none), where (of a row with a filter: how many can be drawn), weight
// of a row: largest logit; what to do; bins [from, to] and `kth` in question (none: BINS); tokens before the kth bin; of all and before `from` and the kth: weight; does top-p have a say
struct Row { float top; int grid, how, from, to, kth, before_k, by_mass; double sum, mass_k, mass_from; };
static_assert(sizeof(Stat) == 16 && sizeof(Row) == 56, "workspace layout");
enum { PLAIN = 0, LIST = 1, SEARCH = 2, NOTHING = 3, BEST = 4 };

struct Params {
    const void* logits; long ld; int vocab, rows, chunks; bool aligned;
    const void* u; bool u_f64;
    const float *temperature, *top_p, *min_p; const int* top_k;
    float all_temperature, all_top_p, all_min_p; int all_top_k; double all_inv;   // (1 / T of all: a division of 64 bits was a tenth of a chunk's work)
    long* token; float* prob;
    Stat* stat; Row* row; int* hist_n; u64* hist_w; u64* kept; int* count; uint2* list;
};

struct How { double inv, by_two; float scale, far, p, least; int k; bool best, wrong, filtered, few, plain; };
__device__ __forceinline__ How settings(const Params& p, int row) {
    How h;
    const float T = p.temperature ? p.temperature[row] : p.all_temperature;
    h.p = p.top_p ? p.top_p[row] : p.all_top_p;
    h.least = p.min_p ? p.min_p[row] : p.all_min_p;
    h.k = p.top_k ? p.top_k[row] : p.all_top_k;
    h.wrong = !(T >= 0.f) || !(h.p >= 0.f) || !(h.least >= 0.f);
    h.best = T == 0.f;
    h.inv = p.temperature ? 1.0 / (double)T : p.all_inv;
    h.by_two = h.inv * 1.4426950408889634;
    h.scale = fminf(fmaxf(BINS_PER_UNIT / T, 0x1p-126f), 3e38f);   // (T infinite: an infinite logit times 0 would have no place)
    h.far = 60.f * T;
    h.plain = T < 1e36f;   // (far is finite)
    if (h.k <= 0 || h.k >= p.vocab) h.k = 0;
    if (h.p == 0.f) {   // the first alone
        h.p = 1.f;
        h.k = 1;
    }
    if (h.k == 1) h.best = true;
    h.least = fminf(h.least, 1.f);   // (what weighs as much as the largest stays: under an infinite T that is all finite ones)
    h.filtered = h.k || h.p < 1.f || h.least > 0.f;
    h.few = h.k && h.k <= FEW;
    return h;
}

__device__ __forceinline__ unsigned ordered(float x) {   // larger for larger x
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ float value(u64 number) { return unordered(~(unsigned)(number >> 32)); }
__device__ __forceinline__ u64 number(float x, unsigned at) { return (u64)~ordered(x + 0.f) << 32 | at; }   // smaller: earlier in the order (zeros are equal whatever their sign)

// a token's place on the grid of bins; never falls as x grows
__device__ __forceinline__ int place(float x, float scale) { return (int)floorf(__builtin_amdgcn_fmed3f(x * scale, -1e9f, 1e9f)); }

// 2^t, t <= 0: the whole part by the exponent, the rest (at most a half) by the series of exp, whose 13th term is 2^-52 of the sum
__device__ __forceinline__ double power(double t) {
    t = fmax(t, -1000.0);
    const double whole = t + 0x1.8p52, f = t - (whole - 0x1.8p52);   // (the nearest whole number, in the last bits)
    double c[13] = {1.0};
#pragma unroll
    for (int k = 1; k <= 12; k++) c[k] = c[k - 1] * (0.69314718055994530942 / k);
    double y = c[12];
#pragma unroll
    for (int k = 11; k >= 0; k--) y = __builtin_fma(y, f, c[k]);
    return __longlong_as_double(__double_as_longlong(y) + ((long long)(int)__double_as_longlong(whole) << 52));
}
// The same for a chunk's logits, where vector instructions are what takes longest beside the loads.  With t = x / (T ln 2) in 256ths and B the whole number next to the
// largest logit's t: n = round(t) - B and what is left of t come of one product-and-sum each, exact but for the last bits; 2^(n / 256) by a table in LDS and the exponent, the rest by a
// polynomial of degree 3 through the Chebyshev points of -1/2 .. 1/2 (off by 2^-45.7 at most), whose coefficients hold what the largest logit's own t is off from B: it weighs 1 to
// 2^-44.  (320 rows of 262,144 logits: 90 us in all.  With differences from the largest logit, 32nds and degree 4 99, with the series above 120, with the library's exp 195.)
constexpr int STEPS = 256;
struct Steps { double of[STEPS]; };
constexpr Steps make_steps() {   // 2^(j / 256) by its series, the smallest terms first
    Steps s = {};
    for (int j = 0; j < STEPS; j++) {
        double term[18] = {1.0}, y = 0.0;
        for (int k = 1; k < 18; k++) term[k] = term[k - 1] * (j * (0.69314718055994530942 / STEPS) / k);
        for (int k = 17; k >= 0; k--) y += term[k];
        s.of[j] = y;
    }
    return s;
}
__constant__ const Steps all_steps = make_steps();
__device__ __forceinline__ void fill_steps(double* steps) {
    static_assert(STEPS <= LANES, "one a lane");
    if (threadIdx.x < STEPS) steps[threadIdx.x] = all_steps.of[threadIdx.x];
}
struct Weights {   // of a chunk, by its largest logit
    const double* steps; double by_step, magic; float low;
    double c0, c1, c2, c3;
    __device__ __forceinline__ Weights(const double* steps, float top, const How& h) : steps(steps), by_step(h.by_two * STEPS), low(fminf(top - h.far, nextafterf(top, -INFINITY))) {
        const double B = __builtin_rint(top * by_step), g = part(__builtin_fma(-(double)top, by_step, B), C0, C1, C2, C3);
        magic = 0x1.8p52 - B;
        c0 = g * C0; c1 = g * C1; c2 = g * C2; c3 = g * C3;
    }
    // (where the next number below the largest lies hundreds of T away, the exponent would not hold its weight; beyond 2^30 steps the whole number its place; where there is no number 60 T below the largest, masked logits
    // would have no weight to be given)
    static __device__ __forceinline__ bool fits(float top, const How& h) {
        return h.plain && fabs(top * (h.by_two * STEPS)) < 0x1p30 && top - nextafterf(top, -INFINITY) <= 8.f * h.far && top - h.far > -INFINITY;
    }
    // exp((x - top) / T) to 2^-44 of it; of what lies some 60 T and more below, and of NaN: less than 2^-70
    __device__ __forceinline__ double of(float x) const {
        const double t = fmaxf(x, low), whole = __builtin_fma(t, by_step, magic), f = __builtin_fma(t, by_step, magic - whole);
        const int n = (int)__double_as_longlong(whole);
        const double y = part(f, c0, c1, c2, c3) * steps[n & (STEPS - 1)];
        return __hiloint2double(__double2hiint(y) + ((n & ~(STEPS - 1)) << 12), __double2loint(y));   // (n / 256 into the exponent)
    }
    static __device__ __forceinline__ double part(double f, double c0, double c1, double c2, double c3) { return __builtin_fma(__builtin_fma(__builtin_fma(c3, f, c2), f, c1), f, c0); }
    static constexpr double C0 = 0.9999999999999825, C1 = 0.0027076061740622767, C2 = 3.6655661567589336e-06, C3 = 3.308302983711395e-09;
};
// exp((x - top) / T); where the largest are infinite, only they have a weight
__device__ __forceinline__ double weight(float x, float top, double by_two) { return x == top ? 1.0 : top == INFINITY || x == -INFINITY ? 0.0 : power(((double)x - (double)top) * by_two); }
// in units of 2^-47: the last bits of w + 32, rounded there
__device__ __forceinline__ u64 units(double w) { return (u64)(__double_as_longlong(w + 32.0) - __double_as_longlong(32.0)); }
constexpr double UNIT = 0x1p-47;
// units of a chunk's (or, by a row's largest logit, a row's) logits, the same in every kernel
struct Units {
    Weights w; float top; double by_two; bool fits;
    __device__ __forceinline__ Units(const double* steps, float top, const How& h) : w(steps, top, h), top(top), by_two(h.by_two), fits(Weights::fits(top, h)) {}
    __device__ __forceinline__ u64 of(float x) const { return fits ? units(w.of(x)) : units(weight(x, top, by_two)); }
};

template <bool BF16>
__device__ __forceinline__ float load1(const Params& p, int row, int i) {
    const long at = (long)row * p.ld + i;
    return BF16 ? (float)((const __bf16*)p.logits)[at] : ((const float*)p.logits)[at];
}
template <bool BF16>
constexpr int VEC = BF16 ? 8 : 4;
// index of a lane's e-th logit
template <bool BF16>
__device__ __forceinline__ int index_of(int chunk, int e) { return chunk * CHUNK + (e / VEC<BF16> * LANES + (int)threadIdx.x) * VEC<BF16> + e % VEC<BF16>; }
template <bool BF16>
__device__ __forceinline__ float load_one(const Params& p, int row, int i) { return i < p.vocab ? fmaxf(load1<BF16>(p, row, i), -INFINITY) : -INFINITY; }
template <bool BF16>
__device__ __forceinline__ void load_vec(const Params& p, int row, int at, float* x) {   // 16 bytes, aligned
    if (BF16) {
        const bf16x8 y = *(const bf16x8*)((const __bf16*)p.logits + (long)row * p.ld + at);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = (float)y[j];
    } else {
        const float4 y = *(const float4*)((const float*)p.logits + (long)row * p.ld + at);
        x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
    }
}
template <bool BF16>
__device__ __forceinline__ void load(const Params& p, int row, int chunk, float (&x)[EACH]) {
    constexpr int V = VEC<BF16>;
#pragma unroll
    for (int i = 0; i < EACH / V; i++) {
        const int at = index_of<BF16>(chunk, i * V);
        if (p.aligned && at + V <= p.vocab) {
            load_vec<BF16>(p, row, at, x + i * V);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) x[i * V + j] = at + j < p.vocab ? load1<BF16>(p, row, at + j) : -INFINITY;
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) x[e] = fmaxf(x[e], -INFINITY);   // (NaN: never drawn)
}

template <class T, class F>
__device__ __forceinline__ T over_all(T x, T* room, F f) {   // room: one place per wave
    x = over_lanes(x, f);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = x;
    __syncthreads();
    x = room[0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) x = f(x, room[w]);
    return x;
}
__device__ __forceinline__ u64 sum_all(u64 x, u64* room) { return over_all(x, room, [](u64 a, u64 b) { return a + b; }); }
__device__ __forceinline__ float top_all(float x, float* room) { return over_all(x, room, [](float a, float b) { return fmaxf(a, b); }); }
// what the lanes up to this one hold, itself counted in, always added in the same order; total: of all
template <class T>
__device__ __forceinline__ T scan_all(T x, T* room, T& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) room[wave] = x;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        if (w == wave) before = total;
        total += room[w];
    }
    return before + x;
}

template <bool BF16, bool FILTERS>   // FILTERS: some row may have one (without, fewer registers: 4 workgroups to a CU where it would be 3)
__global__ __launch_bounds__(LANES, FILTERS ? 6 : 8) void sample_chunks_kernel(const Params p) {
    __shared__ u64 room[WAVES];
    __shared__ u64 weights[FILTERS ? BINS : 1];
    __shared__ int numbers[FILTERS ? BINS : 1];
    __shared__ double steps[STEPS];
    const int chunk = blockIdx.x, row = blockIdx.y;
    const How h = settings(p, row);
    if (h.wrong) return;
    float x[EACH];
    load<BF16>(p, row, chunk, x);
    const long at = (long)row * p.chunks + chunk;
    fill_steps(steps);   // (read behind the barriers of top_all)
    if (h.best) {
        u64 first = ~0ull;   // the least number of the chunk
#pragma unroll
        for (int e = 0; e < EACH; e++) first = std::min(first, number(x[e], index_of<BF16>(chunk, e)));
        first = over_all(first, (u64*)room, [](u64 a, u64 b) { return a < b ? a : b; });
        if (threadIdx.x == 0) p.stat[at] = {unordered(~(unsigned)(first >> 32)), (unsigned)first, 0};
        return;
    }
    float top = x[0];
#pragma unroll
    for (int e = 1; e < EACH; e++) top = fmaxf(top, x[e]);
    top = top_all(top, (float*)room);
    Stat s = {top, 0, 0};
    if (top == -INFINITY) {   // (an empty chunk's bins are not looked at)
        if (threadIdx.x == 0) p.stat[at] = s;
        return;
    }
    if (!FILTERS || !h.filtered) {
        double sum = 32.0;   // (16 weights of at most 1 leave it below 64: it counts in units of 2^-47)
        if (Weights::fits(top, h)) {
            const Weights w(steps, top, h);
#pragma unroll
            for (int e = 0; e < EACH; e++) sum += w.of(x[e]);
        } else {
#pragma unroll 1
            for (int e = 0; e < EACH; e++) sum += weight(load_one<BF16>(p, row, index_of<BF16>(chunk, e)), top, h.by_two);
        }
        s.sum = sum_all((u64)(__double_as_longlong(sum) - __double_as_longlong(32.0)), room);
        if (threadIdx.x == 0) p.stat[at] = s;
        return;
    }
    if constexpr (FILTERS) {
    if (threadIdx.x < BINS) {
        weights[threadIdx.x] = 0;
        numbers[threadIdx.x] = 0;
    }
    __syncthreads();
    const int grid = place(top, h.scale);
    if (h.few) {   // counts alone
        int there = 0;   // logits that can be drawn
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            there += x[e] > -INFINITY;
            const int b = grid - place(x[e], h.scale);
            if (x[e] > -INFINITY && b < BINS - 1) atomicAdd(&numbers[b], 1);
        }
        there = over_all(there, (int*)room, [](int a, int b) { return a + b; });   // (its barriers are behind the bins' last addition)
        if (threadIdx.x == 0) p.stat[at] = {top, (unsigned)there, 0};
        if (threadIdx.x < BINS) p.hist_n[at * BINS + threadIdx.x] = numbers[threadIdx.x];
        return;
    }
    const auto take = [&](float x, u64 w) __attribute__((always_inline)) {
        const bool on = x > -INFINITY;
        if (h.k) s.at += on;
        const int b = grid - place(x, h.scale);
        if (on && b < BINS - 1) {
            atomicAdd(&weights[b], w);
            if (h.k) atomicAdd(&numbers[b], 1);
        } else s.sum += w;   // (what lies in bins is added up from these)
    };
    if (Weights::fits(top, h)) {
        const Weights w(steps, top, h);
#pragma unroll
        for (int e = 0; e < EACH; e++) take(x[e], units(w.of(x[e])));
    } else {
#pragma unroll 1
        for (int e = 0; e < EACH; e++) {
            const float y = load_one<BF16>(p, row, index_of<BF16>(chunk, e));
            take(y, units(weight(y, top, h.by_two)));
        }
    }
    __syncthreads();
    s.sum = sum_all(s.sum + (threadIdx.x < BINS ? weights[threadIdx.x] : 0), room);
    if (h.k) s.at = over_all((int)s.at, (int*)room, [](int a, int b) { return a + b; });
    if (threadIdx.x == 0) p.stat[at] = s;
    if (threadIdx.x < BINS) {
        p.hist_w[at * BINS + threadIdx.x] = weights[threadIdx.x];
        if (h.k) p.hist_n[at * BINS + threadIdx.x] = numbers[threadIdx.x];
    }
    }
}

// A row's chunks, one per lane: the largest logit of all; factor: what a unit of a chunk's weights is worth of the row's largest weight
__device__ __forceinline__ float stage(const Params& p, int row, const How& h, Stat& s, float* tops, double* factor, float* room) {
    s = {-INFINITY, 0, 0};
    if ((int)threadIdx.x < p.chunks && !h.wrong) s = p.stat[(long)row * p.chunks + threadIdx.x];
    const float top = top_all(s.top, room);
    if ((int)threadIdx.x < p.chunks) {
        tops[threadIdx.x] = s.top;
        factor[threadIdx.x] = s.top == -INFINITY || h.best ? 0.0 : weight(s.top, top, h.by_two) * UNIT;
    }
    __syncthreads();
    return top;
}

__global__ __launch_bounds__(LANES) void sample_rows_kernel(const Params p) {
    static_assert(LANES == 2 * BINS && LANES >= MOST_CHUNKS, "two lanes a bin, one a chunk");
    __shared__ double masses[BINS], room[WAVES];
    __shared__ int counts[BINS], room_n[WAVES];
    __shared__ int found[4];
    __shared__ float tops[MOST_CHUNKS];
    __shared__ double factor[MOST_CHUNKS];
    const int row = blockIdx.x, tid = threadIdx.x, b = tid & (BINS - 1), half = tid / BINS;
    const How h = settings(p, row);
    Row r = {};
    Stat mine;
    r.top = stage(p, row, h, mine, tops, factor, (float*)room);
    r.how = r.top == -INFINITY ? NOTHING : h.best ? BEST : PLAIN;
    if (r.how != PLAIN || !h.filtered) {
        if (tid == 0) p.row[row] = r;
        return;
    }
    r.grid = place(r.top, h.scale);
    if (tid < 4) found[tid] = tid < 3 ? BINS : 0;
    __syncthreads();
    if (mine.top > -INFINITY) atomicAdd(&found[3], (int)mine.at);
    double mass = 0.0;
    int n = 0, above = 0, below = BINS;   // bins of min-p's border, and of two numbers to either side of it
    {   // (the halves' chunks and their order are always the same)
        constexpr int AHEAD = 16;
        for (int c0 = half; c0 < p.chunks; c0 += 2 * AHEAD) {
            u64 w[AHEAD];
            int m[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int c = c0 + 2 * i;
                int x = BINS;
                if (c < p.chunks && tops[c] > -INFINITY) x = b - (r.grid - place(tops[c], h.scale));
                const long at = ((long)row * p.chunks + c) * BINS + x;
                const bool on = x >= 0 && x < BINS - 1 && b < BINS - 1;
                w[i] = on && !h.few ? p.hist_w[at] : 0;
                m[i] = on && h.k ? p.hist_n[at] : 0;
            }
            if (c0 == half && h.least > 0.f && !h.few) {   // (while the bins are on their way)
                const double border = (double)r.top + log((double)h.least) / h.inv;
                if (border == border && r.top < INFINITY) {
                    float x = (float)fmin(fmax(border, -0x1.fffffep127), 0x1.fffffep127), up = x, down = x;
                    for (int i = 0; i < 2; i++) {
                        up = nextafterf(up, INFINITY);
                        down = nextafterf(down, -INFINITY);
                    }
                    above = std::max(0, r.grid - place(up, h.scale));
                    below = std::max(0, r.grid - place(down, h.scale));
                }
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                n += m[i];
                if (w[i]) mass += factor[c0 + 2 * i] * (double)w[i];
            }
        }
    }
    if (half) {
        masses[b] = mass;
        counts[b] = n;
    }
    __syncthreads();
    if (!half) {
        mass += masses[b];
        n += counts[b];
    }
    const int there = found[3], k = h.k < there ? h.k : 0;
    const bool in = !half && b < BINS - 1;
    r.kth = BINS;
    if (h.k) {
        const int own = n;
        int all;
        n = scan_all(half ? 0 : n, room_n, all);   // tokens up to the bin
        if (!half) counts[b] = n;
        if (in && n >= k && n - own < k) found[2] = b;
        __syncthreads();
        r.kth = found[2];
    }
    if (h.few) {
        r.how = k && r.kth == BINS ? SEARCH : LIST;   // (the k-th lies below the bins)
        r.to = k ? r.kth : INT_MAX;                   // (all that can be drawn are the first k)
        r.kth = k ? r.kth : BINS;
        r.before_k = k && r.kth < BINS && r.kth ? counts[r.kth - 1] : 0;
        r.by_mass = h.p < 1.f;
        if (tid == 0) p.row[row] = r;
        return;
    }
    r.sum = over_all(tid < p.chunks ? factor[tid] * (double)mine.sum : 0.0, room, [](double a, double b) { return a + b; });
    double all;
    mass = scan_all(half ? 0.0 : mass, room, all);   // weight up to the bin
    if (!half) masses[b] = mass;
    __syncthreads();
    double low = r.sum, high = r.sum;   // the weight of the first k lies between
    if (r.kth < BINS) {
        high = masses[r.kth];
        low = r.kth ? masses[r.kth - 1] : 0.0;
    }
    if (h.p < 1.f && in) {   // (what the sums' rounding could move across a border is in question too)
        if (mass >= (double)h.p * low * (1.0 - 1e-10)) atomicMin(&found[0], b);
        if (mass >= (double)h.p * high * (1.0 + 1e-10)) atomicMin(&found[1], b);
    }
    __syncthreads();
    if (tid) return;
    r.how = k && r.kth == BINS ? SEARCH : LIST;
    r.by_mass = h.p < 1.f;
    r.from = r.to = r.kth;
    if (r.by_mass) {
        r.to = std::min(found[1], r.kth);
        r.from = std::min(found[0], r.to);
        if (r.to == BINS) r.how = SEARCH;
    }
    if (h.least > 0.f && r.how == LIST) {
        if (below < r.from) {   // it decides alone
            r.from = above;
            r.to = below;
            r.kth = BINS;
            r.by_mass = 0;
        } else {
            r.from = std::min(r.from, above);
            if (r.from < BINS && r.to >= BINS - 1 && r.kth == BINS) r.how = SEARCH;   // (it lies below the bins, and nothing else decides)
        }
    }
    if (r.from >= BINS - 1) r.how = SEARCH;
    if (r.how == LIST) {
        if (r.kth < BINS) {
            r.before_k = r.kth ? counts[r.kth - 1] : 0;
            r.mass_k = low;
        }
        r.mass_from = r.from > 0 ? masses[r.from - 1] : 0.0;
    }
    p.row[row] = r;
}

template <bool BF16>
__global__ __launch_bounds__(LANES) void sample_gather_kernel(const Params p) {
    __shared__ u64 room[WAVES];
    __shared__ int n;
    const int chunk = blockIdx.x, row = blockIdx.y;
    const Row r = p.row[row];
    if (r.how != LIST) return;
    const long at = (long)row * p.chunks + chunk;
    const float top = p.stat[at].top;
    if (threadIdx.x == 0) n = 0;
    __syncthreads();
    const How h = settings(p, row);
    const int begin = top == -INFINITY ? INT_MAX : r.grid - place(top, h.scale);   // its first bin
    u64 kept = begin < r.from && (int)threadIdx.x < std::min(r.from - begin, BINS - 1) ? p.hist_w[at * BINS + threadIdx.x] : 0;   // all of the bins ahead of those in question
    if (begin <= r.to || begin == r.kth || (begin < r.kth && r.kth < BINS)) {
        float x[EACH];
        load<BF16>(p, row, chunk, x);
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int b = r.grid - place(x[e], h.scale);
            if (x[e] > -INFINITY && b >= r.from && (b <= r.to || b == r.kth)) {
                const int i = atomicAdd(&n, 1);
                if (i < SEGMENT) p.list[at * SEGMENT + i] = make_uint2(ordered(x[e] + 0.f), index_of<BF16>(chunk, e));
            }
        }
    }
    kept = sum_all(kept, room);   // (its barriers are behind the last count)
    if (threadIdx.x == 0) {
        p.kept[at] = kept;
        p.count[at] = n;
    }
}

// What tokens are worth in a sum: weights of a list, or counts, in `whole`, whatever their unit is; of a row's up to 2^22 tokens 2^40ths of its largest weight in `whole` and what is left of them in
// 2^40ths of that in `rest` (signed), so that a sum stays below 2^63 and is off by 2^-59 at most.  (Top-p below 1 leaves 2^-24 of the weight behind its border at least, which among 2^22 tokens is one of 2^-46 at the border:
// with units of 2^-38 alone, tails of equal logits 20 T and more below the largest were rounded to few units or none.)
typedef unsigned __int128 u128;
constexpr int REST = 40;
struct Worth {
    u64 whole, rest;
    static __device__ __forceinline__ Worth of(double w) {   // the last bits of w + 2^12 and of what that leaves + 2^-28, rounded there
        const double up = w + 0x1p12, left = w - (up - 0x1p12);
        return {(u64)(__double_as_longlong(up) - __double_as_longlong(0x1p12)), (u64)(__double_as_longlong(left + 0x1.8p-28) - __double_as_longlong(0x1.8p-28))};
    }
    __device__ __forceinline__ u128 all() const { return ((u128)whole << REST) + (u128)(__int128)(long long)rest; }
};
// the least whole number that is at least p times x; p below 1, x below 2^104
__device__ __forceinline__ u128 share(float p, u128 x) {
    const unsigned b = __float_as_uint(p), e = b >> 23, m = (b & 0x7fffff) | (e ? 0x800000 : 0);
    const int down = 150 - (int)(e ? e : 1);   // p = m / 2^down
    const u64 low = (u64)x, high = (u64)(x >> 64);
    const u128 y = ((u128)(high * m + __umul64hi(low, m)) << 64) + (u128)(low * m);
    return down < 127 ? (y + (((u128)1 << down) - 1)) >> down : (u128)(y != 0);
}

// The least number up to which (it counted in) those of `each` hold at least `need` in all; ~0: all of them hold less.  each(f) calls f(number, worth) for every one in question,
// each lane for its share; worth() is what it counts (rests: there are some); `some`: a number next to them.  By 256 stretches of them (`stretch`, where there is one, never falls from one number to a later one: floats near
// zero differ in all of their bits, and lie close together), then by eight bits from the first that differs among those that are left (bf16 has few values to a bin: what is left may differ in its index
// alone), until they are few and counted against each other.
constexpr int LEFT = 64;
struct SearchRoom { u64 whole[256], rest[256], one[256], found[4]; int counts[256]; };   // found: the digit or number, how many of the few are placed, what is still needed
template <class E, class S>
__device__ __forceinline__ u64 search(u128 need, u64 some, bool stretches, bool rests, SearchRoom& at, u64* room, E each, S stretch) {
    u64 known = 0, prefix = some;
    int line = -1;   // the stretch, once it is known
    const auto sum_of = [&](int d) __attribute__((always_inline)) { return Worth{at.whole[d], at.rest[d]}.all(); };
#pragma unroll 1
    while (true) {
        const bool by_stretch = stretches && line < 0;
        const auto in = [&](u64 c) __attribute__((always_inline)) { return ((c ^ prefix) & known) == 0 && (line < 0 || stretch(c) == line); };
        u64 bits = 0;
        int low = 0;
        if (!by_stretch) {
            u64 open = 0;
            each([&](u64 c, auto) __attribute__((always_inline)) { open |= in(c) ? c ^ prefix : 0; });
            open = over_all(open, room, [](u64 a, u64 b) { return a | b; });
            const int top = 63 - __builtin_clzll(open | 1);
            low = top > 7 ? top - 7 : 0;
            bits = ~0ull << low & (~0ull >> (63 - top));
        }
        __syncthreads();
        if (threadIdx.x < 256) {
            at.whole[threadIdx.x] = at.rest[threadIdx.x] = 0;
            at.counts[threadIdx.x] = 0;
        }
        if (threadIdx.x == 0) {
            at.found[0] = ~0ull;
            at.found[1] = 0;
        }
        __syncthreads();
        each([&](u64 c, auto worth) __attribute__((always_inline)) {
            if (!in(c)) return;
            const int digit = by_stretch ? stretch(c) : (int)((c & bits) >> low);
            const Worth w = worth();
            atomicAdd(&at.whole[digit], w.whole);
            if (rests) atomicAdd(&at.rest[digit], w.rest);
            atomicAdd(&at.counts[digit], 1);
            at.one[digit] = c;   // (any of them)
        });
        __syncthreads();
        if (threadIdx.x < 64) {   // four digits a lane
            const int d0 = 4 * threadIdx.x;
            const auto upto = [&](const u64 (&x)[256]) __attribute__((always_inline)) {
                u64 y = x[d0] + x[d0 + 1] + x[d0 + 2] + x[d0 + 3];
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const u64 z = __shfl_up(y, d);
                    if ((int)threadIdx.x >= d) y += z;
                }
                return y;
            };
            const u128 end = Worth{upto(at.whole), rests ? upto(at.rest) : 0}.all();
            u128 before = end - sum_of(d0) - sum_of(d0 + 1) - sum_of(d0 + 2) - sum_of(d0 + 3);
            if (before < need && end >= need) {
                int d = d0;
                while (before + sum_of(d) < need) before += sum_of(d++);
                at.found[0] = d;
                at.found[2] = (u64)(need - before);
                at.found[3] = (u64)((need - before) >> 64);
            }
        }
        __syncthreads();
        const u64 digit = at.found[0];
        if (digit == ~0ull) return ~0ull;   // (of the first pass alone)
        need = (u128)at.found[3] << 64 | at.found[2];
        const int left = at.counts[digit];
        if (left > LEFT) {   // (no two numbers are equal: it ends)
            prefix = at.one[digit];   // (its bits up to here are the number's)
            if (by_stretch) line = (int)digit;
            else known |= bits;
            continue;
        }
        __syncthreads();   // (`one` and the sums take the few)
        each([&](u64 c, auto worth) __attribute__((always_inline)) {
            if (!in(c) || digit != (u64)(by_stretch ? stretch(c) : (int)((c & bits) >> low))) return;
            const int i = (int)atomicAdd(&at.found[1], 1);
            const Worth w = worth();
            at.one[i] = c;
            at.whole[i] = w.whole;
            at.rest[i] = w.rest;
        });
        __syncthreads();
        if ((int)threadIdx.x < left) {
            const u64 c = at.one[threadIdx.x];
            Worth ahead = {0, 0};
#pragma unroll 4
            for (int i = 0; i < left; i++) {
                ahead.whole += at.one[i] < c ? at.whole[i] : 0;
                if (rests) ahead.rest += at.one[i] < c ? at.rest[i] : 0;
            }
            const u128 before = ahead.all();
            if (before < need && before + sum_of(threadIdx.x) >= need) at.found[0] = c;
        }
        __syncthreads();
        return at.found[0];
    }
}

template <bool BF16, bool FILTERS>
__global__ __launch_bounds__(LANES) void sample_draw_kernel(const Params p) {
    __shared__ u64 room[WAVES];
    __shared__ u64 listed[FILTERS ? LISTED : 1], worth[FILTERS ? LISTED : 1];   // numbers of the tokens in question, and their weights
    __shared__ u64 chunks[MOST_CHUNKS];
    __shared__ SearchRoom looked;
    __shared__ u64 found[2];
    __shared__ int begins[MOST_CHUNKS + 1], room_n[WAVES];
    __shared__ float tops[MOST_CHUNKS];
    __shared__ double factor[MOST_CHUNKS], target[2], steps[STEPS];
    const int row = blockIdx.x, tid = threadIdx.x;
    const How h = settings(p, row);
    Row r = {};
    if (FILTERS) r = p.row[row];
    // (what does not depend on anything is asked for at once: every wait for memory is a microsecond of a row's time)
    const long mine_at = (long)row * p.chunks + tid;
    const int own_count = FILTERS && tid < p.chunks ? p.count[mine_at] : 0;
    const u64 own_kept = FILTERS && tid < p.chunks ? p.kept[mine_at] : 0;
    const double given = p.u_f64 ? ((const double*)p.u)[row] : (double)((const float*)p.u)[row];
    fill_steps(steps);   // (read behind the barriers of stage)
    Stat own;
    r.top = stage(p, row, h, own, tops, factor, (float*)room);
    if (!FILTERS) r.how = r.top == -INFINITY ? NOTHING : h.best ? BEST : PLAIN;
    if (r.how == NOTHING || r.how == BEST) {   // (chunks lie in the order of their indices)
        const u64 first = r.how == BEST ? over_all(own.top == r.top ? (u64)own.at : ~0ull, room, [](u64 a, u64 b) { return a < b ? a : b; }) : ~0ull;
        if (tid == 0) {
            p.token[row] = (long)first;
            if (p.prob) p.prob[row] = r.how == BEST ? 1.f : 0.f;
        }
        return;
    }
    const double least = h.least > 0.f ? log((double)h.least) : -INFINITY;
    const auto stays = [&](float x) __attribute__((always_inline)) { return !(h.least > 0.f) || x == r.top || ((double)x - (double)r.top) * h.inv >= least; };   // min-p
    u64 last = ~0ull;   // the last number that is kept
    int direct = 0;     // so many tokens in question, one a lane, are all that are kept
    u64 mine_w = 0;     // ... and this lane's weight, by its chunk
    int n = 0;          // tokens in question
    if (FILTERS && r.how == LIST) {
        const int m = own_count, upto = scan_all(m, room_n, n);
        if (tid < p.chunks) begins[tid + 1] = upto;
        if (tid == 0) begins[0] = 0;
        if (__syncthreads_or(m > SEGMENT) || n > LISTED) r.how = SEARCH;
    }
    if (FILTERS && r.how != PLAIN) {
        const bool list = r.how == LIST;
        const auto bin = [&](u64 c) __attribute__((always_inline)) { return r.grid - place(value(c), h.scale); };
        const Units by_row(steps, r.top, h);
        if (list) {
            for (int c = tid >> 6; c < p.chunks; c += WAVES)
                for (int i = begins[c] + (tid & 63); i < begins[c + 1]; i += 64) {
                    const uint2 y = p.list[((long)row * p.chunks + c) * SEGMENT + i - begins[c]];
                    listed[i] = (u64)~y.x << 32 | y.y;
                    worth[i] = by_row.of(unordered(y.x));
                }
            __syncthreads();
        }
        const bool by_number = list ? r.kth < BINS : h.k > 0, by_mass = list ? r.by_mass : h.p < 1.f;
        if (list && n <= 128) {   // each token counted against all
            const u64 x = tid < n ? listed[tid] : ~0ull, w = tid < n ? worth[tid] : 0;
            if (tid == 0) found[0] = found[1] = ~0ull;
            __syncthreads();
            if (by_number) {
                const bool on = tid < n && bin(x) == r.kth;
                int before = 0;
                if (tid < n)
                    for (int i = 0; i < n; i++) before += listed[i] < x;
                // (those of other bins come before or behind all of the kth)
                const int ahead = over_all(on ? before : INT_MAX, room_n, [](int a, int b) { return a < b ? a : b; });
                if (on && before - ahead == h.k - r.before_k - 1) found[0] = x;
                __syncthreads();
                last = found[0];
            }
            if (by_mass) {
                u64 before = 0;
                const bool on = tid < n && x <= last && (h.few || bin(x) <= r.to);
                if (tid < n)
                    for (int i = 0; i < n; i++) before += listed[i] < x ? worth[i] : 0;
                double all = r.sum;   // weight of the first k
                if (r.kth < BINS || h.few) all = (h.few ? 0.0 : r.mass_k) + UNIT * (double)sum_all(tid < n && x <= last && (h.few || bin(x) == r.kth) ? w : 0, room);
                const double need = ceil(((double)h.p * all - r.mass_from) * 0x1p47);
                const u64 least_of = need < 1.0 ? 1 : (u64)need;
                if (on && before < least_of && before + w >= least_of) found[1] = x;
                __syncthreads();
                last = std::min(last, found[1]);
            }
        } else {
            const auto of_row = [&](auto f) __attribute__((always_inline)) {   // f(logit, index) of all that can be drawn
                constexpr int AHEAD = 4;
#pragma unroll 1
                for (int i0 = tid; i0 < p.vocab; i0 += AHEAD * LANES) {
                    float x[AHEAD];
#pragma unroll
                    for (int a = 0; a < AHEAD; a++) x[a] = load_one<BF16>(p, row, i0 + a * LANES);
#pragma unroll
                    for (int a = 0; a < AHEAD; a++)
                        if (x[a] > -INFINITY) f(x[a], i0 + a * LANES);
                }
            };
            const auto fine = [&](float x) __attribute__((always_inline)) { return Worth::of(by_row.fits ? by_row.w.of(x) : weight(x, r.top, h.by_two)); };   // of a whole row
#pragma unroll 1
            for (int mass = 0; mass < 2; mass++) {
                if (mass ? !by_mass : !by_number) continue;
                const auto each = [&](auto f) __attribute__((always_inline)) {
                    if (list) {
#pragma unroll 1
                        for (int i = tid; i < n; i += LANES) {
                            const u64 c = listed[i];
                            if (mass ? c <= last && (h.few || bin(c) <= r.to) : bin(c) == r.kth) f(c, [&]() __attribute__((always_inline)) { return Worth{mass ? worth[i] : 1, 0}; });
                        }
                    } else
                        of_row([&](float x, int i) __attribute__((always_inline)) {
                            const u64 c = number(x, i);
                            if (c <= last) f(c, [&]() __attribute__((always_inline)) { return mass ? fine(x) : Worth{1, 0}; });
                        });
                };
                u128 need = (u128)(list ? h.k - r.before_k : h.k) << REST;
                if (mass && list) {
                    double mine = r.sum;   // weight of the first k
                    if (r.kth < BINS || h.few) {
                        u64 w = 0;
#pragma unroll 1
                        for (int i = tid; i < n; i += LANES)
                            if (listed[i] <= last && (h.few || bin(listed[i]) == r.kth)) w += worth[i];
                        mine = (h.few ? 0.0 : r.mass_k) + UNIT * (double)sum_all(w, room);
                    }
                    const double least_of = ceil(((double)h.p * mine - r.mass_from) * 0x1p47);
                    need = (u128)(least_of < 1.0 ? 1 : (u64)least_of) << REST;
                } else if (mass) {
                    Worth w = {0, 0};
                    of_row([&](float x, int i) __attribute__((always_inline)) {
                        if (number(x, i) > last) return;
                        const Worth y = fine(x);
                        w.whole += y.whole;
                        w.rest += y.rest;
                    });
                    w.whole = sum_all(w.whole, room);
                    w.rest = sum_all(w.rest, room);
                    need = share(h.p, w.all());
                }
                // (a list's stretches: of the bins that it comes from)
                const float begin = (float)(r.grid + 1 - (h.few ? 0 : mass ? r.from : r.kth)), wide = 256.f / (h.few ? std::min(r.kth, BINS) + 1 : mass ? r.to - r.from + 1 : 1);
                const auto stretch = [&](u64 c) __attribute__((always_inline)) { return (int)__builtin_amdgcn_fmed3f((begin - value(c) * h.scale) * wide, 0.f, 255.f); };
                last = std::min(last, search(need, number(r.top, 0), list, !list && mass, looked, room, each, stretch));
            }
        }
        // what is kept, by chunk
        if (list) {
            if (tid < p.chunks) chunks[tid] = own_kept;
            __syncthreads();
            for (int i = tid; i < n; i += LANES) {
                const float x = value(listed[i]);
                const int c = (int)((unsigned)listed[i] / CHUNK);
                if (listed[i] <= last && (h.few || bin(listed[i]) <= r.to) && stays(x)) {
                    mine_w = Units(steps, tops[c], h).of(x);
                    atomicAdd(&chunks[c], mine_w);
                }
            }
            if (h.few && n <= 128) direct = n;
        } else {
            for (int c = 0; c < p.chunks; c++) {
                u64 w = 0;
                if (tops[c] > -INFINITY) {
                    const Units by_chunk(steps, tops[c], h);
                    float x[EACH];
                    load<BF16>(p, row, c, x);
#pragma unroll
                    for (int e = 0; e < EACH; e++)
                        if (x[e] > -INFINITY && number(x[e], index_of<BF16>(c, e)) <= last && stays(x[e])) w += by_chunk.of(x[e]);
                }
                w = sum_all(w, room);
                if (tid == 0) chunks[c] = w;
            }
        }
    } else if (r.how == PLAIN) {
        if (tid < p.chunks) chunks[tid] = own.sum;
    }
    __syncthreads();
    {   // the chunk, and how much of it lies before the token
        const double mine = tid < p.chunks ? factor[tid] * (double)chunks[tid] : 0.0;
        double all;
        const double upto = scan_all(mine, (double*)room, all);
        const double u = given > 0.0 ? (given < 1.0 ? given : 1.0) : 0.0;
        const double want = u * all;
        const bool some = mine > 0.0;
        const int hit = over_all(some && upto > want ? tid : LANES, room_n, [](int a, int b) { return a < b ? a : b; });
        const int end = over_all(some ? tid : -1, room_n, [](int a, int b) { return a > b ? a : b; });
        if (tid == 0) begins[0] = -1;
        __syncthreads();
        if (tid == (hit < LANES ? hit : end)) {   // (where rounding left no chunk: the last that has any)
            begins[0] = tid;
            target[0] = (want - (upto - mine)) / factor[tid];
            target[1] = all;
        }
    }
    __syncthreads();
    const int chunk = begins[0];
    if (chunk < 0) {   // (no row comes here: its largest logit is kept)
        if (tid == 0) {
            p.token[row] = -1;
            if (p.prob) p.prob[row] = 0.f;
        }
        return;
    }
    const u64 want = target[0] > 0.0 ? (u64)target[0] : 0;
    const auto chance = [&](float x) __attribute__((always_inline)) { return (float)(weight(x, r.top, h.by_two) / target[1]); };   // (units would round a small one)
    const float top = tops[chunk];
    if (FILTERS && direct) {   // the token among those that are listed: each adds up what lies before it
        const unsigned at = tid < direct ? (unsigned)listed[tid] : 0;
        const bool here = tid < direct && mine_w && (int)(at / CHUNK) == chunk;
        if (tid < direct) worth[tid] = here ? mine_w : 0;
        __syncthreads();
        u64 before = 0;
        if (here)
            for (int i = 0; i < direct; i++) before += (unsigned)listed[i] < at ? worth[i] : 0;
        bool hit = here && before <= want && before + mine_w > want;
        if (!__syncthreads_or(hit)) {   // (where rounding left none, the last token that is kept)
            const unsigned end = over_all(here ? at + 1 : 0u, (unsigned*)room_n, [](unsigned a, unsigned b) { return a > b ? a : b; });
            hit = here && at + 1 == end;
        }
        if (hit) {
            p.token[row] = at;
            if (p.prob) p.prob[row] = chance(value(listed[tid]));
        }
        return;
    }
    // a lane's 16 logits one after the other
    const int first = chunk * CHUNK + tid * EACH;
    const auto kept = [&](float x, int i) __attribute__((always_inline)) {
        return x > -INFINITY && (r.how == PLAIN || (number(x, i) <= last && stays(x) && (r.how == SEARCH || h.few || r.grid - place(x, h.scale) <= r.to)));
    };
    u64 total, mine = 0, before = 0;
    int hit = -1, some = -1;
    const auto look = [&](int i, u64 w) __attribute__((always_inline)) {
        const u64 ahead = before;
        before += w;
        if (w) some = i;
        if (ahead <= want && before > want) hit = i;   // (of all lanes' tokens one, or none)
    };
    if (Weights::fits(top, h)) {
        const Weights by_chunk(steps, top, h);
        float x[EACH];
        u64 w[EACH];
        if (p.aligned && first + EACH <= p.vocab) {
            constexpr int V = VEC<BF16>;
#pragma unroll
            for (int i = 0; i < EACH; i += V) load_vec<BF16>(p, row, first + i, x + i);
        } else {
#pragma unroll
            for (int e = 0; e < EACH; e++) x[e] = first + e < p.vocab ? load1<BF16>(p, row, first + e) : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            x[e] = fmaxf(x[e], -INFINITY);
            w[e] = kept(x[e], first + e) ? units(by_chunk.of(x[e])) : 0;
            mine += w[e];
        }
        before = scan_all(mine, room, total) - mine;   // sums ahead of the lane
#pragma unroll
        for (int e = 0; e < EACH; e++) look(first + e, w[e]);
    } else {   // (rare: not unrolled, what is not fetched costs nothing)
        const auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll 1
            for (int i = first; i < first + EACH; i++) {
                const float x = load_one<BF16>(p, row, i);
                f(i, kept(x, i) ? units(weight(x, top, h.by_two)) : 0);
            }
        };
        each([&](int, u64 w) __attribute__((always_inline)) { mine += w; });
        before = scan_all(mine, room, total) - mine;
        each(look);
    }
    (void)total;
    if (!__syncthreads_or(hit >= 0)) {   // (where rounding left none, the last token that is kept)
        const int end = over_all(some, room_n, [](int a, int b) { return a > b ? a : b; });
        if (some == end) hit = some;
    }
    if (hit >= 0) {
        p.token[row] = hit;
        if (p.prob) p.prob[row] = chance(load1<BF16>(p, row, hit));
    }
}

struct Sizes { int64_t stat, row, hist_n, hist_w, kept, count, list, all; int chunks; };
Sizes sizes(const spinf_sample_args* a, bool filters) {
    Sizes s;
    s.chunks = (int)((a->vocab + CHUNK - 1) / CHUNK);
    const int64_t n = a->rows * s.chunks;
    int64_t at = 0;
    const auto take = [&](int64_t bytes) { const int64_t x = at; at += (bytes + 15) / 16 * 16; return x; };
    s.stat = take(n * (int64_t)sizeof(Stat));
    s.row = take(filters ? a->rows * (int64_t)sizeof(Row) : 0);
    s.hist_w = take(filters ? n * BINS * 8 : 0);
    s.hist_n = take(filters ? n * BINS * 4 : 0);
    s.kept = take(filters ? n * 8 : 0);
    s.count = take(filters ? n * 4 : 0);
    s.list = take(filters ? n * SEGMENT * 8 : 0);
    s.all = at;
    return s;
}

bool any_filter(const spinf_sample_args* a) { return a->top_k || a->top_p || a->min_p || a->all_top_k > 0 || a->all_top_p < 1.f || a->all_min_p > 0.f; }

int check(const spinf_sample_args* a, const char* what) {
    if (!a) return spinf_fail(SPINF_E_ARG, "%s: null args", what);
    if (a->rows < 0 || a->rows > 65535 || a->vocab < 1 || a->vocab > (int64_t)CHUNK * MOST_CHUNKS) return spinf_fail(SPINF_E_ARG, "%s: %lld rows (at most 65,535) of %lld logits (1 .. 2^22)", what, (long long)a->rows, (long long)a->vocab);
    if (a->dtype != 0 && a->dtype != 1) return spinf_fail(SPINF_E_ARG, "%s: dtype %d (0 = fp32, 1 = bf16)", what, a->dtype);
    if (a->ld < a->vocab) return spinf_fail(SPINF_E_ARG, "%s: rows %lld apart of %lld logits", what, (long long)a->ld, (long long)a->vocab);
    if ((!a->temperature && !(a->all_temperature >= 0.f)) || (!a->top_p && !(a->all_top_p >= 0.f)) || (!a->min_p && !(a->all_min_p >= 0.f)))
        return spinf_fail(SPINF_E_ARG, "%s: temperature %g, top-p %g, min-p %g must not be negative", what, (double)a->all_temperature, (double)a->all_top_p, (double)a->all_min_p);
    return SPINF_OK;
}

template <bool BF16>
hipError_t launch(const Params& p, bool filters, hipStream_t s) {
    if (filters) hipLaunchKernelGGL((sample_chunks_kernel<BF16, true>), dim3(p.chunks, p.rows), dim3(LANES), 0, s, p);
    else hipLaunchKernelGGL((sample_chunks_kernel<BF16, false>), dim3(p.chunks, p.rows), dim3(LANES), 0, s, p);
    hipError_t e = hipGetLastError();
    if (filters) {
        if (e == hipSuccess) {
            hipLaunchKernelGGL(sample_rows_kernel, dim3(p.rows), dim3(LANES), 0, s, p);
            e = hipGetLastError();
        }
        if (e == hipSuccess) {
            hipLaunchKernelGGL(sample_gather_kernel<BF16>, dim3(p.chunks, p.rows), dim3(LANES), 0, s, p);
            e = hipGetLastError();
        }
    }
    if (e == hipSuccess) {
        if (filters) hipLaunchKernelGGL((sample_draw_kernel<BF16, true>), dim3(p.rows), dim3(LANES), 0, s, p);
        else hipLaunchKernelGGL((sample_draw_kernel<BF16, false>), dim3(p.rows), dim3(LANES), 0, s, p);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace

extern "C" int spinf_sample_workspace(const spinf_sample_args* a, int64_t* bytes) {
    const int rc = check(a, "sample_workspace");
    if (rc) return rc;
    if (!bytes) return spinf_fail(SPINF_E_ARG, "sample_workspace: null pointer");
    *bytes = sizes(a, any_filter(a)).all;
    return SPINF_OK;
}

extern "C" int spinf_sample(const spinf_sample_args* a, void* stream) {
    const int rc = check(a, "sample");
    if (rc) return rc;
    if (a->rows == 0) return SPINF_OK;
    if (!a->logits || !a->u || !a->token) return spinf_fail(SPINF_E_ARG, "sample: null pointer");
    const bool filters = any_filter(a);
    const Sizes z = sizes(a, filters);
    if (!a->workspace || a->workspace_bytes < z.all || (uintptr_t)a->workspace % 16) return spinf_fail(SPINF_E_ARG, "sample: needs a 16-byte aligned workspace of %lld bytes", (long long)z.all);
    Params p = {};
    p.logits = a->logits; p.ld = a->ld; p.vocab = (int)a->vocab; p.rows = (int)a->rows; p.chunks = z.chunks;
    p.aligned = (uintptr_t)a->logits % 16 == 0 && a->ld % (a->dtype ? 8 : 4) == 0;
    p.u = a->u; p.u_f64 = a->u_f64 != 0;
    p.temperature = a->temperature; p.top_k = a->top_k; p.top_p = a->top_p; p.min_p = a->min_p;
    p.all_temperature = a->all_temperature; p.all_inv = 1.0 / (double)a->all_temperature; p.all_top_k = a->all_top_k; p.all_top_p = a->all_top_p; p.all_min_p = a->all_min_p;
    p.token = (long*)a->token; p.prob = a->prob;
    char* w = (char*)a->workspace;
    p.stat = (Stat*)(w + z.stat); p.row = (Row*)(w + z.row); p.hist_n = (int*)(w + z.hist_n); p.hist_w = (u64*)(w + z.hist_w);
    p.kept = (u64*)(w + z.kept); p.count = (int*)(w + z.count); p.list = (uint2*)(w + z.list);
    const hipError_t e = a->dtype ? launch<true>(p, filters, (hipStream_t)stream) : launch<false>(p, filters, (hipStream_t)stream);
    return e == hipSuccess ? SPINF_OK : spinf_fail(SPINF_E_HIP, "sample: launch: %s", hipGetErrorString(e));
}
