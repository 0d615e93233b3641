// The books of seats on the GPU, for gfx950 (MI355X): which keys go, which pages come back and are handed out, where new tokens' keys and values lie, and the work lists of the
// attention over them (seats_attn.hip), all from lengths in device memory: a recorded step can be replayed for the next one.  No counterpart in the reference, whose
// contents are read anew with every request.
//
// Mathematics: whole numbers only.  Of seat r with n_r keys the last min(drop_r, n_r) go, then new_r come.  Pages given back are pushed on a stack, pages needed are popped
// from it; with running sums over the seats (of pages back, of pages and tokens asked for) every push, pop and row has a place of its own, so the result is that of going seat by
// seat, whatever order the lanes run in.  Pushed in the reverse of the order they are popped in: a step that takes back what the last one added leaves stack and tables as they were.
//
// Bound by latency: kernels of one workgroup of 8 waves, whose lanes hold a share of the at most 2,048 seats; pages, items and rows are dealt out to lanes by a search in the sums.
//   books   three running sums over the seats; 64 seats 6 us, 1,344 seats 11
//   lists   of each head geometry in a workgroup of its own: 16 us for 24 seats below one content, 25 us for 24 x 56 (once a step for all layers).  In one kernel with the books they need
//           more registers than there are.
//   rows    over the whole GPU, where a step has more than SEATS_ROWS_AT_ONCE rows (prompts of 100,800 rows: 5 us, 12 with the books)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "spinf_tree.h"
#include "common.h"
#include "seats.h"
#include "lanes.h"

namespace {

constexpr int LANES = 512, WAVES = LANES / 64;
constexpr int LOTS = 1 << 30;   // sums stop there

struct Kind { int* wave; int* single; int* block; int* last; int* counts; int* parts; int* seat_parts; int hq, hkv, d, window, room[4]; };
struct Params {
    const int* come; const int* drop; const int* content;
    int* lens; int* table; int* free; int* left; int* first; int* took; int* stay;
    long* slots; int* pos;
    const int* shared;      // of each content: stored keys, positions of its text, first page in the page lists
    int seats, rows, page, keys, width, pool, contents, table_at, kinds;
    Kind kind[SEATS_KINDS];
};

__device__ __forceinline__ int add(int a, int b) {   // of numbers in 0 .. LOTS
    const int s = a + b;
    return s < LOTS ? s : LOTS;
}
__device__ __forceinline__ int most(int a, int b) { return a > b ? a : b; }

// Running sums over the workgroup: N values per lane -> what the lanes before hold in all, and the total
template <int N, class T, class F>
__device__ __forceinline__ void scan(T (&x)[N], T (&total)[N], long (*room)[WAVES], T none, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T y[N];
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = x[i];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
#pragma unroll
        for (int i = 0; i < N; i++) {
            const T z = __shfl_up(y[i], d);
            if (lane >= d) y[i] = f(z, y[i]);
        }
    __syncthreads();   // (the room is free)
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; i++) room[i][wave] = y[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        T before = none, all = none;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            if (w == wave) before = all;
            all = f(all, (T)room[i][w]);
        }
        const T z = __shfl_up(y[i], 1);
        x[i] = lane ? f(before, z) : before;
        total[i] = all;
    }
}

// the last r with sums[r] <= i < sums[r + 1] (sums[0] = 0, sums[n] > i)
__device__ __forceinline__ int find(const int* sums, int n, int i) {
    int a = 0, b = n;   // sums[a] <= i < sums[b]
    while (b - a > 1) {
        const int m = (a + b) >> 1;
        if (sums[m] <= i) a = m; else b = m;
    }
    return a;
}

__device__ __forceinline__ void store(int* items, int at, const SeatItem& it) {
    int4* p = (int4*)(items + sizeof(SeatItem) / 4 * (long)at);
    p[0] = make_int4(it.tok0, it.T, it.row0, it.piece);
    p[1] = make_int4(it.only, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const SeatSpan& s = it.span[i];
        p[2 + 2 * i] = make_int4(s.tab, s.L, s.kt0, s.tiles);
        p[3 + 2 * i] = make_int4(s.flo, s.fhi, s.own, 0);
    }
}

// Sums over the workgroup alone
template <int N, class T>
__device__ __forceinline__ void add_up(const T (&x)[N], T (&all)[N], long (*room)[WAVES]) {
    T y[N];
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = over_lanes<64>(x[i], [](T a, T b) { return a + b; });
    __syncthreads();   // (the room may be read still)
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; i++) room[i][threadIdx.x >> 6] = (long)y[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        all[i] = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) all[i] += (T)room[i][w];
    }
}

// Places and positions of rows.  Of more than 512 seats the first rows of each are its lane's own, later ones are searched for (1,344 seats of one row: 11 us, by search alone 12; 64 seats of
// four 6.6, by search 5.8)
constexpr int FIRST_ROWS = 4;
__device__ __forceinline__ void place_row(const Params& p, int row, int total, int seat, int first, int stay, int content) {
    long slot = -1;
    int pos = 0;
    if (row < total) {
        const int at = stay + row - first;
        const int page = p.table[p.table_at + (long)seat * p.width + at / p.page];
        slot = (long)page * p.page + at % p.page;
        pos = at + (content >= 0 && content < p.contents ? p.shared[3 * content + 1] : 0);
    }
    p.slots[row] = slot;
    p.pos[row] = pos;
}
// where a row's partial results begin
__device__ __forceinline__ void place_parts(const Params& p, const Kind& kd, int row, int total, int seat, int first) {
    const int* sp = kd.seat_parts;
    const int base = sp[2 * (row < total ? seat : p.seats)];
    kd.parts[row] = row < total ? ((base & INT_MAX) + (row - first) * sp[2 * seat + 1]) | (base & INT_MIN) : base;
}

__global__ __launch_bounds__(256) void seats_rows_kernel(const Params p) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row > p.rows) return;
    const int total = p.first[p.seats];
    const int seat = row < total ? find(p.first, p.seats, row) : 0;
    if (row < p.rows) place_row(p, row, total, seat, p.first[seat], p.stay[seat], p.content[seat]);
    for (int k = 0; k < p.kinds; k++) place_parts(p, p.kind[k], row, total, seat, p.first[seat]);
}

template <int SPT>   // seats per lane
__global__ __launch_bounds__(LANES) void seats_step_kernel(const Params p) {
    constexpr int MOST = SPT * LANES;
    __shared__ long room[2][WAVES];
    __shared__ int stay[MOST], took[MOST], content[MOST], first[MOST + 1];
    __shared__ int sums[2][MOST + 1];
    const int R = p.seats, tid = threadIdx.x;
    const auto plus = [](int a, int b) __attribute__((always_inline)) { return add(a, b); };
    const auto pages = [&](int n) __attribute__((always_inline)) { return (n + p.page - 1) / p.page; };

    // ---- what goes: pages back on the stack, the first of the order last
    int before[SPT], here[SPT], sum[1] = {0}, all[1];
#pragma unroll
    for (int i = 0; i < SPT; i++) {
        const int r = tid * SPT + i;
        before[i] = here[i] = 0;
        if (r < R) {
            int n = p.lens[r], c = p.content[r];
            n = n < 0 ? 0 : n < p.keys ? n : p.keys;
            const int d = p.drop ? p.drop[r] : 0;
            before[i] = n;
            here[i] = n - (d < 0 ? 0 : d < n ? d : n);
            stay[r] = here[i];
            content[r] = c < 0 || c >= p.contents ? -1 : c;
            sum[0] = add(sum[0], pages(n) - pages(here[i]));
        }
    }
    int left = *p.left;
    left = left < 0 ? 0 : left < p.pool ? left : p.pool;
    scan(sum, all, room, 0, plus);
#pragma unroll
    for (int i = 0; i < SPT; i++) {
        const int r = tid * SPT + i;
        if (r < R) {
            sums[0][r] = sum[0];
            sum[0] = add(sum[0], pages(before[i]) - pages(here[i]));
        }
    }
    if (tid == 0) sums[0][R] = all[0];
    __syncthreads();
    for (int i = tid; i < all[0]; i += LANES) {
        const int r = find(sums[0], R, i), to = left + all[0] - 1 - i;
        if (to < p.pool) p.free[to] = p.table[p.table_at + (long)r * p.width + pages(stay[r]) + i - sums[0][r]];
    }
    left = add(left, all[0]);
    left = left < p.pool ? left : p.pool;

    // ---- what comes: a seat asks for rows and pages where its keys have room; it gets them where what was asked up to it is there
    int ask[2] = {0, 0}, asked[2], want[SPT], need[SPT];
#pragma unroll
    for (int i = 0; i < SPT; i++) {
        const int r = tid * SPT + i, n = r < R ? p.come[r] : 0;
        want[i] = n > 0 && n <= p.keys - here[i] ? n : 0;
        need[i] = pages(here[i] + want[i]) - pages(here[i]);
        ask[0] = add(ask[0], want[i]);
        ask[1] = add(ask[1], need[i]);
    }
    scan(ask, asked, room, 0, plus);
    int got[2] = {0, 0}, given[2];
#pragma unroll
    for (int i = 0; i < SPT; i++) {
        const int r = tid * SPT + i;
        ask[0] = add(ask[0], want[i]);
        ask[1] = add(ask[1], need[i]);
        if (ask[0] > p.rows || (need[i] && ask[1] > left)) want[i] = need[i] = 0;
        got[0] += want[i];
        got[1] += need[i];
        if (r < R) took[r] = want[i];
    }
    scan(got, given, room, 0, plus);
#pragma unroll
    for (int i = 0; i < SPT; i++) {
        const int r = tid * SPT + i;
        if (r < R) {
            first[r] = got[0];
            sums[1][r] = got[1];
            p.first[r] = got[0];
            p.took[r] = want[i];
            p.stay[r] = here[i];
            p.lens[r] = here[i] + want[i];
            got[0] += want[i];
            got[1] += need[i];
        }
    }
    const int total = given[0];
    if (tid == 0) {
        first[R] = p.first[R] = total;
        sums[1][R] = given[1];
        *p.left = left - given[1];
    }
    __syncthreads();   // (also: the pages given back are on the stack)
    for (int i = tid; i < given[1]; i += LANES) {
        const int r = find(sums[1], R, i);
        p.table[p.table_at + (long)r * p.width + pages(stay[r]) + i - sums[1][r]] = p.free[left - 1 - i];
    }

    __syncthreads();
    if (p.rows > SEATS_ROWS_AT_ONCE) return;
    constexpr int BY_SEAT = SPT > 1 ? FIRST_ROWS : 0;
    bool more = SPT == 1;
    if (BY_SEAT) {
#pragma unroll
        for (int i = 0; i < SPT; i++) {
            const int r = tid * SPT + i;
            if (r < R) {
#pragma unroll
                for (int j = 0; j < BY_SEAT; j++)
                    if (j < want[i]) place_row(p, first[r] + j, total, r, first[r], stay[r], content[r]);
                more |= want[i] > BY_SEAT;
            }
        }
        more = __syncthreads_or(more);
    }
    for (int row = more ? tid : total + tid; row < p.rows; row += LANES) {
        const int seat = row < total ? find(first, R, row) : 0;
        if (row >= total || row - first[seat] >= BY_SEAT) place_row(p, row, total, seat, first[seat], stay[seat], content[seat]);
    }
}

// Running sums in place, of N arrays of n numbers in LDS at a time: a[i] becomes the sum of those before it, a[n] of all
template <int N>
__device__ __forceinline__ void running(int* const (&a)[N], int n, long (*room)[WAVES]) {
    const int per = (n + LANES - 1) / LANES, from = seats_least(n, (int)threadIdx.x * per), to = seats_least(n, from + per);
    int sum[N], all[N];
    __syncthreads();
#pragma unroll
    for (int x = 0; x < N; x++) {
        sum[x] = 0;
        for (int i = from; i < to; i++) sum[x] += a[x][i];
    }
    scan(sum, all, room, 0, [](int a, int b) { return a + b; });
#pragma unroll
    for (int x = 0; x < N; x++) {
        for (int i = from; i < to; i++) {
            const int y = a[x][i];
            a[x][i] = sum[x];
            sum[x] += y;
        }
        if (threadIdx.x == 0) a[x][n] = all[x];
    }
    __syncthreads();
}

// The work lists of a head geometry, a workgroup each.
template <int MOST>
__global__ __launch_bounds__(LANES) void seats_lists_kernel(const Params p) {
    __shared__ long room[7][WAVES];
    __shared__ int stay[MOST], took[MOST], content[MOST], first[MOST + 1], stored[MOST], listed[MOST];   // stored, listed: keys of the seat's content, where its page list begins
    __shared__ int heads[MOST + 1], low[MOST], high[MOST], of_group[MOST + 1], cut[MOST];   // of groups: seats one after the other that share their content; cut: pieces of its keys
    __shared__ int sums[5][MOST + 1];
    __shared__ int best[2];
    const int R = p.seats, tid = threadIdx.x;
    const Kind& kd = p.kind[blockIdx.x];
    const int group = kd.hq / kd.hkv, W = kd.window;
    const int far = W ? W : LOTS, deep = 128;   // rows of an item on shared tiles
    const auto each_seat = [&](auto f) __attribute__((always_inline)) {
        for (int r = tid; r < R; r += LANES) f(r);
    };
    each_seat([&](int r) __attribute__((always_inline)) {
        stay[r] = p.stay[r];
        took[r] = p.took[r];
        first[r] = p.first[r];
        const int c = p.content[r];
        const bool below = c >= 0 && c < p.contents;
        content[r] = below ? c : -1;
        stored[r] = below ? p.shared[3 * c] : 0;
        listed[r] = below ? p.shared[3 * c + 2] : 0;
        heads[r] = took[r] ? r + 1 : 0;
        low[r] = INT_MAX;
        high[r] = 0;
    });
    const int total = p.first[R];
    if (tid == 0) first[R] = total;
    const int most_rows = (long)total * kd.hq > 32 * seats_wave_places(kd.d) ? 32 : SEAT_WAVE_ROWS;   // below a content, for waves that divide the tiles
    // (a seat of many rows reads its content for itself)
    const auto alone = [&](int r) __attribute__((always_inline)) { return took[r] * group > SEAT_SHARED_ROWS; };
    // ---- tokens on few keys of their own
    const auto few_keys = [&](int r) __attribute__((always_inline)) { const int L = stay[r] + 1; return took[r] == 1 && (L < far ? L : far) <= SEAT_LAST_KEYS; };
    bool by_vector = false;
    if (seats_last(group, kd.d)) {
        long of[2] = {0, 0}, in_all[2];   // tokens, keys
        each_seat([&](int r) __attribute__((always_inline)) {
            if (few_keys(r)) {
                of[0]++;
                of[1] += seats_least(stay[r] + 1, far);
            }
        });
        add_up(of, in_all, room);
        by_vector = seats_last_pays(in_all[0], in_all[1], kd.hkv);
    }
    // ---- groups: seats with new tokens below one content, one after the other (seats without any in between do not part them)
    {   // the last seat with new tokens ahead of each: one more than its index
        const int per = (R + LANES - 1) / LANES, from = seats_least(R, tid * per), to = seats_least(R, from + per);
        int last[1] = {0}, all[1];
        __syncthreads();
        for (int r = from; r < to; r++) last[0] = most(last[0], heads[r]);
        scan(last, all, room, 0, [](int a, int b) { return a > b ? a : b; });
        for (int r = from; r < to; r++) {
            const int ahead = last[0] - 1;
            last[0] = most(last[0], heads[r]);
            of_group[r] = took[r] && (ahead < 0 || content[ahead] != content[r] || alone(r) || alone(ahead));
        }
    }
    __syncthreads();
    each_seat([&](int r) __attribute__((always_inline)) { sums[0][r] = of_group[r]; });   // (does one begin here?)
    {
        int* const a[1] = {of_group};
        running(a, R, room);   // groups that begin before the seat
    }
    const int G = of_group[R];
    __syncthreads();
    each_seat([&](int r) __attribute__((always_inline)) {
        const int begins = sums[0][r], g = of_group[r] + begins - 1;
        if (begins) heads[g] = r;   // (of a group and a seat: no seat's place in `heads` is read any more)
        of_group[r] = g;            // (means something only where the seat has new tokens)
    });
    if (tid == 0) heads[G] = R;
    __syncthreads();
    each_seat([&](int r) __attribute__((always_inline)) {   // the least and the largest place among the seats' own keys of a group's new tokens
        if (took[r]) {
            atomicMin(&low[of_group[r]], stay[r]);
            atomicMax(&high[of_group[r]], stay[r] + took[r] - 1);
        }
    });
    __syncthreads();
    // ---- what there is to do, as sets of `blocks` blocks of rows on `tiles` tiles.  Sorts: 0 waves that divide the tiles, 1 a wave to 32 rows, 2 shared tiles, 3 the last word, -1 nothing
    const auto group_set = [&](int g, int& blocks, int& tiles) __attribute__((always_inline)) {
        const int r = heads[g], c = content[r];
        blocks = tiles = 0;
        if (c < 0 || alone(r)) return -1;
        const int P = stored[r], rows = (first[heads[g + 1]] - first[r]) * group, lo = most(0, P + low[g] - far + 1);
        if (lo >= P) return -1;
        const bool few = rows <= most_rows;
        tiles = seats_up(P, PAGED_TILE) - lo / PAGED_TILE;
        blocks = seats_up(rows, few ? 32 : deep);
        return few ? 0 : 2;
    };
    // tiles: of its own keys; shared: of its content's, where it reads them itself
    const auto seat_set = [&](int r, int& blocks, int& tiles, int& shared) __attribute__((always_inline)) {
        const int n = took[r], rows = n * group, L = stay[r] + n, lo = most(0, stay[r] - far + 1);
        blocks = tiles = shared = 0;
        if (n == 0) return -1;
        tiles = seats_up(L, PAGED_TILE) - lo / PAGED_TILE;
        blocks = 1;
        if (by_vector && few_keys(r)) return 3;
        if (alone(r)) {
            const int P = stored[r], from = most(0, P + stay[r] - far + 1);
            shared = from < P ? seats_up(P, PAGED_TILE) - from / PAGED_TILE : 0;
            blocks = seats_up(rows, deep);
            return 2;
        }
        const int sort = tiles <= SEAT_SINGLE_TILES ? 1 : rows <= 32 ? 0 : 2;
        blocks = seats_up(rows, sort == 2 ? deep : 32);
        return sort;
    };
    const auto each_set = [&](auto f) __attribute__((always_inline)) {   // f(sort, blocks, tiles)
        for (int i = tid; i < R; i += LANES) {
            int blocks, tiles, shared;
            if (i < G) {
                const int sort = group_set(i, blocks, tiles);
                f(sort, blocks, tiles);
            }
            const int sort = seat_set(i, blocks, tiles, shared);
            f(sort, blocks, tiles + shared);
        }
    };
    // ---- tiles of a piece: of some sizes at and above those that make as many pieces as there are places, the one whose rounds of workgroups end first
    long work[2] = {0, 0}, all_work[2];   // by waves that divide the tiles, on shared tiles
    each_set([&](int sort, int blocks, int tiles) __attribute__((always_inline)) {
        const long n = (long)blocks * tiles;
        work[0] += sort == 0 ? n : 0;
        work[1] += sort == 2 ? n : 0;
    });
    add_up(work, all_work, room);
    if (tid < 2) best[tid] = 1;
    constexpr int SIZES = 6;
#pragma unroll
    for (int y = 0; y < 2; y++) {
        if (all_work[y] == 0) continue;
        static_assert((PAGED_PLACES & (PAGED_PLACES - 1)) == 0, "divisions by places are shifts");
        const int places = y ? seats_block_places(kd.d) : seats_wave_places(kd.d), shift = __builtin_ctz(places);
        int size[SIZES], items[SIZES], all[SIZES];
#pragma unroll
        for (int j = 0; j < SIZES; j++) {
            const long tiles = ((all_work[y] * kd.hkv * (8 + j * (j + 1) / 2) >> 3) + places - 1) >> shift;   // 1, 1 1/8, 1 3/8, 1 3/4, 2 1/4, 2 7/8
            size[j] = most(y ? SEAT_BLOCK_TILES : SEAT_WAVE_TILES, (int)(tiles < LOTS ? tiles : LOTS));
            items[j] = 0;
        }
        each_set([&](int sort, int blocks, int tiles) __attribute__((always_inline)) {
            if (sort == 2 * y)
#pragma unroll
                for (int j = 0; j < SIZES; j++) items[j] += blocks * seats_up(tiles, size[j]);
        });
        add_up(items, all, room);
        if (tid == 0) {
            long cost = LONG_MAX;
#pragma unroll
            for (int j = 0; j < SIZES; j++) {
                // (a workgroup's start and end are worth some tiles; what a piece leaves, written and read again, a 12th of a tile's time over the whole GPU: a 24th made pieces of eight tiles of 24 contents with 112 rows each, 76 us for 69)
                const long n = (long)all[j] * kd.hkv, rounds = (n + places - 1) >> shift, here = 24 * rounds * (size[j] + (y ? 4 : 12)) + (y ? 2 * n : n / 4);
                if (here < cost) {
                    cost = here;
                    best[y] = size[j];
                }
            }
        }
    }
    __syncthreads();
    const int by_wave = best[0], by_block = best[1];
    // ---- items of contents
    for (int g = tid; g < G; g += LANES) {
        int blocks, tiles;
        const int sort = group_set(g, blocks, tiles), n = sort < 0 ? 0 : seats_up(tiles, sort ? by_block : by_wave);
        cut[g] = n;
        sums[0][g] = sort == 0 ? n * blocks : 0;
        sums[1][g] = sort == 2 ? n * blocks : 0;
    }
    {
        int* const a[2] = {sums[0], sums[1]};
        running(a, G, room);
    }
    const int waves = sums[0][G], blocks_in_all = sums[1][G];
    for (int i = tid; i < waves + blocks_in_all; i += LANES) {
        const int y = i >= waves, x = y ? i - waves : i, size = y ? deep : 32;
        const int g = find(sums[y], G, x), r = heads[g], j = x - sums[y][g];
        int blocks, tiles;
        group_set(g, blocks, tiles);
        const int P = stored[r], tok0 = first[r], T = first[heads[g + 1]] - tok0, kt = seats_up(P, PAGED_TILE) - tiles;
        const int s = j / blocks, b = j - s * blocks, n = cut[g];
        const int from = (int)((long)tiles * s / n), to = (int)((long)tiles * (s + 1) / n);
        const SeatItem it = {tok0, T, size * b, s, 0, {}, {{listed[r], P, kt + from, to - from, most(0, P + high[g] - far + 1), P - 1, 0, 0}, {}}};
        if (x < (y ? kd.room[2] : kd.room[0])) store(y ? kd.block : kd.wave, x, it);
    }
    __syncthreads();
    // ---- of the seats' own keys; partial results
    const auto pieces_of = [&](int r, int sort, int tiles) __attribute__((always_inline)) { return sort == 0 ? seats_up(tiles, by_wave) : sort == 2 ? seats_up(tiles, by_block) : 1; };
    const auto parts_of = [&](int r, int sort, int pieces) __attribute__((always_inline)) {   // of each of its tokens
        const int theirs = cut[of_group[r]];                                                  // (of a seat that reads its content itself: none)
        return sort == 3 ? theirs : theirs + pieces > 1 ? theirs + pieces : 0;
    };
    each_seat([&](int r) __attribute__((always_inline)) {
        int blocks, tiles, shared;
        const int sort = seat_set(r, blocks, tiles, shared), n = sort < 0 ? 0 : pieces_of(r, sort, tiles + shared);
#pragma unroll
        for (int x = 0; x < 4; x++) sums[x][r] = sort == x ? n * blocks : 0;
        sums[4][r] = sort < 0 ? 0 : seats_least(LOTS / 2, took[r] * parts_of(r, sort, n));
    });
    {
        int* const a[5] = {sums[0], sums[1], sums[2], sums[3], sums[4]};
        running(a, R, room);
    }
    each_seat([&](int r) __attribute__((always_inline)) {
        int blocks, tiles, shared;
        const int sort = seat_set(r, blocks, tiles, shared), parts = sort < 0 ? 0 : parts_of(r, sort, pieces_of(r, sort, tiles + shared));
        kd.seat_parts[2 * r] = sums[4][r] | (sort == 3 || parts == 0 ? INT_MIN : 0);   // (the sign: no piece is left to be joined)
        kd.seat_parts[2 * r + 1] = parts;
        if (sort == 3 && sums[3][r] < kd.room[3]) {
            const int L = stay[r] + 1, lo = most(0, stay[r] - far + 1), at = p.table_at + r * p.width, a = lo / p.page, b = (L - 1) / p.page;
            int4* to = (int4*)(kd.last + sizeof(SeatLast) / 4 * (long)sums[3][r]);
            int ids[SEAT_PAGES];
#pragma unroll
            for (int x = 0; x < SEAT_PAGES; x++) ids[x] = p.table[at + seats_least(a + x, b)];
            to[0] = make_int4(first[r], L, lo, at);
            to[1] = make_int4(sums[4][r], parts, ids[0], ids[1]);
            to[2] = make_int4(ids[2], ids[3], ids[4], ids[5]);
        }
    });
    if (tid == 0) {
        kd.seat_parts[2 * R] = sums[4][R];
        kd.counts[0] = waves + sums[0][R];
        kd.counts[1] = sums[1][R];
        kd.counts[2] = blocks_in_all + sums[2][R];
        kd.counts[3] = sums[3][R];
        kd.counts[4] = sums[4][R];
    }
    const int n0 = sums[0][R], n1 = sums[1][R], items = n0 + n1 + sums[2][R];
    for (int i = tid; i < items; i += LANES) {
        const int y = i < n0 ? 0 : i < n0 + n1 ? 1 : 2, j = y == 0 ? i : y == 1 ? i - n0 : i - n0 - n1;
        const int r = find(sums[y], R, j), x = j - sums[y][r], n = took[r], L = stay[r] + n;
        int blocks, tiles, shared;
        seat_set(r, blocks, tiles, shared);
        const int pieces = pieces_of(r, y, tiles + shared);
        const int s = x / blocks, b = x - s * blocks, size = y == 2 ? deep : 32;
        const int t0 = b * size / group, t1 = seats_least(n - 1, (b * size + size - 1) / group);   // its first and its last token
        // tiles of the content, then of its own keys, that this block's rows see; the piece's share of them
        const int P = shared ? stored[r] : 0;
        const int lo = most(0, stay[r] + t0 - far + 1), kt = lo / PAGED_TILE, own = seats_up(stay[r] + t1 + 1, PAGED_TILE) - kt;
        const int lo2 = most(0, P + stay[r] + t0 - far + 1), kt2 = lo2 / PAGED_TILE, theirs = lo2 < P ? seats_up(P, PAGED_TILE) - kt2 : 0;
        const int from = (int)((long)(own + theirs) * s / pieces), to = (int)((long)(own + theirs) * (s + 1) / pieces);
        const SeatSpan mine = {p.table_at + r * p.width, L, kt + most(0, from - theirs), most(0, to - most(from, theirs)), most(0, stay[r] + t1 - far + 1), stay[r] + t0, 1, 0};
        const int ahead = cut[of_group[r]];
        SeatItem it = {first[r], n, b * size, ahead + s, ahead + pieces == 1, {}, {mine, {}}};
        if (theirs > 0 && from < theirs) {
            it.span[0] = {listed[r], P, kt2 + from, seats_least(to, theirs) - from, most(0, P + stay[r] + t1 - far + 1), P - 1, 0, 0};
            it.span[1] = mine;
        }
        const int at = y == 0 ? waves + j : y == 1 ? j : blocks_in_all + j;
        if (at < (y == 0 ? kd.room[0] : y == 1 ? kd.room[1] : kd.room[2])) store(y == 0 ? kd.wave : y == 1 ? kd.single : kd.block, at, it);
    }
    if (p.rows > SEATS_ROWS_AT_ONCE) return;
    __syncthreads();
    constexpr int BY_SEAT = MOST > LANES ? FIRST_ROWS : 0;
    bool more = !BY_SEAT;
    if (BY_SEAT) {
        each_seat([&](int r) __attribute__((always_inline)) {
            for (int j = 0; j < seats_least(took[r], BY_SEAT); j++) place_parts(p, kd, first[r] + j, total, r, first[r]);
            more |= took[r] > BY_SEAT;
        });
        more = __syncthreads_or(more);
    }
    for (int row = more ? tid : total + tid; row <= p.rows; row += LANES) {
        const int seat = row < total ? find(first, R, row) : 0;
        if (row >= total || row - first[seat] >= BY_SEAT) place_parts(p, kd, row, total, seat, first[seat]);
    }
}

// How long the lists of a head geometry may get: [0 .. 3] items (waves that divide tiles, a wave to 32 rows, shared tiles, the last word), [4] partial rows (per query head).  A set of `blocks`
// blocks on `tiles` tiles is blocks x ceil(tiles / size) items, size at least the work of all sets over the places: in all no more than the places and a block each.
void rooms(const spinf_seats_args* a, const spinf_seats_kind& k, int64_t out[5]) {
    const int64_t group = k.hq / k.hkv, rows = a->rows, A = std::min<int64_t>(a->seats, rows);   // at most A seats have new tokens, below at most A contents
    const int64_t by_wave = seats_wave_places(k.d) / k.hkv + 1, by_block = seats_block_places(k.d) / k.hkv + 1;
    const bool block = rows * group > 32;
    out[0] = by_wave + 3 * A;                                   // (a content's rows: two blocks at most)
    out[1] = (SEAT_SHARED_ROWS + 31) / 32 * A;
    out[2] = block ? by_block + 2 * (rows * group / 128 + A) : 0;
    out[3] = seats_last((int)group, k.d) && seats_last_pays(A, 0, k.hkv) ? A : 0;
    // Partial rows: tokens x pieces.  A set's pieces are at most tiles / size + 1, its tokens at most a block's rows over `group` for each block, and blocks x tiles / size of all sets no more than
    // the places: a term for the places, and one piece for each token of a set.  Tokens of seats that share their content's reading (up to SEAT_SHARED_ROWS rows each) are in two sets.  A
    // seat of more rows is one set, and leaves pieces only where it has two and more: those are less than twice tiles / size, so its tokens have no term of their own (48 prompts of 100,805 rows in all, 16 heads on 8
    // of 256: 13,619 partial rows; two to each row would be 3.4 GB of workspace).
    const int64_t shared = std::min<int64_t>(rows, A * (SEAT_SHARED_ROWS / group));
    out[4] = 2 * shared + (32 / group + 1) * by_wave + (block ? 2 * (128 / group + 1) * by_block : 0);
}

int check(const spinf_seats_args* a, const char* what) {
    if (!a) return spinf_fail(SPINF_E_ARG, "%s: null args", what);
    if (a->seats < 1 || a->seats > SEATS_MOST) return spinf_fail(SPINF_E_ARG, "%s: %d seats (1 .. %d)", what, a->seats, SEATS_MOST);
    if (a->rows < 1 || a->rows > (1 << 22)) return spinf_fail(SPINF_E_ARG, "%s: %lld rows (1 .. 2^22)", what, (long long)a->rows);
    if (a->page < 16 || a->page % 16 || a->page > (1 << 20)) return spinf_fail(SPINF_E_ARG, "%s: pages of %d keys (a multiple of 16)", what, a->page);
    if (a->keys < 1 || a->keys > (1 << 28)) return spinf_fail(SPINF_E_ARG, "%s: %lld keys of a seat (1 .. 2^28)", what, (long long)a->keys);
    if (a->pool < 0 || a->pool > (1 << 28) || a->contents < 0 || a->contents > (1 << 20)) return spinf_fail(SPINF_E_ARG, "%s: %lld pages, %d contents", what, (long long)a->pool, a->contents);
    if (a->pool * a->page > ((int64_t)1 << 36)) return spinf_fail(SPINF_E_ARG, "%s: a pool of %lld keys", what, (long long)(a->pool * a->page));
    if (a->kinds < 0 || a->kinds > SEATS_KINDS) return spinf_fail(SPINF_E_ARG, "%s: %d head geometries (at most %d)", what, a->kinds, SEATS_KINDS);
    if (a->longest < 0 || a->longest > (1 << 28)) return spinf_fail(SPINF_E_ARG, "%s: a content of %lld keys (0 .. 2^28)", what, (long long)a->longest);
    const int64_t width = (a->keys + a->page - 1) / a->page;
    if (a->table_at < 0 || a->table_at % 4 || a->table_at + a->seats * width > INT32_MAX) return spinf_fail(SPINF_E_ARG, "%s: page lists of more than 2^31 entries", what);
    for (int i = 0; i < a->kinds; i++) {
        const spinf_seats_kind& k = a->kind[i];
        if (k.hq <= 0 || k.hkv <= 0 || k.hq % k.hkv || k.hq > 4096) return spinf_fail(SPINF_E_ARG, "%s: %d query heads do not group over %d key / value heads", what, k.hq, k.hkv);
        if (k.d != 64 && k.d != 128 && k.d != 256 && k.d != 512) return spinf_fail(SPINF_E_ARG, "%s: head dim %d not supported (64, 128, 256, 512)", what, k.d);
        if (k.window < 0) return spinf_fail(SPINF_E_ARG, "%s: window %d", what, k.window);
        if (a->rows * k.hq > (1 << 28)) return spinf_fail(SPINF_E_ARG, "%s: %lld rows of %d heads are too many", what, (long long)a->rows, k.hq);
    }
    return SPINF_OK;
}

}  // namespace

extern "C" int spinf_seats_rooms(const spinf_seats_args* a, int32_t kind, int64_t out[5]) {
    const int rc = check(a, "seats_rooms");
    if (rc) return rc;
    if (kind < 0 || kind >= a->kinds || !out) return spinf_fail(SPINF_E_ARG, "seats_rooms: head geometry %d of %d", kind, a->kinds);
    rooms(a, a->kind[kind], out);
    return SPINF_OK;
}

extern "C" int spinf_seats_step(const spinf_seats_args* a, void* stream) {
    const int rc = check(a, "seats_step");
    if (rc) return rc;
    if (!a->come || !a->content || !a->lens || !a->lists || !a->left || !a->first || !a->took || !a->stay || !a->slots || !a->pos || (a->pool && !a->free) || (a->contents && !a->shared))
        return spinf_fail(SPINF_E_ARG, "seats_step: null pointer");
    Params p = {};
    p.come = a->come; p.drop = a->drop; p.content = a->content;
    p.lens = a->lens; p.table = a->lists; p.free = a->free; p.left = a->left; p.first = a->first; p.took = a->took; p.stay = a->stay;
    p.slots = (long*)a->slots; p.pos = a->pos;
    p.shared = a->shared;
    p.seats = a->seats; p.rows = (int)a->rows; p.page = a->page; p.keys = (int)a->keys; p.width = (int)((a->keys + a->page - 1) / a->page); p.pool = (int)a->pool;
    p.contents = a->contents; p.table_at = (int)a->table_at; p.kinds = a->kinds;
    for (int i = 0; i < a->kinds; i++) {
        const spinf_seats_kind& k = a->kind[i];
        int64_t n[5];
        rooms(a, k, n);
        if (!k.wave || !k.single || !k.block || !k.last || !k.counts || !k.parts || !k.seat_parts) return spinf_fail(SPINF_E_ARG, "seats_step: null lists of head geometry %d", i);
        if ((uintptr_t)k.wave % 16 || (uintptr_t)k.single % 16 || (uintptr_t)k.block % 16 || (uintptr_t)k.last % 16) return spinf_fail(SPINF_E_ARG, "seats_step: lists must be 16-byte aligned");
        p.kind[i] = {k.wave, k.single, k.block, k.last, k.counts, k.parts, k.seat_parts, k.hq, k.hkv, k.d, k.window < LOTS ? k.window : LOTS, {(int)n[0], (int)n[1], (int)n[2], (int)n[3]}};
    }
    hipStream_t s = (hipStream_t)stream;
    if (a->seats <= LANES) hipLaunchKernelGGL(seats_step_kernel<1>, dim3(1), dim3(LANES), 0, s, p);
    else hipLaunchKernelGGL(seats_step_kernel<SEATS_MOST / LANES>, dim3(1), dim3(LANES), 0, s, p);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a->kinds) {
        if (a->seats <= LANES) hipLaunchKernelGGL(seats_lists_kernel<LANES>, dim3(a->kinds), dim3(LANES), 0, s, p);
        else hipLaunchKernelGGL(seats_lists_kernel<SEATS_MOST>, dim3(a->kinds), dim3(LANES), 0, s, p);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a->rows > SEATS_ROWS_AT_ONCE) {
        hipLaunchKernelGGL(seats_rows_kernel, dim3((unsigned)(a->rows / 256 + 1)), dim3(256), 0, s, p);
        e = hipGetLastError();
    }
    return e == hipSuccess ? SPINF_OK : spinf_fail(SPINF_E_HIP, "seats_step: launch: %s", hipGetErrorString(e));
}
