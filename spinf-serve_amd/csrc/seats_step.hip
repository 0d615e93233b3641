// The books of seats on the GPU, for gfx950 (MI355X): which keys go, which pages come back and are handed out, where new tokens' keys and values lie, and the work lists of the
// attention over them (seats_attn.hip), all from lengths in device memory: a recorded step can be replayed for the next one.  No counterpart in the reference, whose
// contents are read anew with every request.
//
// Mathematics: whole numbers only.  Of seat r with n_r keys the last min(drop_r, n_r) go, then new_r come.  Pages given back are pushed on a stack, pages needed are popped
// from it; with running sums over the seats (of pages back, of pages and tokens asked for) every push, pop and row has a place of its own, so the result is that of going seat by
// seat, whatever order the lanes run in.  Pushed in the reverse of the order they are popped in: a step that takes back what the last one added leaves stack and tables as they were.
//
// Bound by latency: one workgroup of 16 waves, some ten running sums over at most 2,048 seats in LDS; pages, items and rows are dealt out to lanes by a search in the sums.  More than
// SEATS_ROWS_AT_ONCE rows (prompts) get a second launch over the whole GPU.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "spinf_tree.h"
#include "common.h"
#include "seats.h"

namespace {

constexpr int LANES = 1024, WAVES = LANES / 64;
constexpr int LOTS = 1 << 30;   // sums stop there

struct Kind { int* wave; int* single; int* block; int* counts; int* parts; int* seat_parts; int hq, hkv, d, window, wave_room, single_room, block_room; };
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
template <int N, class F>
__device__ __forceinline__ void scan(int (&x)[N], int (&total)[N], int (*room)[WAVES], int none, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int y[N];
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = x[i];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int z = __shfl_up(y[i], d);
            if (lane >= d) y[i] = f(z, y[i]);
        }
    __syncthreads();   // (the room is free)
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; i++) room[i][wave] = y[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        int before = none, all = none;
        for (int w = 0; w < WAVES; w++) {
            if (w == wave) before = all;
            all = f(all, room[i][w]);
        }
        const int z = __shfl_up(y[i], 1);
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
    int4* p = (int4*)(items + 12 * (long)at);
    p[0] = make_int4(it.tok0, it.T, it.L, it.tab);
    p[1] = make_int4(it.row0, it.kt0, it.tiles, it.piece);
    p[2] = make_int4(it.flo, it.fhi, it.flags, 0);
}

// Places and positions of rows, and where their partial results begin
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
    for (int k = 0; k < p.kinds; k++) {
        const int* sp = p.kind[k].seat_parts;
        p.kind[k].parts[row] = row < total ? sp[2 * seat] + (row - first) * sp[2 * seat + 1] : sp[2 * p.seats];
        if (row == p.rows - 1) p.kind[k].parts[p.rows] = sp[2 * p.seats];
    }
}

__global__ __launch_bounds__(256) void seats_rows_kernel(const Params p) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= p.rows) return;
    const int total = p.first[p.seats];
    const int seat = row < total ? find(p.first, p.seats, row) : 0;
    place_row(p, row, total, seat, p.first[seat], p.stay[seat], p.content[seat]);
}

template <int SPT>   // seats per lane
__global__ __launch_bounds__(LANES) void seats_step_kernel(const Params p) {
    constexpr int MOST = SPT * LANES;
    __shared__ int room[4][WAVES];
    __shared__ int stay[MOST], took[MOST], content[MOST], first[MOST + 1];
    __shared__ int sums[3][MOST + 1];
    __shared__ int heads[MOST + 1], low[MOST], high[MOST], of_group[MOST], cut[MOST];   // by group of seats in a row below one content; cut: pieces of the content's keys
    const int R = p.seats, tid = threadIdx.x;
    const auto plus = [](int a, int b) __attribute__((always_inline)) { return add(a, b); };
    const auto larger = [](int a, int b) __attribute__((always_inline)) { return most(a, b); };
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

    // ---- groups: seats with new tokens, one after the other below the same content (seats without any in between do not part them)
    int last[1] = {-1}, none[1];
#pragma unroll
    for (int i = 0; i < SPT; i++) {
        const int r = tid * SPT + i;
        if (r < R && want[i]) last[0] = r;
    }
    scan(last, none, room, -1, larger);
    int head[1] = {0}, groups[1];
    bool begins[SPT];
#pragma unroll
    for (int i = 0; i < SPT; i++) {
        const int r = tid * SPT + i;
        begins[i] = r < R && want[i] && (last[0] < 0 || content[last[0]] != content[r]);
        head[0] += begins[i];
        if (r < R && want[i]) last[0] = r;
    }
    scan(head, groups, room, 0, plus);
    const int G = groups[0];
#pragma unroll
    for (int i = 0; i < SPT; i++) {
        const int r = tid * SPT + i;
        if (r < R) {
            if (begins[i]) {
                heads[head[0]] = r;
                low[head[0]] = INT_MAX;
                high[head[0]] = 0;
            }
            head[0] += begins[i];
            of_group[r] = head[0] - 1;   // (means something only where the seat has new tokens)
        }
    }
    if (tid == 0) heads[G] = R;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SPT; i++) {   // the least and the largest place among the seats' own keys of a group's new tokens
        const int r = tid * SPT + i;
        if (want[i]) {
            atomicMin(&low[of_group[r]], here[i]);
            atomicMax(&high[of_group[r]], here[i] + want[i] - 1);
        }
    }

    // ---- the lists of every head geometry
    for (int k = 0; k < p.kinds; k++) {
        const Kind& kd = p.kind[k];
        const int group = kd.hq / kd.hkv, W = kd.window;
        const int far = W ? W : LOTS;
        __syncthreads();
        // contents: sums[0] over groups
        int n0[1] = {0}, all0[1];
#pragma unroll
        for (int i = 0; i < SPT; i++) {
            const int g = tid * SPT + i;
            if (g < G) {
                const int r = heads[g], c = content[r];
                int pieces = 0, count = 0;
                if (c >= 0) {
                    const int P = p.shared[3 * c], T = first[heads[g + 1]] - first[r], blocks = seats_up(T * group, 128);
                    const int lo = most(0, P + low[g] - far + 1), tiles = lo < P ? seats_up(P, PAGED_TILE) - lo / PAGED_TILE : 0;
                    if (tiles > 0) {
                        pieces = seats_block_pieces(tiles, kd.d, kd.hkv, blocks, true);
                        count = pieces * blocks;
                    }
                }
                cut[g] = pieces;
                n0[0] += count;
                sums[0][g] = count;
            }
        }
        scan(n0, all0, room, 0, plus);
#pragma unroll
        for (int i = 0; i < SPT; i++) {
            const int g = tid * SPT + i;
            if (g < G) {
                const int count = sums[0][g];
                sums[0][g] = n0[0];
                n0[0] += count;
            }
        }
        if (tid == 0) sums[0][G] = all0[0];
        __syncthreads();
        for (int i = tid; i < all0[0]; i += LANES) {
            const int g = find(sums[0], G, i), r = heads[g], c = content[r], j = i - sums[0][g];
            const int P = p.shared[3 * c], tok0 = first[r], T = first[heads[g + 1]] - tok0, blocks = seats_up(T * group, 128);
            const int lo = most(0, P + low[g] - far + 1), kt = lo / PAGED_TILE, tiles = seats_up(P, PAGED_TILE) - kt;
            const int s = j / blocks, b = j - s * blocks, n = cut[g];
            const int from = (int)((long)tiles * s / n), to = (int)((long)tiles * (s + 1) / n);
            if (i < kd.block_room)
                store(kd.block, i, {tok0, T, P, p.shared[3 * c + 2], 128 * b, kt + from, to - from, s, most(0, P + high[g] - far + 1), P - 1, 0, 0});
        }
        // seats: how many items of each sort, and partial results
        __syncthreads();
        int n1[4] = {0, 0, 0, 0}, all1[4];
        int c1[SPT][3], parts[SPT];
        const auto plan = [&](int r, int n, int& blocks, int& tiles, int& sort, int& pieces) __attribute__((always_inline)) {
            const int rows = n * group, L = stay[r] + n, lo = most(0, stay[r] - far + 1);
            tiles = seats_up(L, PAGED_TILE) - lo / PAGED_TILE;
            const bool few = rows <= SEAT_WAVE_ROWS;
            blocks = seats_up(rows, few ? 32 : 128);
            sort = !few ? 2 : tiles <= SEAT_SINGLE_TILES ? 1 : 0;
            pieces = sort == 0 ? seats_wave_pieces(tiles, kd.d, kd.hkv, blocks) : sort == 1 ? 1 : seats_block_pieces(tiles, kd.d, kd.hkv, blocks, false);
        };
#pragma unroll
        for (int i = 0; i < SPT; i++) {
            const int r = tid * SPT + i;
            c1[i][0] = c1[i][1] = c1[i][2] = parts[i] = 0;
            if (want[i]) {
                int blocks, tiles, sort, pieces;
                plan(r, want[i], blocks, tiles, sort, pieces);
                c1[i][sort] = blocks * pieces;
                parts[i] = cut[of_group[r]] + pieces;
            }
#pragma unroll
            for (int x = 0; x < 3; x++) n1[x] += c1[i][x];
            n1[3] = add(n1[3], parts[i] > 1 ? want[i] * parts[i] : 0);
        }
        scan(n1, all1, room, 0, plus);
#pragma unroll
        for (int i = 0; i < SPT; i++) {
            const int r = tid * SPT + i;
            if (r < R) {
#pragma unroll
                for (int x = 0; x < 3; x++) {
                    sums[x][r] = n1[x];
                    n1[x] += c1[i][x];
                }
                kd.seat_parts[2 * r] = n1[3];
                kd.seat_parts[2 * r + 1] = parts[i] > 1 ? parts[i] : 0;
                n1[3] = add(n1[3], parts[i] > 1 ? want[i] * parts[i] : 0);
            }
        }
        if (tid < 3) sums[tid][R] = tid == 0 ? all1[0] : tid == 1 ? all1[1] : all1[2];
        if (tid == 0) {
            kd.seat_parts[2 * R] = all1[3];
            kd.counts[0] = all1[0];
            kd.counts[1] = all1[1];
            kd.counts[2] = add(all0[0], all1[2]);
            kd.counts[3] = all1[3];
        }
        __syncthreads();
        const int counts = all1[0] + all1[1] + all1[2];
        for (int i = tid; i < counts; i += LANES) {
            const int sort = i < all1[0] ? 0 : i < all1[0] + all1[1] ? 1 : 2, j = sort == 0 ? i : sort == 1 ? i - all1[0] : i - all1[0] - all1[1];
            const int r = find(sums[sort], R, j), x = j - sums[sort][r], n = took[r], L = stay[r] + n;
            int blocks, tiles, is, pieces;
            plan(r, n, blocks, tiles, is, pieces);
            const int s = x / blocks, b = x - s * blocks, size = sort == 2 ? 128 : 32;
            const int t0 = b * size / group, t1 = seats_least(n - 1, (b * size + size - 1) / group);   // its first and its last token
            const int lo = most(0, stay[r] + t0 - far + 1), kt = lo / PAGED_TILE, mine = seats_up(stay[r] + t1 + 1, PAGED_TILE) - kt;
            const int from = (int)((long)mine * s / pieces), to = (int)((long)mine * (s + 1) / pieces);
            const int ahead = cut[of_group[r]];
            const SeatItem it = {first[r], n, L, p.table_at + r * p.width, b * size, kt + from, to - from, ahead + s, most(0, stay[r] + t1 - far + 1), stay[r] + t0,
                                 SEAT_OWN | (ahead + pieces == 1 ? SEAT_ONLY : 0), 0};
            if (sort == 0) { if (j < kd.wave_room) store(kd.wave, j, it); }
            else if (sort == 1) { if (j < kd.single_room) store(kd.single, j, it); }
            else if (all0[0] + j < kd.block_room) store(kd.block, all0[0] + j, it);
        }
    }
    __syncthreads();
    if (p.rows > SEATS_ROWS_AT_ONCE) return;
    for (int row = tid; row < p.rows; row += LANES) {
        const int seat = row < total ? find(first, R, row) : 0;
        place_row(p, row, total, seat, first[seat], stay[seat], content[seat]);
    }
}

// How long the lists of a head geometry may get: [0 .. 2] items, [3] partial rows (per query head)
void rooms(const spinf_seats_args* a, const spinf_seats_kind& k, int64_t out[4]) {
    const int64_t R = a->seats, rows = a->rows, group = k.hq / k.hkv, A = std::min(R, rows);   // at most A seats have new tokens
    const int64_t tiles = (a->keys + PAGED_TILE - 1) / PAGED_TILE, in_all = a->pool * a->page / PAGED_TILE + R;
    const int64_t waves = seats_wave_pieces((int)tiles, k.d, k.hkv, 1), pieces = std::min(A * waves, in_all / SEAT_WAVE_TILES + A);
    out[0] = 2 * pieces;   // (at most 64 rows: two blocks)
    out[1] = 2 * A;
    // blocks x pieces of a set is its blocks, or at most places / hkv; tokens x pieces its tokens, or at most those of 128 rows per place
    const int64_t places = (k.d == 512 ? PAGED_PLACES / 2 : PAGED_PLACES) / k.hkv + 1;
    const int64_t big = std::min(A, rows * group / (SEAT_WAVE_ROWS + 1));
    const auto items = [&](int64_t sets, int64_t most) { return std::min((rows * group / 128 + sets) * most, rows * group / 128 + sets + sets * places); };
    const auto parts = [&](int64_t sets, int64_t most) { return std::min(rows * most, rows + sets * (128 / group + 1) * places); };
    const int64_t own = seats_block_pieces((int)tiles, k.d, k.hkv, 1, false);
    out[2] = big ? items(big, own) : 0;
    out[3] = rows + std::min(rows * waves, std::max<int64_t>(1, SEAT_WAVE_ROWS / group) * pieces) + (big ? parts(big, own) : 0);
    if (a->longest) {
        const int64_t shared = seats_block_pieces((int)((a->longest + PAGED_TILE - 1) / PAGED_TILE), k.d, k.hkv, 1, true);
        out[2] += items(A, shared);
        out[3] += parts(A, shared);
    }
    for (int i = 0; i < 3; i++) out[i] = std::max<int64_t>(out[i], 1);
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
        int64_t n[4];
        rooms(a, k, n);
        if (a->rows * k.hq > (1 << 30) || n[0] > (1 << 26) || n[2] > (1 << 26) || n[3] > (1 << 30)) return spinf_fail(SPINF_E_ARG, "%s: %lld rows of %d heads are too many", what, (long long)a->rows, k.hq);
    }
    return SPINF_OK;
}

}  // namespace

extern "C" int spinf_seats_rooms(const spinf_seats_args* a, int32_t kind, int64_t out[4]) {
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
        int64_t n[4];
        rooms(a, k, n);
        if (!k.wave || !k.single || !k.block || !k.counts || !k.parts || !k.seat_parts) return spinf_fail(SPINF_E_ARG, "seats_step: null lists of head geometry %d", i);
        if ((uintptr_t)k.wave % 16 || (uintptr_t)k.single % 16 || (uintptr_t)k.block % 16) return spinf_fail(SPINF_E_ARG, "seats_step: lists must be 16-byte aligned");
        p.kind[i] = {k.wave, k.single, k.block, k.counts, k.parts, k.seat_parts, k.hq, k.hkv, k.d, k.window < LOTS ? k.window : LOTS, (int)n[0], (int)n[1], (int)n[2]};
    }
    hipStream_t s = (hipStream_t)stream;
    if (a->seats <= LANES) hipLaunchKernelGGL(seats_step_kernel<1>, dim3(1), dim3(LANES), 0, s, p);
    else hipLaunchKernelGGL(seats_step_kernel<SEATS_MOST / LANES>, dim3(1), dim3(LANES), 0, s, p);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a->rows > SEATS_ROWS_AT_ONCE) {
        hipLaunchKernelGGL(seats_rows_kernel, dim3((unsigned)((a->rows + 255) / 256)), dim3(256), 0, s, p);
        e = hipGetLastError();
    }
    return e == hipSuccess ? SPINF_OK : spinf_fail(SPINF_E_HIP, "seats_step: launch: %s", hipGetErrorString(e));
}
