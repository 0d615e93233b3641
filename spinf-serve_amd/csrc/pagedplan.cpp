// Host compiler of the paged cache's work lists (include/spinf_tree.h, "paged cache"): which 32-key tiles a group of query rows visits, how they
// are cut into work items, and in which order the items are launched.  Deterministic, no global state.
//
// The rows of a (request, key / value head) are its new tokens x the query heads of the group, row = token * group + head, in row groups of 32.
// A row group's tiles come as runs {first tile, tiles, bits}: one long run of tiles that every row sees whole, and around it single
// tiles that the kernel masks element by element or whose rows see none of them.
//
// How a request is cut depends on its own lengths, its own tree and the head geometry alone, never on what shares the call: its outputs are the same
// bits whatever it is batched with.
#include <algorithm>
#include <cstdint>
#include <exception>
#include <new>
#include <vector>

#include "spinf_tree.h"
#include "common.h"
#include "paged.h"

namespace {

constexpr int TK = PAGED_TILE, GROUP = PAGED_ROWS, BLOCK_GROUPS = PAGED_BLOCK_GROUPS;
constexpr int XCDS = 8;
using Run = PagedRun;
using Item = PagedItem;
using Join = PagedJoin;

// what the keys of a request's new tokens (a tile of them) need of their rows: the largest and the smallest subtree end
struct TileEnds { int32_t lo, hi; };

}  // namespace

struct spinf_pagedplan {
    std::vector<Item> wave, block;    // items of the kernel whose waves share rows / share tiles
    std::vector<Run> runs;
    std::vector<Join> joins;
    int64_t part_rows = 0;
};

namespace {

struct Request {
    int32_t T, L, c, cu, tab;
    const int32_t* end;   // of this request's rows, in rows of the call (NULL: a chain)
    const int32_t* pos;
    std::vector<TileEnds> ends;   // of the tiles from c / 32 on
};

// bits of tile kt for the tokens a .. b of a request: bit 0 some row sees some key, bit 4 some pair is masked
unsigned tile_bits(const Request& r, int window, int kt, int a, int b, int pos_lo, int pos_hi) {
    const int64_t s0 = (int64_t)kt * TK, s1 = s0 + TK - 1;
    if (s0 >= r.L || s0 > (int64_t)r.c + b) return 0;
    bool all = s1 < r.L && s1 <= (int64_t)r.c + a;
    if (window > 0) {
        // the key at the stored place s lies at position s; a new token of a tree anywhere up to it, which the kernel settles key by key
        const int64_t k_hi = r.end && s1 >= r.c ? INT64_MAX / 2 : s1, k_lo = r.end && s1 >= r.c ? 0 : s0;
        if (pos_lo - k_hi >= window) return 0;
        all = all && pos_hi - k_lo < window;
    }
    if (r.end && s1 >= r.c) {   // new tokens: a row sees the keys whose subtree it lies in
        const TileEnds& e = r.ends[kt - std::max(r.c, 0) / TK];
        const int first = r.cu + a;
        if (s0 >= r.c && e.hi <= first) return 0;
        all = all && e.lo > r.cu + b;
        if (!all && s0 >= r.c) {
            bool any = false;
            const int u1 = (int)std::min<int64_t>(std::min<int64_t>(s1 - r.c, r.T - 1), b);
            for (int u = (int)(s0 - r.c); u <= u1 && !any; u++) any = std::max(u, a) < r.end[u] - r.cu;
            if (!any) return 0;
        }
    }
    return all ? 1u : 0x11u;
}

class Builder {
  public:
    Builder(const spinf_paged_plan_args* a, spinf_pagedplan* p) : a_(a), p_(p), group_(a->hq / a->hkv), window_(a->window) {}

    void run() {
        int64_t cu = 0, tab = 0;
        for (int64_t i = 0; i < a_->reqs; i++) {
            Request r;
            r.T = a_->q_lens[i];
            r.L = a_->kv_lens[i];
            r.c = r.L - r.T;
            r.cu = (int32_t)cu;
            r.tab = (int32_t)tab;
            r.end = a_->end ? a_->end + cu : nullptr;
            r.pos = a_->pos ? a_->pos + cu : nullptr;
            if (r.end)
                for (int kt = std::max(r.c, 0) / TK; (int64_t)kt * TK < r.L; kt++) {
                    TileEnds e{INT32_MAX, 0};
                    for (int64_t s = std::max<int64_t>((int64_t)kt * TK, r.c); s < std::min<int64_t>((int64_t)kt * TK + TK, r.L); s++) {
                        e.lo = std::min(e.lo, r.end[s - r.c]);
                        e.hi = std::max(e.hi, r.end[s - r.c]);
                    }
                    r.ends.push_back(e);
                }
            if (r.T > 0) request(r, (int)i);
            cu += r.T;
            tab += (r.L + a_->page - 1) / a_->page;
        }
        order(p_->wave);
        order(p_->block);
    }

  private:
    // the runs of one row group set: rows row0 .. row0 + 32 groups - 1
    void list(const Request& r, int row0, int groups, std::vector<Run>& out) {
        out.clear();
        const int N = r.T * group_;
        struct G { int a, b, lo, hi; } g[BLOCK_GROUPS];
        int n = 0;
        int64_t full1 = INT64_MAX, full0 = 0, kt0 = INT64_MAX, kt1 = 0;
        for (; n < groups && row0 + GROUP * n < N; n++) {
            G& x = g[n];
            x.a = (row0 + GROUP * n) / group_;
            x.b = (std::min(row0 + GROUP * n + GROUP, N) - 1) / group_;
            x.lo = r.c + x.a;
            x.hi = r.c + x.b;
            if (r.pos) {
                x.lo = *std::min_element(r.pos + x.a, r.pos + x.b + 1);
                x.hi = *std::max_element(r.pos + x.a, r.pos + x.b + 1);
            }
            // tiles that every row of the group sees whole: below the rows themselves (in a tree: of stored tokens), inside the window
            full1 = std::min<int64_t>(full1, r.end ? std::max(r.c, 0) / TK : std::max<int64_t>((int64_t)r.c + x.a + 1, 0) / TK);
            if (window_ > 0) full0 = std::max<int64_t>(full0, std::max<int64_t>((int64_t)x.hi - window_ + 1 + TK - 1, 0) / TK);
            kt0 = std::min<int64_t>(kt0, window_ > 0 ? std::max<int64_t>((int64_t)x.lo - window_ + 1, 0) / TK : 0);
            kt1 = std::max<int64_t>(kt1, std::min<int64_t>(r.L, std::max<int64_t>((int64_t)r.c + x.b + 1, 0)) + TK - 1);
        }
        kt1 /= TK;
        auto add = [&](int64_t kt, int64_t count, uint32_t bits) {
            if (!out.empty() && out.back().bits == bits && out.back().kt + out.back().count == kt) out.back().count += (int32_t)count;
            else out.push_back({(int32_t)kt, (int32_t)count, bits, 0});
        };
        const uint32_t all = (1u << n) - 1;
        for (int64_t kt = kt0; kt < kt1;) {
            if (kt >= full0 && kt < full1) {
                add(kt, full1 - kt, all);
                kt = full1;
                continue;
            }
            uint32_t bits = 0;
            for (int i = 0; i < n; i++) bits |= tile_bits(r, window_, (int)kt, g[i].a, g[i].b, g[i].lo, g[i].hi) << i;
            // (a group that sees nothing of a tile that another one sees computes it too: all of its pairs are masked)
            if (bits & all) add(kt, 1, bits | (all & ~bits) << 4);
            kt++;
        }
    }

    void request(const Request& r, int index) {
        const int64_t N = (int64_t)r.T * group_;
        // The kernel whose waves share their rows and divide the keys takes what the other one would leave the GPU mostly idle with.
        const int64_t blocks = (N + GROUP * BLOCK_GROUPS - 1) / (GROUP * BLOCK_GROUPS) * a_->hkv;
        bool by_wave = a_->variant ? a_->variant == 1 : N <= 2 * GROUP || blocks <= PAGED_WAVE_MAX;
        if (by_wave && !a_->variant && N > 2 * GROUP) {
            int64_t work = 0;
            for (int64_t row0 = 0; row0 < N; row0 += GROUP) {
                list(r, (int)row0, 1, runs_);
                for (const Run& x : runs_) work += x.count;
            }
            by_wave = work * a_->hkv * a_->d / 128 <= PAGED_WAVE_WORK;
        }
        const int groups = by_wave ? 1 : BLOCK_GROUPS, rows = groups * GROUP;
        const int64_t row_items = (N + rows - 1) / rows * a_->hkv * (by_wave && a_->d == 512 ? 2 : 1);   // (the wave kernel has a workgroup per half of 512 dims)
        std::vector<Run>& runs = runs_;
        for (int64_t row0 = 0; row0 < N; row0 += rows) {
            list(r, (int)row0, groups, runs);
            int64_t tiles = 0;
            for (const Run& x : runs) tiles += x.count;
            // Keys are divided where the request's own items leave places free, into pieces of about `size` tiles or more (at least half of it): there the partial results, written
            // and read back in 32 bits, are an eighth of the bytes of a piece's keys and values in the wave kernel and a sixth in the shared one, at most twice that.
            const int64_t places = a_->d == 512 || (by_wave && a_->d == 256) ? PAGED_PLACES / 2 : PAGED_PLACES, size = by_wave ? PAGED_WAVE_TILES : PAGED_BLOCK_TILES;
            int64_t want = std::max<int64_t>(1, places / row_items);
            const int64_t per = std::max(size, (tiles + want - 1) / want);
            const int64_t nsplit = std::max<int64_t>(1, (tiles + per - 1) / per);
            const int64_t here = std::min<int64_t>(rows, N - row0);
            cut_.clear();
            size_t at = 0;
            int64_t off = 0;
            for (int64_t s = 0; s < nsplit; s++) {
                int64_t left = tiles * (s + 1) / nsplit - tiles * s / nsplit;
                const int32_t here = (int32_t)left, first = (int32_t)p_->runs.size();
                while (left > 0) {
                    const int64_t take = std::min<int64_t>(left, runs[at].count - off);
                    p_->runs.push_back({(int32_t)(runs[at].kt + off), (int32_t)take, runs[at].bits, here - (int32_t)left});
                    left -= take;
                    off += take;
                    if (off == runs[at].count) { at++; off = 0; }
                }
                cut_.push_back({first, (int32_t)p_->runs.size() - first, here});
            }
            for (int h = 0; h < a_->hkv; h++) {
                const int64_t part = p_->part_rows;
                if (nsplit > 1) {
                    int share = 1;   // (each group asks for four pieces at a time)
                    while (share < PAGED_JOIN && share * 4 < nsplit) share *= 2;
                    for (int64_t j = 0; j < here; j += PAGED_JOIN / share)
                        p_->joins.push_back({r.cu, h, (int32_t)(row0 + j), (int32_t)std::min<int64_t>(PAGED_JOIN / share, here - j), (int32_t)(part + j), (int32_t)nsplit, rows, share});
                    p_->part_rows += nsplit * rows;
                }
                for (int64_t s = 0; s < nsplit; s++)
                    (by_wave ? p_->wave : p_->block)
                        .push_back({r.cu, r.T, r.L, r.tab, h, (int32_t)row0, cut_[s].first, cut_[s].runs, cut_[s].tiles, nsplit > 1 ? (int32_t)(part + s * rows) : -1, index,
                                    (int32_t)nsplit});
            }
        }
    }

    // Launch order.  Workgroup i runs on XCD i % 8: the items of one (request, key / value head) go to one XCD, whose L2 then holds what they
    // share, unless there are too few of these sets to fill eight; inside a set the longest items come first, and so do the heaviest sets.
    void order(std::vector<Item>& items) const {
        if (items.empty()) return;
        const int hkv = a_->hkv;
        // items by set (they were made request by request, so a set lies inside its request's stretch), longest first
        std::vector<int32_t> idx(items.size()), at(hkv + 1);
        int64_t total = 0;
        for (size_t i = 0; i < items.size();) {
            size_t j = i;
            std::fill(at.begin(), at.end(), 0);
            for (; j < items.size() && items[j].req == items[i].req; j++) at[items[j].kvh + 1]++;
            for (int h = 0; h < hkv; h++) at[h + 1] += at[h];
            for (size_t k = i; k < j; k++) {
                idx[i + at[items[k].kvh]++] = (int32_t)k;
                total += weight(items[k]);
            }
            for (int h = 0; h < hkv; h++) {   // (at[h] is the end of head h's items now)
                const auto first = idx.begin() + i + (h ? at[h - 1] : 0), last = idx.begin() + i + at[h];
                const auto longer = [&](int32_t x, int32_t y) { return items[x].tiles > items[y].tiles; };
                if (!std::is_sorted(first, last, longer)) std::stable_sort(first, last, longer);
            }
            i = j;
        }
        struct Set { size_t at, n; int64_t weight; };
        std::vector<Set> sets;
        for (size_t i = 0; i < idx.size();) {
            size_t j = i;
            int64_t w = 0;
            const Item& lead = items[idx[i]];
            // (a set heavier than a sixteenth of the call is dealt out in pieces)
            while (j < idx.size() && items[idx[j]].req == lead.req && items[idx[j]].kvh == lead.kvh && (j == i || w * 16 < total)) w += weight(items[idx[j++]]);
            sets.push_back({i, j - i, w});
            i = j;
        }
        std::stable_sort(sets.begin(), sets.end(), [](const Set& x, const Set& y) { return x.weight > y.weight; });
        std::vector<int32_t> lists[XCDS];
        for (auto& l : lists) l.reserve(items.size() / 4);
        int64_t load[XCDS] = {};
        for (const Set& s : sets) {
            const int x = (int)(std::min_element(load, load + XCDS) - load);
            load[x] += s.weight;
            lists[x].insert(lists[x].end(), idx.begin() + s.at, idx.begin() + s.at + s.n);
        }
        size_t longest = 0;
        for (const auto& l : lists) longest = std::max(longest, l.size());
        std::vector<Item> out;
        out.reserve(items.size());
        for (size_t i = 0; i < longest; i++)
            for (const auto& l : lists)
                if (i < l.size()) out.push_back(items[l[i]]);   // (a list that has run out shifts the others by one: placement, not results)
        items.swap(out);
    }
    static int64_t weight(const Item& x) { return (int64_t)x.tiles + 4; }

    struct Piece { int32_t first, runs, tiles; };

    const spinf_paged_plan_args* a_;
    spinf_pagedplan* p_;
    std::vector<Piece> cut_;   // of the row block in hand
    std::vector<Run> runs_;
    const int group_, window_;
};

int check(const spinf_paged_plan_args* a) {
    if (!a) return spinf_fail(SPINF_E_ARG, "paged_plan: null args");
    if (a->reqs < 0 || (a->reqs > 0 && (!a->q_lens || !a->kv_lens))) return spinf_fail(SPINF_E_ARG, "paged_plan: null lengths");
    if (a->hq <= 0 || a->hkv <= 0 || a->hq % a->hkv) return spinf_fail(SPINF_E_ARG, "paged_plan: %d query heads do not group over %d key / value heads", a->hq, a->hkv);
    if (a->d != 64 && a->d != 128 && a->d != 256 && a->d != 512) return spinf_fail(SPINF_E_ARG, "paged_plan: head dim %d not supported (64, 128, 256, 512)", a->d);
    if (a->page < 16 || a->page % 16 || a->page > (1 << 20)) return spinf_fail(SPINF_E_ARG, "paged_plan: pages of %d keys (a multiple of 16)", a->page);
    if ((a->end == nullptr) != (a->pos == nullptr)) return spinf_fail(SPINF_E_ARG, "paged_plan: a tree needs both end and pos");
    if (a->variant < 0 || a->variant > 2) return spinf_fail(SPINF_E_ARG, "paged_plan: variant %d", a->variant);
    if (a->window < 0) return spinf_fail(SPINF_E_ARG, "paged_plan: window %d", a->window);
    int64_t T = 0, pages = 0;
    for (int64_t r = 0; r < a->reqs; r++) {
        if (a->q_lens[r] < 0 || a->kv_lens[r] < 0 || a->kv_lens[r] > (1 << 30)) return spinf_fail(SPINF_E_ARG, "paged_plan: request %lld has %d new and %d stored tokens", (long long)r, a->q_lens[r], a->kv_lens[r]);
        if (a->end && a->q_lens[r] > a->kv_lens[r]) return spinf_fail(SPINF_E_ARG, "paged_plan: request %lld: a tree of %d new tokens, %d stored ones", (long long)r, a->q_lens[r], a->kv_lens[r]);
        T += a->q_lens[r];
        pages += ((int64_t)a->kv_lens[r] + a->page - 1) / a->page;
    }
    if (T * (a->hq / a->hkv) > (1 << 30) || pages > (1 << 30)) return spinf_fail(SPINF_E_ARG, "paged_plan: %lld new tokens, %lld pages are too many", (long long)T, (long long)pages);
    if (a->end)
        for (int64_t r = 0, t = 0; r < a->reqs; r++)
            for (int64_t i = 0; i < a->q_lens[r]; i++, t++)   // (in pre-order a token's depth is at most the number of tokens before it)
                if (a->pos[t] < 0 || a->pos[t] > a->kv_lens[r] - a->q_lens[r] + i || a->end[t] < 0 || a->end[t] > T)
                    return spinf_fail(SPINF_E_ARG, "paged_plan: row %lld has position %d and subtree end %d", (long long)t, a->pos[t], a->end[t]);
    return SPINF_OK;
}

}  // namespace

extern "C" int spinf_paged_plan_build(const spinf_paged_plan_args* a, spinf_pagedplan** out) {
    const int rc = check(a);
    if (rc) return rc;
    if (!out) return spinf_fail(SPINF_E_ARG, "paged_plan: null output");
    spinf_pagedplan* p = nullptr;
    try {
        p = new spinf_pagedplan;
        Builder(a, p).run();
        if (p->part_rows > INT32_MAX || p->runs.size() > (size_t)INT32_MAX / 16 || p->wave.size() + p->block.size() > (size_t)INT32_MAX / 16) {
            delete p;
            return spinf_fail(SPINF_E_ARG, "paged_plan: the call is too large for one plan");
        }
    } catch (const std::exception&) {
        delete p;
        return spinf_fail(SPINF_E_NOMEM, "paged_plan: out of memory");
    }
    *out = p;
    return SPINF_OK;
}

extern "C" int spinf_paged_plan_counts(const spinf_pagedplan* p, int64_t counts[5]) {
    if (!p || !counts) return spinf_fail(SPINF_E_ARG, "paged_plan_counts: null pointer");
    counts[0] = (int64_t)p->wave.size();
    counts[1] = (int64_t)p->block.size();
    counts[2] = (int64_t)p->runs.size();
    counts[3] = (int64_t)p->joins.size();
    counts[4] = p->part_rows;
    return SPINF_OK;
}

extern "C" int spinf_paged_plan_export(const spinf_pagedplan* p, int32_t* wave, int32_t* block, int32_t* runs, int32_t* joins) {
    if (!p || (!wave && !p->wave.empty()) || (!block && !p->block.empty()) || (!runs && !p->runs.empty()) || (!joins && !p->joins.empty()))
        return spinf_fail(SPINF_E_ARG, "paged_plan_export: null pointer");
    std::copy(p->wave.begin(), p->wave.end(), (Item*)wave);
    std::copy(p->block.begin(), p->block.end(), (Item*)block);
    std::copy(p->runs.begin(), p->runs.end(), (Run*)runs);
    std::copy(p->joins.begin(), p->joins.end(), (Join*)joins);
    return SPINF_OK;
}

extern "C" void spinf_paged_plan_free(spinf_pagedplan* p) { delete p; }
