// What the kernel that keeps the seats' books and the attention over seats share: the work lists' layout, and the rules by which keys are cut, which the host needs too for how
// long the lists may get.
#pragma once
#include <cstdint>

#include "paged.h"

#if defined(__HIPCC__)
#define SEATS_BOTH __host__ __device__ __forceinline__
#else
#define SEATS_BOTH inline
#endif

constexpr int SEATS_MOST = 2048;      // seats: their lengths and running sums lie in LDS
constexpr int SEATS_KINDS = 8;        // head geometries
constexpr int SEATS_ROWS_AT_ONCE = 8192;   // rows that the workgroup of the books places itself; more get a launch of their own

// Rows row0 .. of a set of new tokens (tokens tok0 .. tok0 + T - 1 of the call, `group` rows each) over tiles kt0 .. kt0 + tiles - 1 of a span of L keys whose pages begin
// at `tab` of the page lists.  A span is a content, shared by the set's seats, or a seat's own keys (SEAT_OWN: row t sees them up to L - T + t).  Every row of the item sees the
// keys flo .. fhi; piece: which of its rows' partial results this is (SEAT_ONLY: there is no other).
struct SeatItem { int32_t tok0, T, L, tab, row0, kt0, tiles, piece, flo, fhi, flags, unused; };
static_assert(sizeof(SeatItem) == 48, "written and read as 16-byte pieces");
constexpr int SEAT_OWN = 1, SEAT_ONLY = 2;

// A seat's own keys, few rows: one wave takes up to SEAT_SINGLE_TILES tiles by itself (no join of waves, four such items per workgroup); more are divided among the waves
// of a workgroup, and from SEAT_WAVE_TILES on among workgroups.  Many rows, and contents, go to four waves of 32 rows each on shared tiles.
constexpr int SEAT_SINGLE_TILES = 4;
constexpr int SEAT_WAVE_ROWS = 64;
constexpr int SEAT_WAVE_TILES = 16;
constexpr int SEAT_BLOCK_TILES = 48;
constexpr int SEAT_SHARED_TILES = 16;
SEATS_BOTH int seats_least(int a, int b) { return a < b ? a : b; }
SEATS_BOTH int seats_most(int a, int b) { return a > b ? a : b; }
SEATS_BOTH int seats_up(int a, int b) { return (a + b - 1) / b; }
// pieces of `tiles` tiles: as many as pieces of `size` would be begun, where `items` workgroups each leave places for that many
SEATS_BOTH int seats_pieces(int tiles, int size, int places, int items) { return seats_most(1, seats_least(seats_up(tiles, size), places / seats_most(items, 1))); }
SEATS_BOTH int seats_wave_pieces(int tiles, int d, int hkv, int blocks) { return seats_pieces(tiles, SEAT_WAVE_TILES, d >= 256 ? PAGED_PLACES / 2 : PAGED_PLACES, blocks * hkv * (d == 512 ? 2 : 1)); }
SEATS_BOTH int seats_block_pieces(int tiles, int d, int hkv, int blocks, bool shared) {
    return seats_pieces(tiles, shared ? SEAT_SHARED_TILES : SEAT_BLOCK_TILES, d == 512 ? PAGED_PLACES / 2 : PAGED_PLACES, blocks * hkv);
}
