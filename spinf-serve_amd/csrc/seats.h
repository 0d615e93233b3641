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

// Tiles kt0 .. kt0 + tiles - 1 of L keys whose pages begin at `tab` of the page lists: a content's, or (own) a seat's, of which row t of T sees those up to L - T + t.  Every row
// of the item sees the keys flo .. fhi.
struct SeatSpan { int32_t tab, L, kt0, tiles, flo, fhi, own, unused; };
// Rows row0 .. of a set of new tokens (tokens tok0 .. tok0 + T - 1 of the call, `group` rows each) over one span, or over a content and then the seat's own keys; piece: which of
// its rows' partial results this is (only: there is no other).
struct SeatItem { int32_t tok0, T, row0, piece, only, unused[3]; SeatSpan span[2]; };
// One token of a seat whose own keys lo .. L - 1 are few: their pages (more than SEAT_PAGES are looked up from `tab` on), and the partial results that its content left
constexpr int SEAT_PAGES = 6;
struct SeatLast { int32_t tok, L, lo, tab, part, parts, page[SEAT_PAGES]; };
static_assert(sizeof(SeatSpan) == 32 && sizeof(SeatItem) == 96 && sizeof(SeatLast) == 48, "written and read as 16-byte pieces");

// Who takes what, by a seat's rows (new tokens x query heads per key / value head) and the keys of its own that they see:
//   a token on few keys, in a step of many such                     a wave, without LDS, that also joins what the content's pieces left (seats_last)
//   up to SEAT_SHARED_ROWS rows on at most SEAT_SINGLE_TILES tiles  a wave to 32 rows
//   up to 32 rows                                                   four waves that divide the tiles
//   up to SEAT_SHARED_ROWS rows                                     four waves of 32 rows each on shared tiles
//   more                                                            the same, over the content's keys and then its own: such a seat gains nothing by sharing its content's reading, and this way its
//                                                                   results need no joining (150 tokens of 2 heads on 1,024 + 211 keys, 35 seats: 260 us with the content shared and all pieces joined)
// The other seats' contents go to four waves of 32 rows each, or up to SEAT_WAVE_ROWS rows below one content (32, where the step has more rows than waves run at a time: 48 contents of 300
// keys with 56 rows each 112 us, with 64 127; one content of 228 with 36 rows 21 us on shared tiles, 15 so) to waves that divide the tiles.
constexpr int SEAT_LAST_HEADS = 2, SEAT_LAST_KEYS = 128;
constexpr int SEAT_SINGLE_TILES = 4;
constexpr int SEAT_WAVE_ROWS = 64;
constexpr int SEAT_SHARED_ROWS = 96;
// Keys are cut so that the items of a step fill the places that run at a time, and into pieces of no less than these; which piece size that is goes by all of a step's lengths.
constexpr int SEAT_WAVE_TILES = 8, SEAT_BLOCK_TILES = 4;

SEATS_BOTH int seats_least(int a, int b) { return a < b ? a : b; }
SEATS_BOTH int seats_most(int a, int b) { return a > b ? a : b; }
SEATS_BOTH int seats_up(int a, int b) { return (a + b - 1) / b; }
// Are tokens on up to SEAT_LAST_KEYS keys the vector unit's, without LDS, or the matrix unit's, a wave to each?  `tokens` of them on `keys` keys in all; one way for all, since each costs the
// latency of a list.  The vector unit reads eight keys of 256 dims at a time, each a wait for memory, but with four times as many waves at a time; the work of a tile hardly depends on its keys.
//   16 on 8 heads of 256, seats x keys, us vector / matrix: 1 x 14 18 / 14, 24 x 14 23 / 19, 96 x 6 25 / 31, 96 x 28 36 / 35, 192 x 28 41 / 50, 192 x 60 53 / 56, 192 x 120 93 / 74, 1344 x 14 82 / 138
// At 64 dims, and from four heads to a key / value head on, tiles are never slower by much (1,344 x 14, 32 on 4 of 128: 94 / 70; 16 on 4 of 64: 49 / 42).
SEATS_BOTH bool seats_last(int group, int d) { return group <= SEAT_LAST_HEADS && d >= 128; }
SEATS_BOTH bool seats_last_pays(long tokens, long keys, int hkv) { return tokens * hkv >= 640 && keys <= 64 * tokens && 50 * keys <= tokens * tokens * hkv; }
// workgroups that run at a time: of waves that divide the tiles (512 dims: two to an item), of waves on shared tiles
SEATS_BOTH int seats_wave_places(int d) { return d == 512 ? PAGED_PLACES / 4 : d == 256 ? PAGED_PLACES / 2 : PAGED_PLACES; }
SEATS_BOTH int seats_block_places(int d) { return d == 512 ? PAGED_PLACES / 2 : PAGED_PLACES; }
