// What the plan compiler and the kernels of the paged cache share: the work lists' layout, and the limits that decide how a request is cut.
#pragma once
#include <cstdint>

constexpr int PAGED_TILE = 32;           // keys per tile
constexpr int PAGED_ROWS = 32;           // rows per row group (row = new token * query heads per key / value head + head)
constexpr int PAGED_BLOCK_GROUPS = 4;    // row groups of a block item

// `count` tiles from kt on, the item's tiles start .. start + count - 1; bits: 1 << g some row of row group g sees a key, 16 << g some pair of it is
// masked (all of them, where the group sees nothing: the kernel computes the tile for every group of the item)
struct PagedRun { int32_t kt, count; uint32_t bits; int32_t start; };
// rows row0 .. of key / value head kvh of the request whose new tokens are rows cu .. cu + T - 1 of the call and whose L stored keys lie in the pages
// tab .. of the page list; runs first .. first + runs - 1 (`tiles` tiles); part: first partial row, -1: the only piece
struct PagedItem { int32_t cu, T, L, tab, kvh, row0, first, runs, tiles, part, req, nsplit; };
constexpr int PAGED_JOIN = 16;            // groups of 16 lanes that join rows: up to PAGED_JOIN / share rows, `share` groups to each
// rows row0 .. row0 + rows - 1, whose nsplit pieces (partial rows part + s * stride + j) are to be joined
struct PagedJoin { int32_t cu, kvh, row0, rows, part, nsplit, stride, share; };
static_assert(sizeof(PagedRun) == 16 && sizeof(PagedItem) == 48 && sizeof(PagedJoin) == 32, "read by the kernels as 16-byte pieces");

// Workgroups that run at a time (two per compute unit, one where a workgroup's tiles fill its LDS: 512 dims, and 256 dims in the wave kernel).  A request's keys are cut
// for that many, and not more: a second round of workgroups costs its start and its share of the join (one token over 131,071 keys of 512 dims, one
// key / value head: 256 workgroups 45.8 + 4.9 us for the join, 482 52.9 + 6.6).
constexpr int PAGED_PLACES = 512;
// Which kernel takes a request, by its own size alone.  The waves that divide the keys read them once per 32 rows and are the faster where the request leaves the GPU
// mostly idle; the shared tiles read them once per 128 rows and are the faster where it, or others like it, fill the GPU (us, 1 / 16 such requests in a call, wave -> shared):
//   16 heads on 8 of 256 dims, 160 new on 2,000 stored  36 / 378 -> 58 / 187     48 new on 8,000  37 / 438 -> 71 / 257     160 new on 400  20 / 101 -> 34 / 50
//   32 heads on 16 of 128,     160 new on 2,000         25 / 252 -> 44 / 185     48 new on 8,000  25 / 319 -> 55 / 245     160 new on 400  18 / 76 -> 26 / 43
// Up to PAGED_WAVE_MAX workgroups of the shared kernel and PAGED_WAVE_WORK tiles of 32 rows x 32 keys x 128 dims the request goes to the waves: there the two are
// even at about four such requests in a call (80 new on 2,000, 8 heads of 256 dims: 56 / 59 us; 16 heads of 128: 43 / 45).
// Up to 64 rows per key / value head it always does: half and more of the shared kernel's rows would idle (48 rows on 8,000 keys, 8 heads of 256 dims: 23 / 314 -> 67 / 247).
constexpr int PAGED_WAVE_MAX = 64;
constexpr int PAGED_WAVE_WORK = 5000;
// Tiles of a piece there: a row group's keys are cut into as many equal pieces as pieces of this size would be begun, so one holds at least half of it (17 tiles: 8 and 9), where
// the request's places allow that many (us at 8 / 16 / 32: one token over 4,000 keys, 8 heads of 256 dims 11 / 14 / 21; 64 such requests of 3,000 keys, 4 heads: 171 / 149 / 140).
constexpr int PAGED_WAVE_TILES = 16;
// The same for the shared kernel (us at 32 / 48 / 64; a call of 1 and of 16 requests, 640 rows per key / value head on 8,000 stored keys: 8 heads of
// 256 dims 79 / 80 / 98 and 963 / 889 / 861, 16 heads of 128 dims 70 / 72 / 84 and 892 / 907 / 882; a window of 1,024 under 512 new tokens 143 / 98 / 98).
constexpr int PAGED_BLOCK_TILES = 48;
