// What the plan compiler and the kernels of the paged cache share: the work lists' layout, and the limits that decide how a request is cut.
#pragma once
#include <cstdint>

constexpr int PAGED_TILE = 32;           // keys per tile
constexpr int PAGED_ROWS = 32;           // rows per row group (row = new token * query heads per key / value head + head)
constexpr int PAGED_BLOCK_GROUPS = 4;    // row groups of a block item

// `count` tiles from kt on, the item's tiles start .. start + count - 1; bits: 1 << g some row of row group g sees a key, 16 << g some pair is masked
struct PagedRun { int32_t kt, count; uint32_t bits; int32_t start; };
// rows row0 .. of key / value head kvh of the request whose new tokens are rows cu .. cu + T - 1 of the call and whose L stored keys lie in the pages
// tab .. of the page list; runs first .. first + runs - 1 (`tiles` tiles); part: first partial row, -1: the only piece
struct PagedItem { int32_t cu, T, L, tab, kvh, row0, first, runs, tiles, part, req, nsplit; };
constexpr int PAGED_JOIN = 16;            // groups of 16 lanes that join rows: up to PAGED_JOIN / share rows, `share` groups to each
// rows row0 .. row0 + rows - 1, whose nsplit pieces (partial rows part + s * stride + j) are to be joined
struct PagedJoin { int32_t cu, kvh, row0, rows, part, nsplit, stride, share; };
static_assert(sizeof(PagedRun) == 16 && sizeof(PagedItem) == 48 && sizeof(PagedJoin) == 32, "read by the kernels as 16-byte pieces");

constexpr int PAGED_PLACES = 512;        // workgroups of either kernel that run at a time (two per compute unit)
constexpr int PAGED_WAVE_MAX = 64;      // block items of a request up to which its rows go to the kernel whose waves divide the keys
constexpr int PAGED_WAVE_TILES = 16;     // least tiles of a piece there
constexpr int PAGED_BLOCK_TILES = 64;    // least tiles of a piece of a block item
