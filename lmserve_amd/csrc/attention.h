// What the kernels of the attention over a 16-bit cache and over an 8-bit one share: the step's layout, as the plan's launch
// writes it, and the launch's arguments.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "types.h"

namespace kvc {
namespace attn {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 16;          // rows of a narrow item
constexpr int kWide = 32 * kWaves; // rows of a wide item: 32 to a wavefront
constexpr int kStep = 64;          // keys that a workgroup takes at once of a wide item
constexpr int kAhead = 3;          // pieces of a wide item's K and V that are read from LDS ahead of their product
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

struct Item {  // 32 bytes: a tile or a part of one
  int32_t q_begin;  // first token of the request; -1: the rows of all sharing requests, through shared_tokens
  int32_t row0, rows, table, key_begin, key_end;
  int32_t slot;     // of its partial; -1: the whole tile
  int32_t limit;    // keys that the request's first token sees, each further one a key more (less than 1: none)
};
struct Parts {  // 16 bytes: of a tile: the slot of the first, and of the c-th further one next + c * step
  int32_t slot, next, step, count;
};
struct Entry {  // 32 bytes: rows of one tile that are joined from partials
  int32_t q_begin, row0;
  int16_t rows, many;   // (a single one, of many parts)
  int32_t shared_row0;  // the first row among those of the sharing requests, or -1
  Parts parts;
};
struct Range {
  int32_t begin, end;
};
struct Header {
  int32_t wide_items, narrow_entries, wide_entries, shared_wide;  // (narrow entries from the front, wide ones from the back)
  int32_t shared_tiles, shared_count;  // of wide tiles of the sharing rows: tile t's parts are t + c * shared_tiles
};

struct Layout {  // the plan's device buffer
  Header* header;
  int32_t* shares;         // [B] 1: its leading pages are the shared ones
  int2* shared_tokens;     // [T] token, and the keys it sees
  Range* ranges;           // [groups] narrow items of a workgroup
  Item* items[2];          // narrow: tile t's part in workgroup w at t + w: those of a workgroup lie side by side
  Parts* shared_parts;     // of the narrow tiles of the sharing requests' rows (of wide ones the header has them)
  Entry* entries;
};

__device__ __forceinline__ int32_t clamp(int32_t x, int32_t lo, int32_t hi) { return x < lo ? lo : x > hi ? hi : x; }

struct AttendArgs {
  const char* query;
  const char* cache;
  const int32_t* kv_indices;
  char* out;
  float* lse;              // may be null
  float* partial[2];       // narrow, wide: [slots][kv heads][rows of a tile][head_dim]
  float* partial_lse[2];   // [slots][kv heads][rows of a tile], to base 2
  int64_t q_stride;        // bytes
  uint32_t page_stride, row_stride, plane;  // bytes: page to page, key to key in a page (none in an 8-bit cache), K to V
  int32_t num_pages, page_size, page_shift;
  int32_t kv_heads, group, head_dim;
  int32_t narrow_groups, wide_groups;  // workgroups, of all key heads
  int32_t max_entries;
  uint32_t group_stride, exponents;    // of an 8-bit cache, bytes: group to group of 16 keys, a group's exponents
  float scale;             // times log2(e)
  Layout l;
};

// Row r of the tile of a key head whose partial is in a slot. In 64 bits: with 8 columns a workspace of 155 GB has 2^32 rows.
__host__ __device__ constexpr int64_t partial_row(int32_t slot, int32_t kv_heads, int32_t h, int32_t tile, int32_t r) {
  return ((int64_t)slot * kv_heads + h) * tile + r;
}

// The larger of a lane's value and that of the lane 32 (16) further on or before, without LDS
__device__ __forceinline__ float max_across32(float x) {
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ __forceinline__ float max_across16(float x) {
  const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ bool finite(float x) { return __builtin_fabsf(x) <= 3.402823466e38f; }
// The least weight of a part: however far below the others it is, what is infinite in it stays
constexpr float kLeastWeight = 1.401298464e-45f;

// A workgroup of a key head takes its share's items one after the other
template <typename Narrow>
__device__ __forceinline__ void take_share(const AttendArgs& a, int32_t at, const Narrow& narrow) {
  const int32_t group = at / a.kv_heads, h = at - group * a.kv_heads;
  const Range range = a.l.ranges[group];
  for (int32_t i = range.begin; i < range.end; ++i) narrow(a.l.items[0][i], h);
}

// Steps that may have wide tiles: both kinds in one launch, side by side on the card, as the narrow ones wait for memory and
// the wide ones for the matrix units. 32 workgroups of a kind in turn: they are dealt to the 8 XCDs and there to 4 shader
// engines in rotation (8 in turn put all wide ones on half of the engines: 2048 new tokens 1218 us, 917 so). The wide items, of one key head
// after the other, are dealt to the XCDs in eight runs, so that items that read the same keys share an L2.
// Over 8 bits the wide ones go first: narrow ones take half the time, and what is left at the end are wide ones (3 chunks of 259 tokens and 60 single
// ones 65 us in turn and 56 so, 2 of 300 and 58 63 and 58, 256 single ones behind a shared prompt 68 and 69).
template <bool WIDE_FIRST, typename Narrow, typename Wide>
__device__ __forceinline__ void take_step(const AttendArgs& a, const Narrow& narrow_item, const Wide& wide_item) {
  const int32_t narrow = a.narrow_groups;
  const int32_t both = WIDE_FIRST ? 0 : (narrow < a.wide_groups ? narrow : a.wide_groups) & ~31;
  int32_t at = blockIdx.x;
  bool is_wide;
  if (at < 2 * both) {
    is_wide = (at & 32) == 0;
    at = (at >> 6) * 32 + (at & 31);
  } else {
    at -= both;  // what is left of either, the wide first
    is_wide = at < a.wide_groups;
    if (!is_wide) at = at - a.wide_groups + both;
  }
  if (!is_wide) {
    take_share(a, at, narrow_item);
    return;
  }
  const int32_t items = a.l.header->wide_items, all = items * a.kv_heads, run = (all + 7) / 8;
  for (int32_t i = at >> 3; i < run; i += a.wide_groups >> 3) {
    const int32_t x = (at & 7) * run + i;
    if (x >= all) break;
    const int32_t h = x / items;
    const Item item = a.l.items[1][x - h * items];
    if (item.rows) wide_item(item, h);
  }
}

// The 8-bit cache's kernels (attention_q8.hip): the step's tiles, `wide` where there may be wide ones
void launch_q8(const AttendArgs& a, bool f16, bool wide, bool past_the_caches, hipStream_t s);
constexpr int q8_narrow_residents(int dim) { return dim <= 64 ? 3 : dim <= 128 ? 2 : 1; }  // narrow workgroups of a CU

}  // namespace attn
}  // namespace kvc
