// Causal attention of a step's queries over the paged K/V cache (gfx950).
//
// Row r of a request is (token, query head): with G = query heads per key head, the G heads of a token that share a key
// head are G rows of one matrix, so grouped heads read a key once. For a row with limit `lim` (its position + 1):
//   s_k = scale q.k,  m = max s,  l = sum_k exp(s_k - m),  o = sum_k exp(s_k - m) v_k / l     over k < lim,
// in one pass over the keys: where the running maximum grows, what was summed is scaled by exp(m_old - m_new).
// Ranges of keys that different workgroups took are joined by their lse = m + log l: o = sum_c exp(lse_c - lse) o_c.
// Exponentials are taken to base 2, with scale * log2(e) in the exponent's multiply-add.
//
// A step's work is laid out on the device, from the index tensors (a small launch, two with a shared prefix, once per step): items of
// (row tile, key range) of about equal length, as many as fill the card, however the lengths are spread. The leading
// pages that the requests of a batch share are items of their own, whose rows are those of ALL these requests.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <type_traits>

#include "common.h"
#include "device.h"
#include "kvcache.h"

namespace {

using kvc::fail;
using kvc::log2_exact;
using kvc::u32x4;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 16;          // rows of a narrow item
constexpr int kWide = 32 * kWaves; // rows of a wide item: 32 to a wavefront
constexpr int kBlock = 32;         // keys that a wavefront takes at once of a narrow item
constexpr int kStep = 64;          // keys that a workgroup takes at once of a wide item
constexpr int kVPad = 64;          // bytes between a wide item's rows of V in LDS
constexpr int kAhead = 3;          // pieces of a wide item's K and V that are read from LDS ahead of their product
constexpr int kMaxGroups = 1024;    // workgroups of a key head
// In keys: what a narrow tile costs beside its own, a workgroup's least share, the least part of a tile. With the least
// share there are workgroups to spare, and a part is half of it: a short tile in one piece is done sooner than cut
// and joined (900 keys of one request: 17.4 us whole, 18.6 to 19.7 in two to four). Behind a shared prefix every tile is joined.
__device__ constexpr int kTileWork = 64, kMinShare = 1024, kMinSharedShare = 256, kMinPart = 256;
// the least range of a wide tile; what an item costs beside its keys, and what one that leaves a partial does
__device__ constexpr int kMinChunk = 512, kWideTileWork = 128, kWidePartWork = 384;
constexpr int32_t kMaxKeys = INT32_MAX - 8192;  // of a request: a key that is looked up ahead stays below 2^31
// The rows of all sharing requests are wide tiles where they are more than kNarrowSharedRows, or more than a narrow tile and
// rows times keys above kNarrowWork. 8 key heads of 128, wide and narrow: 96 rows over 4096 keys 27.3 and 33.9 us, 128 rows 28.5 and
// 40.8, 64 rows 25.7 and 26.6; 96 over 1024 23.2 and 21.2, 24 over 2000 23.1 and 16.7. (With fewer key heads the narrow tiles have
// more of the card to themselves, which the rule does not look at: one key head, 128 rows over 4096 keys 25.2 and 18.1.)
__host__ __device__ constexpr bool wide_prefix(int64_t rows, int64_t keys) {
  constexpr int64_t kNarrowSharedRows = 128, kNarrowWork = 1 << 18;
  return rows > kNarrowSharedRows || (rows > kTile && rows * keys > kNarrowWork);
}
constexpr int kManyParts = 16;     // a row of more partials is joined by a workgroup
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

// ---- the step's layout ---------------------------------------------------------------------------------------------
// Row tiles are of 16 rows (narrow, of requests of few rows) or of 128 (wide), each over the keys that its last row sees.
//   Narrow tiles lie end to end on a line of work, measured in keys, that is cut into as many equal shares as there are
//   workgroups for a key head: a workgroup takes the pieces of tiles in its share, so that every one has the same work
//   whatever the lengths are. Of a share only the first and the last piece can be parts of a tile. A cut that would leave
//   a sliver moves to the tile's end.
//   Wide tiles of a request read the same keys: they are cut at the same keys, and the tiles of one range of keys are
//   neighbours in the list and run on one XCD, whose L2 the range then comes to once (2048 new
//   tokens behind 13 to 30 thousand keys 834 us; the tiles dealt to all XCDs in turn 854).
// A part of a tile leaves its rows' unfinished result in a slot of the workspace, and the parts are joined at the end.
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
};

struct Layout {  // the plan's device buffer
  Header* header;
  int32_t* shares;         // [B] 1: its leading pages are the shared ones
  int2* shared_tokens;     // [T] token, and the keys it sees
  Range* ranges;           // [groups] narrow items of a workgroup
  Item* items[2];          // narrow: tile t's part in workgroup w at t + w: those of a workgroup lie side by side
  Parts* shared_parts;     // of the tiles of the sharing requests' rows
  Entry* entries;
};

struct PlanArgs {
  const int32_t *qo_indptr, *kv_indices, *kv_indptr, *kv_last_page_len;
  int32_t batch_size, num_tokens, num_kv_indices, page_size, shared_pages, group;
  int32_t narrow_rows;                      // the most rows of a request for narrow tiles
  int32_t groups, residents;                // of a key head: workgroups for narrow tiles, wide tiles on the card at a time
  int32_t max_items[2], max_entries;
  Layout l;
};

__device__ __forceinline__ int32_t clamp(int32_t x, int32_t lo, int32_t hi) { return x < lo ? lo : x > hi ? hi : x; }

struct Table {
  int32_t begin, pages;
};
__device__ __forceinline__ Table table_of(const PlanArgs& a, int32_t b) {
  const int32_t begin = clamp(a.kv_indptr[b], 0, a.num_kv_indices);
  return {begin, clamp(a.kv_indptr[b + 1], begin, a.num_kv_indices) - begin};
}
__device__ __forceinline__ Table tokens_of(const PlanArgs& a, int32_t b) {
  const int32_t begin = clamp(a.qo_indptr[b], 0, a.num_tokens);
  return {begin, clamp(a.qo_indptr[b + 1], begin, a.num_tokens) - begin};
}

__device__ __forceinline__ int32_t keys_of(const PlanArgs& a, int32_t b, int32_t pages) {
  if (!pages) return 0;
  const int64_t keys = (int64_t)(pages - 1) * a.page_size + clamp(a.kv_last_page_len[b], 0, a.page_size);
  return (int32_t)(keys < kMaxKeys ? keys : kMaxKeys);
}

// A workgroup per request: does it begin with the shared pages? Which pages these are is what the first request with few
// tokens and that many pages holds; a request that holds others is a request by itself, so that the number of shared
// pages changes how the work is cut and never the result. (Of the requests of many rows none share: they read a key for 128
// rows as it is.)
__device__ __forceinline__ bool may_share(const PlanArgs& a, int32_t b) {
  const int32_t n = tokens_of(a, b).pages;
  return n > 0 && n * a.group <= a.narrow_rows && table_of(a, b).pages >= a.shared_pages;
}
__global__ __launch_bounds__(256) void attend_shares_kernel(PlanArgs a) {
  __shared__ int32_t first, differ;
  const int32_t b = blockIdx.x, tid = threadIdx.x;
  bool shares = may_share(a, b);
  if (shares) {
    if (tid == 0) {
      first = b;
      differ = 0;
    }
    __syncthreads();
    for (int32_t c0 = 0; c0 < b; c0 += 256) {
      if (c0 + tid < b && may_share(a, c0 + tid)) atomicMin(&first, c0 + tid);
      __syncthreads();
      const bool found = first < b;
      __syncthreads();  // everyone has looked before someone lowers it further
      if (found) break;
    }
    const int32_t* mine = a.kv_indices + table_of(a, b).begin;
    const int32_t* theirs = a.kv_indices + table_of(a, first).begin;
    bool other = false;
    for (int32_t i = tid; i < a.shared_pages; i += 256) other = other || mine[i] != theirs[i];
    if (other) differ = 1;
    __syncthreads();
    shares = !differ;
  }
  if (tid == 0) a.l.shares[b] = shares;
}

__device__ __forceinline__ int32_t ceil_div(int32_t x, int32_t y) { return (int32_t)(((uint32_t)x + (uint32_t)y - 1) / (uint32_t)y); }
__device__ __forceinline__ int32_t round_up(int32_t x, int32_t to) { return ceil_div(x, to) * to; }

// A request's tiles
struct Tiles {
  uint32_t at;              // narrow: where the first begins on the line of work, in units
  int32_t q_begin, n, len, table;
  int32_t begin;            // first key of its own
  int32_t tiles, first;     // and the first's place in its list
  int32_t first_slot;       // wide
  int32_t shared_token0;    // its first token among the sharing ones, or -1
  int32_t wide;
  __device__ __forceinline__ int32_t rows_of_tile() const { return wide ? kWide : kTile; }
  // Work of the narrow tiles before the i-th: each sees tile / group keys more than the one before, and costs something by itself
  __device__ __forceinline__ int64_t before(int32_t i, int32_t group) const {
    const int32_t keys = min(len, len - n + ceil_div(kTile, group)) - begin;
    const int64_t more = i < 2 ? 0 : (int64_t)i * (i - 1) / 2 * kTile / group;
    return (int64_t)i * ((keys > 0 ? keys : 0) + kTileWork) + more;
  }
  // Ranges of keys that wide tiles are cut into where none is to be longer than `chunk`
  __device__ __forceinline__ int32_t chunks(int32_t chunk) const { return max(ceil_div(len, chunk), 1); }
};
__device__ __forceinline__ Tiles tiles_of(const PlanArgs& a, int32_t b) {
  const Table q = tokens_of(a, b), table = table_of(a, b);
  Tiles t = {};
  t.q_begin = q.begin;
  t.n = q.pages;
  t.len = keys_of(a, b, table.pages);
  t.table = table.begin;
  t.wide = t.n * a.group > a.narrow_rows;
  const bool shares = a.shared_pages > 0 && a.l.shares[b];
  t.shared_token0 = shares ? 0 : -1;
  t.begin = shares ? min(a.shared_pages * a.page_size, t.len) : 0;
  t.tiles = ceil_div(t.n * a.group, t.rows_of_tile());
  return t;
}

// The parts of a narrow tile at `at`, `work` long, when the line is cut every `share`
struct Cuts {
  int32_t group, count;  // the first part's workgroup, and how many parts there are
};
__device__ __forceinline__ Cuts cuts_of(const PlanArgs& a, uint32_t at, uint32_t work, uint32_t share, uint32_t sliver) {
  // (the line may end within a sliver of the last share's end)
  const int32_t first = min((int32_t)((at + sliver - 1) / share), a.groups - 1);
  const int32_t last = at + work < sliver ? 0 : (int32_t)((at + work - sliver) / share);
  return {first, (last > first ? last - first : 0) + 1};
}
// Rows of an entry: one of many parts is by itself
__device__ __forceinline__ int32_t joined_rows(int32_t parts) { return parts > kManyParts ? 1 : kTile; }

// One workgroup: the share and the wide tiles' ranges, from all the work there is; where each request's tiles begin, by a scan;
// the lists. The line of work is measured in units of as many keys as let it end below 2^30. A thread does a request of
// few items, a wavefront one of many.
__global__ __launch_bounds__(1024) void attend_schedule_kernel(PlanArgs a) {
  constexpr int SUMS = 5;  // narrow work, narrow tiles, wide items, wide slots, sharing tokens
  constexpr int kFew = 4;  // items of a request that its thread does
  __shared__ unsigned long long narrow_work, wide_work, best;
  __shared__ int32_t wave_sums[16][SUMS], carry[SUMS], shared_tokens, some_request, entries[2], longest, num_long, out_of_order;
  __shared__ int32_t first_item[kMaxGroups], last_item[kMaxGroups];
  __shared__ int2 wide_tiles[1024];  // tiles and keys of those of the first requests that are wide
  __shared__ Tiles long_requests[1024];
  const int32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Tiles mine = {};
  mine.shared_token0 = -1;
  if (tid < a.batch_size) mine = tiles_of(a, tid);
  if (tid == 0) {
    narrow_work = wide_work = 0;
    best = ~0ull;
    shared_tokens = entries[0] = entries[1] = longest = out_of_order = 0;
    some_request = INT32_MAX;
  }
  for (int32_t w = tid; w < a.groups; w += 1024) {
    first_item[w] = INT32_MAX;
    last_item[w] = -1;
  }
  __syncthreads();
  wide_tiles[tid] = mine.wide ? make_int2(mine.tiles, mine.len) : make_int2(0, 0);
  for (int32_t b = tid; b < a.batch_size; b += 1024) {
    const Tiles t = b < 1024 ? mine : tiles_of(a, b);
    if (a.qo_indptr[b] > a.qo_indptr[b + 1] || a.kv_indptr[b] > a.kv_indptr[b + 1]) out_of_order = 1;
    if (t.tiles && !t.wide) atomicAdd(&narrow_work, (unsigned long long)t.before(t.tiles, a.group));
    if (t.wide) {
      atomicAdd(&wide_work, (unsigned long long)t.tiles * t.len);
      atomicMax(&longest, t.len);
    }
    if (t.shared_token0 >= 0) {
      atomicAdd(&shared_tokens, t.n);
      atomicMin(&some_request, b);
    }
  }
  __syncthreads();
  // Requests that are to have the same rows or pages: the lists' sizes hold for those that have their own. Nothing is done.
  if (out_of_order) {
    if (tid == 0) *a.l.header = {};
    for (int32_t w = tid; w < a.groups; w += 1024) a.l.ranges[w] = Range{0, 0};
    return;
  }
  const int32_t shared_rows = shared_tokens * a.group, shared_len = a.shared_pages * a.page_size;
  const bool shared_wide = wide_prefix(shared_rows, shared_len);
  const int32_t shared_tile = shared_wide ? kWide : kTile, shared_tiles = ceil_div(shared_rows, shared_tile);
  const int64_t all_narrow = (int64_t)narrow_work + (shared_wide ? 0 : shared_tiles * ((int64_t)shared_len + kTileWork));
  const int32_t unit = max(0, 34 - (int32_t)__clzll((unsigned long long)all_narrow + 1));  // log2 of the keys of a unit
  const uint32_t shared_work = (uint32_t)(((int64_t)shared_len + kTileWork) >> unit);      // of a narrow tile
  // (rounding down tile by tile, the line is no longer than this)
  const uint32_t least = max((shared_rows ? kMinSharedShare : kMinShare) >> unit, 1);
  const uint32_t share = max((uint32_t)ceil_div((int32_t)(all_narrow >> unit), a.groups), least);
  const uint32_t sliver = max(share <= least ? share / 2 : min(share / 2, (uint32_t)(kMinPart >> unit)), 1u);

  // The wide tiles' ranges: of lengths that make from a 16th of a round of the card to 4 of them, the one that ends soonest.
  // Every round lasts as long as a range, and what an item costs beside its keys, more so where it leaves a partial. No step
  // ends before all its work is done, the narrow tiles' (a key of which takes about 4/5 of the time) among it; where that is the
  // larger part, ranges may last as long, at two thirds of the time that they take beside their like: behind a shared
  // prompt of 4096 keys and 256 requests' own of 1 to 512, ranges of 512 keys 119 us, of 1024 113, of 2048 107.
  int32_t chunk = kMaxKeys;
  const int64_t all_wide = (int64_t)wide_work + (shared_wide ? (int64_t)shared_tiles * shared_len : 0);
  if (all_wide) {
    const int32_t most = max(longest, shared_wide ? shared_len : 0), listed = min(a.batch_size, 1024);
    const auto chunk_of = [&](int32_t x) {
      const double keys = __builtin_ceil((double)all_wide * 16 / ((double)a.residents * (x + 1)));
      return round_up((int32_t)(keys < kMinChunk ? kMinChunk : keys < kMaxKeys ? keys : kMaxKeys), kStep);
    };
    for (int32_t x = wave; x < 64; x += 16) {
      const int32_t keys = chunk_of(x);
      int32_t items = 0;
      for (int32_t i = lane; i < listed; i += 64) if (wide_tiles[i].x) items += wide_tiles[i].x * max(ceil_div(wide_tiles[i].y, keys), 1);
      for (int d = 32; d; d >>= 1) items += __shfl_xor(items, d);
      if (shared_wide) items += shared_tiles * ceil_div(shared_len, keys);
      const int64_t each = min(keys, most) + (keys < most ? kWidePartWork : kWideTileWork);
      const int64_t rounds = (int64_t)ceil_div(items, a.residents) * each, own = items * each, beside = all_narrow * 4 / 5;
      const int64_t cost = max(beside > own ? rounds * 2 / 3 : rounds, (own + beside) / a.residents);
      if (lane == 0) atomicMin(&best, (unsigned long long)cost << 8 | (unsigned)x);
    }
    __syncthreads();
    chunk = chunk_of((int32_t)(best & 255));
  }
  const int32_t shared_chunks = shared_rows && shared_wide ? ceil_div(shared_len, chunk) : 0, shared_items = shared_tiles * shared_chunks;
  if (tid == 0) {
    carry[0] = shared_wide ? 0 : shared_tiles * shared_work;
    carry[1] = shared_wide ? 0 : shared_tiles;
    carry[2] = carry[3] = shared_items;
    carry[4] = 0;
  }
  __syncthreads();

  // a narrow item, and whose it is
  const auto put = [&](int32_t tile, int32_t group, const Item& item) {
    const int32_t at = tile + group;
    if (at >= a.max_items[0] || group >= a.groups) return;
    a.l.items[0][at] = item;
    atomicMin(&first_item[group], at);
    atomicMax(&last_item[group], at);
  };
  // the first key of a narrow tile's c-th part: the share of its work before the cut, in whole blocks
  const auto cut_key = [&](uint32_t at, uint32_t work, const Cuts& p, int32_t c, int32_t begin, int32_t end) {
    if (c == 0) return begin;
    if (c == p.count) return end;
    const double before = (double)((uint64_t)(p.group + c) * share - at) * (end - begin) / work;
    return begin + clamp(((int32_t)before + kStep / 2) / kStep * kStep, 0, end - begin);
  };

  if (shared_rows) {
    const int32_t table = table_of(a, some_request).begin;
    const int32_t each = shared_wide ? round_up(ceil_div(shared_len, shared_chunks), kStep) : 0;
    for (int32_t i = tid; i < shared_tiles; i += 1024) {
      const int32_t row0 = i * shared_tile, rows = min(shared_tile, shared_rows - row0);
      if (shared_wide) {
        a.l.shared_parts[i] = {i, i, shared_tiles, ceil_div(shared_len, each)};
      } else {
        const Cuts p = cuts_of(a, i * shared_work, shared_work, share, sliver);
        a.l.shared_parts[i] = {2 * a.groups + i, 2 * p.group, 2, p.count};
        for (int32_t c = 0; c < p.count; ++c)
          put(i, p.group + c,
              {-1, row0, rows, table, cut_key(i * shared_work, shared_work, p, c, 0, shared_len),
               cut_key(i * shared_work, shared_work, p, c + 1, 0, shared_len), c ? 2 * (p.group + c) : 2 * a.groups + i, 0});
      }
    }
    for (int32_t i = tid; i < shared_items && i < a.max_items[1]; i += 1024) {
      const int32_t c = i / shared_tiles, row0 = (i - c * shared_tiles) * kWide, from = min(c * each, shared_len);
      a.l.items[1][i] = {-1, row0, min(kWide, shared_rows - row0), table, from, min(from + each, shared_len), i, 0};
    }
  }

  // A request's lists, by `lanes` lanes over its tiles, or over the parts where there are few tiles
  const auto lay_out = [&](const Tiles& r, int32_t lane, int32_t lanes) {
    const int32_t rows = r.n * a.group, limit = r.len - r.n + 1;
    const bool sh = r.shared_token0 >= 0;
    // keys that a tile's last row sees
    const auto end_of = [&](int32_t last_row) { return clamp(limit + last_row / a.group, r.begin, r.len); };
    if (r.wide) {
      const int32_t parts = r.chunks(chunk), each = round_up(max(ceil_div(r.len, parts), 1), kStep);
      for (int32_t i = lane; i < r.tiles * parts; i += lanes) {
        const int32_t c = i / r.tiles, row0 = (i - c * r.tiles) * kWide, last_row = min(row0 + kWide, rows) - 1;
        const int32_t end = end_of(last_row), from = min(c * each, end), to = min(from + each, end);
        // (a range that a tile sees nothing of is an item without rows)
        if (r.first + i < a.max_items[1])
          a.l.items[1][r.first + i] = {r.q_begin, row0, c && from == to ? 0 : last_row + 1 - row0, r.table, from, to,
                                       end > each ? r.first_slot + i : -1, limit};
      }
      if (parts > 1)
        for (int32_t i = lane; i < r.tiles; i += lanes) {
          const int32_t row0 = i * kWide, count = ceil_div(end_of(min(row0 + kWide, rows) - 1), each);
          if (count < 2) continue;
          const int32_t lines = joined_rows(count), tile_rows = min(kWide, rows - row0);
          int32_t to = a.max_entries - 1 - atomicAdd(&entries[1], ceil_div(tile_rows, lines));
          for (int32_t e = 0; e < tile_rows && to >= 0; e += lines)
            a.l.entries[to--] = {r.q_begin, row0 + e, (int16_t)min(lines, tile_rows - e), lines == 1, -1,
                                 {r.first_slot + i, r.first_slot + i, r.tiles, count}};
        }
      return;
    }
    const bool by_parts = r.tiles < 8;
    for (int32_t i = by_parts ? 0 : lane; i < r.tiles; i += by_parts ? 1 : lanes) {
      const uint32_t before = (uint32_t)(r.before(i, a.group) >> unit), at = r.at + before;
      const uint32_t tile_work = (uint32_t)(r.before(i + 1, a.group) >> unit) - before;
      const Cuts p = cuts_of(a, at, tile_work, share, sliver);
      const int32_t row0 = i * kTile, last_row = min(row0 + kTile, rows) - 1, end = end_of(last_row);
      const int32_t slot = sh ? 2 * a.groups + r.first + i : p.count > 1 ? 2 * p.group + 1 : -1;
      for (int32_t c = by_parts ? lane : 0; c < p.count; c += by_parts ? lanes : 1)
        put(r.first + i, p.group + c,
            {r.q_begin, row0, last_row + 1 - row0, r.table, cut_key(at, tile_work, p, c, r.begin, end),
             cut_key(at, tile_work, p, c + 1, r.begin, end), c ? 2 * (p.group + c) : slot, limit});
      if (slot >= 0 && (!by_parts || lane == 0)) {
        int32_t parts = p.count;
        if (sh && shared_wide) parts += shared_chunks;
        else if (sh) parts += cuts_of(a, (r.shared_token0 * a.group + row0) / kTile * shared_work, shared_work, share, sliver).count;
        const int32_t lines = joined_rows(parts), tile_rows = last_row + 1 - row0;
        int32_t to = atomicAdd(&entries[0], ceil_div(tile_rows, lines));
        for (int32_t e = 0; e < tile_rows && to < a.max_entries; e += lines)
          a.l.entries[to++] = {r.q_begin, row0 + e, (int16_t)min(lines, tile_rows - e), lines == 1,
                               sh ? r.shared_token0 * a.group + row0 + e : -1, {slot, 2 * p.group, 2, p.count}};
      }
    }
    if (sh)
      for (int32_t i = lane; i < r.n; i += lanes) a.l.shared_tokens[r.shared_token0 + i] = make_int2(r.q_begin + i, limit + i);
  };

  for (int32_t b0 = 0; b0 < a.batch_size; b0 += 1024) {
    Tiles t = mine;
    if (b0) {
      t = {};
      t.shared_token0 = -1;
      if (b0 + tid < a.batch_size) t = tiles_of(a, b0 + tid);
    }
    const int32_t chunks = t.wide ? t.chunks(chunk) : 0;
    const int32_t sums[SUMS] = {t.tiles && !t.wide ? (int32_t)(t.before(t.tiles, a.group) >> unit) : 0, t.wide ? 0 : t.tiles,
                                t.tiles * chunks, chunks > 1 ? t.tiles * chunks : 0, t.shared_token0 >= 0 ? t.n : 0};
    int32_t sums_to[SUMS];  // inclusive
#pragma unroll
    for (int i = 0; i < SUMS; ++i) {
      sums_to[i] = sums[i];
      for (int d = 1; d < 64; d <<= 1) {
        const int32_t x = __shfl_up(sums_to[i], d);
        if (lane >= d) sums_to[i] += x;
      }
      if (lane == 63) wave_sums[wave][i] = sums_to[i];
    }
    if (tid == 0) num_long = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SUMS; ++i) {
      sums_to[i] += carry[i];
      for (int w = 0; w < wave; ++w) sums_to[i] += wave_sums[w][i];
    }
    t.at = sums_to[0] - sums[0];
    t.first = t.wide ? sums_to[2] - sums[2] : sums_to[1] - sums[1];
    t.first_slot = sums_to[3] - sums[3];
    if (t.shared_token0 >= 0) t.shared_token0 = sums_to[4] - sums[4];
    if (t.tiles) {
      if (!t.wide && t.tiles == 1 && cuts_of(a, t.at, sums[0], share, sliver).count <= kFew) lay_out(t, 0, 1);
      else long_requests[atomicAdd(&num_long, 1)] = t;
    }
    __syncthreads();
    if (tid == 1023)
      for (int i = 0; i < SUMS; ++i) carry[i] = sums_to[i];
    for (int32_t x = wave; x < num_long; x += 16) lay_out(long_requests[x], lane, 64);
    __syncthreads();
  }
  if (tid == 0)
    *a.l.header = {min(carry[2], a.max_items[1]), min(entries[0], a.max_entries), min(entries[1], a.max_entries), shared_wide};
  for (int32_t w = tid; w < a.groups; w += 1024)
    a.l.ranges[w] = last_item[w] < 0 ? Range{0, 0} : Range{first_item[w], last_item[w] + 1};
}

// ---- storage types -------------------------------------------------------------------------------------------------
struct BF16 {
  typedef __bf16 V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b2));
  }
  static __device__ __forceinline__ float wide(uint32_t half) { return __uint_as_float(half << 16); }
  static constexpr uint32_t kExponent = 0x7f80u;
  static constexpr float kScaledUp = 0;
};
struct F16 {
  typedef _Float16 V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ float wide(uint32_t half) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)half);
  }
  static constexpr uint32_t kExponent = 0x7c00u;
  // log2 of what weights are scaled up by, so that small ones, of which there may be many, are numbers of the type: a weight of 1 is
  // then 2^14 in a narrow tile, and one of kOutgrown, 2^8, is 2^15 in a wide tile. Both keep a step of the type below its largest.
  static constexpr float kScaledUp = 14;
};
// Is an infinity or NaN among the 16-bit values that were taken in? (The largest exponent of either half.)
template <typename T>
struct Oddities {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 top = {};
  __device__ __forceinline__ void take(u32x4 v) {
#pragma unroll
    for (int w = 0; w < 4; ++w)
      top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[w] & (T::kExponent << 16 | T::kExponent)));
  }
  __device__ __forceinline__ bool any() const { return max((uint32_t)top[0], (uint32_t)top[1]) == T::kExponent; }
};
// The infinities and NaN among 4 values, 0 for the others
template <typename T>
__device__ __forceinline__ f32x4 infinite_part(u32x2 four) {
  f32x4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t one = four[e / 2] >> (e % 2 * 16) & 0xffffu;
    x[e] = (one & T::kExponent) == T::kExponent ? T::wide(one) : 0.f;
  }
  return x;
}
template <typename T>
__device__ __forceinline__ u32x4 finite_part(u32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = ((v[i] & T::kExponent) == T::kExponent ? 0 : v[i] & 0xffffu) | ((v[i] >> 16 & T::kExponent) == T::kExponent ? 0 : v[i] & 0xffff0000u);
  return v;
}

struct AttendArgs {
  const char* query;
  const char* cache;
  const int32_t* kv_indices;
  char* out;
  float* lse;              // may be null
  float* partial[2];       // narrow, wide: [slots][kv heads][rows of a tile][head_dim]
  float* partial_lse[2];   // [slots][kv heads][rows of a tile], to base 2
  int64_t q_stride;        // bytes
  uint32_t page_stride, row_stride, plane;  // bytes: page to page, key to key in a page, K to V
  int32_t num_pages, page_size, page_shift;
  int32_t kv_heads, group, head_dim;
  int32_t narrow_groups, wide_groups;  // workgroups, of all key heads
  int32_t max_entries;
  float scale;             // times log2(e)
  Layout l;
};

// Byte offset of a key's row, or -1 where there is none to read: beyond `end`, or on a page that the cache does not have
__device__ __forceinline__ int64_t key_offset(const AttendArgs& a, int32_t table, int32_t key, int32_t end) {
  if (key >= end) return -1;
  const int32_t p = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
  const int32_t page = a.kv_indices[table + p];
  if (page < 0 || page >= a.num_pages) return -1;
  return (int64_t)page * a.page_stride + (int64_t)(key - p * a.page_size) * a.row_stride;
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

// How an item's keys are reached
enum Reach : int {
  kAnyPage,   // pages of any size: a lane looks up every key it loads
  kGroups,    // pages of whole groups of 16 keys: one scalar address a group
  kGroupsFull // and heads that fill the kernel's columns: no lane without a load
};

// The page ids of a wavefront's next 64 groups of 16 keys, one to a lane: looked up once in 32 blocks
struct GroupIds {
  int32_t page, off;  // -1: beyond the item's keys, or a page that the cache does not have
  __device__ __forceinline__ void fetch(const AttendArgs& a, const Item& item, int32_t k0, int32_t lane) {
    const int32_t key = k0 + (lane >> 1) * (kWaves * kBlock) + (lane & 1) * 16;
    page = -1;
    off = 0;
    if (key < item.key_end) {
      const int32_t p = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
      const int32_t id = a.kv_indices[item.table + p];
      off = key - p * a.page_size;
      page = id >= 0 && id < a.num_pages ? id : -1;
    }
  }
};

template <bool NT>
__device__ __forceinline__ u32x4 ld16(const char* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  else return *reinterpret_cast<const u32x4*>(p);
}

// A block of 32 keys in registers, as loaded
template <int DP>
struct Block {
  static constexpr int KSTEPS = DP / 32;
  static constexpr int LPR = DP <= 32 ? 4 : DP <= 64 ? 8 : DP <= 128 ? 16 : 32;  // lanes to a row of V
  static constexpr int RPI = 64 / LPR, VLOADS = kBlock / RPI;
  u32x4 k[2][KSTEPS], v[VLOADS];
  const char* rows[2];  // of the two groups of 16 keys, the same in all lanes

  // Where the (it mod 32)-th block of those that `ids` were fetched for lies; which of its keys are there. Every address is
  // inside a page of the cache; what is not the item's is cleared when it is used.
  __device__ __forceinline__ uint32_t find(const AttendArgs& a, const Item& item, const char* heads, int32_t k0, int32_t it, const GroupIds& ids) {
    uint32_t present = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int32_t page = __builtin_amdgcn_readlane(ids.page, (it & 31) * 2 + i);
      const int32_t off = __builtin_amdgcn_readlane(ids.off, (it & 31) * 2 + i);
      const int32_t left = item.key_end - k0 - i * 16;
      if (page >= 0) present |= (left >= 16 ? 0xffffu : (1u << left) - 1u) << (i * 16);
      rows[i] = heads + (int64_t)max(page, 0) * a.page_stride + (int64_t)off * a.row_stride;
    }
    return present;
  }
  template <Reach REACH, bool NT>
  __device__ __forceinline__ void load_k(const AttendArgs& a, const Item& item, const char* heads, int32_t k0, int32_t lane, uint32_t& present) {
    const int32_t n = lane & 15, quad = lane >> 4, D = a.head_dim;
    if constexpr (REACH == kAnyPage) present = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      bool have = true;
      const char* row;
      if constexpr (REACH == kAnyPage) {
        const int64_t off = key_offset(a, item.table, k0 + i * 16 + n, item.key_end);
        have = off >= 0;
        present |= ((uint32_t)__ballot(have) & 0xffffu) << (i * 16);
        row = heads + off + quad * 16;
      } else {
        row = rows[i] + (n * a.row_stride + quad * 16);
      }
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) {
        if (REACH != kGroupsFull) k[i][s] = u32x4{};
        if (REACH == kGroupsFull || (have && s * 32 + quad * 8 < D)) k[i][s] = ld16<NT>(row + s * 64);
      }
    }
  }
  template <Reach REACH, bool NT>
  __device__ __forceinline__ void load_v(const AttendArgs& a, const Item& item, const char* heads, int32_t k0, int32_t lane) {
    const int32_t vrow = lane / LPR, vcol = lane % LPR, D = a.head_dim;
    const uint32_t at = a.plane + vrow * a.row_stride + vcol * 16;
#pragma unroll
    for (int i = 0; i < VLOADS; ++i) {
      bool have = true;
      const char* row;
      if constexpr (REACH == kAnyPage) {
        const int64_t off = key_offset(a, item.table, k0 + i * RPI + vrow, item.key_end);
        have = off >= 0;
        row = heads + a.plane + off + vcol * 16;
      } else {
        constexpr int HALF = VLOADS / 2;
        row = rows[i / HALF] + (int64_t)(i % HALF * RPI) * a.row_stride + at;
      }
      if (REACH != kGroupsFull) v[i] = u32x4{};
      if (REACH == kGroupsFull || (have && vcol * 8 < D)) v[i] = ld16<NT>(row);
    }
  }
};

// A workgroup per (item, key head); its wavefronts take blocks of 32 keys in turn, each with a maximum and a sum of its
// own, joined at the end through LDS.
//   S^T = K Q^T: the keys' rows are the matrix instruction's A operand as they lie in memory, 16 bytes a lane.
//   O^T = V^T P^T: a lane's 8 probabilities, of keys 4q..4q+3 and 16+4q..16+4q+3 (q = lane / 16), are the B operand as S^T
//   left them; the A operand wants the same keys of one column of V, which the transposing LDS read gives.
// The matrix instruction takes 16 bits: a weight goes in as two numbers of the storage type, itself rounded and the rest
// rounded, off by a half step's square. The second product is on a unit that waits for keys: decode of 256 requests 405.4 us with
// one product and 405.7 with both, one request 17.5 and 17.9, the error against 64 bits 2.02e-3 and 1.65e-3 of the outputs' size,
// which is their own rounding. (f16: from 2^-28 of the largest weight on; smaller ones are off by at most 2^-39 of it.)
template <typename T, int DP>
struct RowTile {
  static constexpr int KSTEPS = DP / 32, DTILES = DP / 16;
  static constexpr int VSTRIDE = DP * 2 + 32;  // rows 32 bytes apart in the banks: a transposing read takes 4 of them
  typedef Block<DP> B;
  u32x4 q[KSTEPS];
  f32x4 o[DTILES];
  float base, l;  // weights are exp2(score * scale - base)
  int32_t limit;
  int32_t odd_from;  // the first block whose infinities and NaN of V were left out

  // One block; `next` asks for the block after it, a half at a time, as soon as the registers are free
  template <Reach REACH, typename Next>
  __device__ __forceinline__ void take(const AttendArgs& a, const Item& item, B& b, uint32_t present, int32_t k0, char* my_v, int32_t lane,
                                       const Next& next) {
    const int32_t n = lane & 15, quad = lane >> 4, vrow = lane / B::LPR, vcol = lane % B::LPR;
    f32x4 s[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) s[i] = T::mfma(b.k[i][k], q[k], s[i]);
    next(0);
    const bool whole = present == 0xffffffffu;
    if (REACH != kAnyPage && !whole)
#pragma unroll
      for (int i = 0; i < B::VLOADS; ++i)
        if (!(present >> (i * B::RPI + vrow) & 1)) b.v[i] = u32x4{};
    // does a row stop inside the block, and is there a value in it that 0 does not cancel?
    const bool ragged = __ballot(n < item.rows && limit < min(k0 + kBlock, item.key_end)) != 0;
    if (ragged) {
      Oddities<T> odd;
#pragma unroll
      for (int i = 0; i < B::VLOADS; ++i) odd.take(b.v[i]);
      if (__ballot(odd.any())) {
        odd_from = min(odd_from, k0);
#pragma unroll
        for (int i = 0; i < B::VLOADS; ++i) b.v[i] = finite_part<T>(b.v[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < B::VLOADS; ++i)
      if (B::LPR * 8 == DP || vcol * 8 < DP) *reinterpret_cast<u32x4*>(my_v + (i * B::RPI + vrow) * VSTRIDE + vcol * 16) = b.v[i];
    next(1);
    if (ragged || !whole) {
      // the keys that the row sees, bit x for key x + 4 quad, so that a lane's are at fixed bits
      const int32_t left = clamp(limit - k0, 0, kBlock);
      const uint32_t sees = (left ? 0xffffffffu >> (kBlock - left) & present : 0) >> quad * 4;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!(sees >> (i * 16 + r) & 1)) s[i][r] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][r]);
    top = max_across32(max_across16(top));
    const float grown = fmaxf(base, top * a.scale - T::kScaledUp);
    const float from = grown == -INFINITY ? 0.f : grown;
    const float shrink = exp2_of(base - from);  // 0 from -inf
    u32x4 p, rest;
    float sum = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float x = exp2_of(__builtin_fmaf(s[i][r], a.scale, -from));
        const float y = exp2_of(__builtin_fmaf(s[i][r + 1], a.scale, -from));
        const uint32_t two = T::pack(x, y);
        p[i * 2 + r / 2] = two;
        rest[i * 2 + r / 2] = T::pack(x - T::wide(two & 0xffffu), y - T::wide(two >> 16));
        sum += x + y;
      }
    l = l * shrink + sum;
    base = grown;
    u32x4 last = {};
#pragma unroll
    for (int d = 0; d < DTILES; ++d) {
      const char* from = my_v + (quad * 4 + n / 4) * VSTRIDE + (d * 16 + n % 4 * 4) * 2;
      typedef __attribute__((address_space(3))) s16x4* Lds;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(from));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(from + 16 * VSTRIDE));
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
      const u32x4 v = {x[0], x[1], y[0], y[1]};
      o[d] = T::mfma(v, p, o[d] * shrink);
      if (d) o[d - 1] = T::mfma(last, rest, o[d - 1]);
      last = v;
    }
    o[DTILES - 1] = T::mfma(last, rest, o[DTILES - 1]);
  }
};

template <typename T, int DP>
constexpr int narrow_lds() { return kWaves * kBlock * RowTile<T, DP>::VSTRIDE + kWaves * 2 * kTile * 4; }

template <typename T, int DP, Reach REACH, bool NT>
__device__ __forceinline__ void narrow_item(const AttendArgs& a, const Item& item, int32_t h, char* lds) {
  typedef RowTile<T, DP> Tile;
  typedef Block<DP> B;
  constexpr int KSTEPS = Tile::KSTEPS, DTILES = Tile::DTILES, VSTRIDE = Tile::VSTRIDE;
  constexpr int OSTRIDE = DP + 4;
  constexpr float kUnscaled = 1.f / (1 << (int)T::kScaledUp);
  static_assert(kTile * OSTRIDE * 4 <= kBlock * VSTRIDE, "a wavefront's O takes the place of its V");
  typedef float Stats[2][kTile];
  Stats* const stats = reinterpret_cast<Stats*>(lds + kWaves * kBlock * VSTRIDE);
  const int32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t n = lane & 15, quad = lane >> 4;
  const int32_t D = a.head_dim;
  {
    Tile tile = {};
    tile.base = -INFINITY;
    tile.odd_from = INT32_MAX;
    if (n < item.rows) {
      const int32_t row = item.row0 + n, i = row / a.group, g = row - i * a.group;
      const int2 x = item.q_begin >= 0 ? make_int2(item.q_begin + i, item.limit + i) : a.l.shared_tokens[i];
      const int32_t token = x.x;
      tile.limit = clamp(x.y, 0, item.key_end);
      const char* p = a.query + (int64_t)token * a.q_stride + ((int64_t)(h * a.group + g) * D + quad * 8) * 2;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
        if (k * 32 + quad * 8 < D) tile.q[k] = *reinterpret_cast<const u32x4*>(p + k * 64);
    }
    const char* heads = a.cache + (int64_t)h * D * 2;
    char* const my_v = lds + wave * (kBlock * VSTRIDE);
    constexpr int32_t STEP = kWaves * kBlock;
    int32_t k0 = item.key_begin + wave * kBlock;
    if (k0 < item.key_end && a.num_pages > 0) {
      GroupIds ids;
      B block;
      uint32_t present = 0;
      if constexpr (REACH != kAnyPage) {
        ids.fetch(a, item, k0, lane);
        present = block.find(a, item, heads, k0, 0, ids);
      }
      block.template load_k<REACH, NT>(a, item, heads, k0, lane, present);
      block.template load_v<REACH, NT>(a, item, heads, k0, lane);
      for (int32_t i = 1;; ++i, k0 += STEP) {
        const bool more = k0 + STEP < item.key_end;
        uint32_t coming = 0;
        if (REACH != kAnyPage && more && (i & 31) == 0) ids.fetch(a, item, k0 + STEP, lane);
        tile.template take<REACH>(a, item, block, present, k0, my_v, lane, [&](int half) {
          if (!more) return;
          if (half == 0) {
            if constexpr (REACH != kAnyPage) coming = block.find(a, item, heads, k0 + STEP, i, ids);
            block.template load_k<REACH, NT>(a, item, heads, k0 + STEP, lane, coming);
          } else {
            block.template load_v<REACH, NT>(a, item, heads, k0 + STEP, lane);
          }
        });
        if (!more) break;
        present = coming;
      }
    }
    // the sum over the four quads' keys
    float l = tile.l;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    // Infinities and NaN of V: those that were left out, where rows stop, and where a product with one of them is in O (that may
    // be NaN, from a weight's second part or a weight of 0), go to the rows that see their keys with a weight of 1: what it scales
    // is infinite. (The opaque zero keeps the compiler from working on this ahead.)
    f32x4 probe = {};
#pragma unroll
    for (int d = 0; d < DTILES; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) probe[e] = __builtin_fmaf(tile.o[d][e], 0.f, probe[e]);
    const bool mine = !finite((probe[0] + probe[1]) + (probe[2] + probe[3])) && finite(l);
    const bool some = __ballot(mine) != 0;
    if (__builtin_expect(some || tile.odd_from < item.key_end, 0)) {
      int32_t zero = 0;
      asm volatile("" : "+v"(zero));
      uint32_t odd[(DTILES + 7) / 8] = {};
      if (mine)
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!finite(tile.o[d][e])) {
              odd[d / 8] |= 1u << (d % 8 * 4 + e);
              tile.o[d][e] = 0;
            }
      for (int32_t b0 = some ? item.key_begin + wave * kBlock : tile.odd_from; b0 < item.key_end; b0 += STEP)
#pragma unroll 1
        for (int32_t key = b0; key < min(b0 + kBlock, item.key_end); ++key) {
          const int64_t off = key_offset(a, item.table, key, item.key_end);
          if (off < 0 || key >= tile.limit) continue;
          const char* row = heads + a.plane + off + quad * 8 + zero;
#pragma unroll
          for (int d = 0; d < DTILES; ++d)
            if (d * 16 + quad * 4 < D) tile.o[d] += infinite_part<T>(*reinterpret_cast<const u32x2*>(row + d * 32));
        }
#pragma unroll
      for (int d = 0; d < DTILES; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((odd[d / 8] >> (d % 8 * 4 + e) & 1) && tile.o[d][e] == 0) tile.o[d][e] = NAN;  // (no value was: a sum left fp32)
          if (l == 0) tile.o[d][e] = 0;
        }
    }
    // over the wavefronts
    if (quad == 0) {
      stats[wave][0][n] = tile.base;
      stats[wave][1][n] = l;
    }
    __syncthreads();
    float top = -INFINITY, all_l = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][0][n]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all_l += stats[w][1][n] * exp2_of(stats[w][0][n] - base);
    const float weight = exp2_of(tile.base - base) * (all_l == 0 ? 0.f : 1.f / all_l);
    const float part = weight < kLeastWeight ? kLeastWeight : weight;  // (NaN stays)
    float* my_o = reinterpret_cast<float*>(my_v);
#pragma unroll
    for (int d = 0; d < DTILES; ++d)
      *reinterpret_cast<f32x4*>(my_o + n * OSTRIDE + d * 16 + quad * 4) = tile.o[d] * part;
    if (wave == 0 && quad == 0 && n < item.rows) {
      const float lse2 = all_l == 0 ? -INFINITY : base + T::kScaledUp + __log2f(all_l * kUnscaled);
      if (item.slot >= 0) {
        a.partial_lse[0][((int64_t)item.slot * a.kv_heads + h) * kTile + n] = lse2;
      } else if (a.lse) {
        const int32_t row = item.row0 + n, i = row / a.group, g = row - i * a.group;
        a.lse[(int64_t)(item.q_begin + i) * a.kv_heads * a.group + h * a.group + g] = lse2 * kLn2;
      }
    }
    __syncthreads();
    for (int32_t e = tid; e < kTile * (DP / 4); e += kThreads) {
      const int32_t r = e / (DP / 4), d = e % (DP / 4) * 4;
      if (r >= item.rows || d >= D) continue;
      f32x4 x = {};
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        x += *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(lds + w * (kBlock * VSTRIDE)) + r * OSTRIDE + d);
      if (item.slot >= 0) {
        *reinterpret_cast<f32x4*>(a.partial[0] + (((int64_t)item.slot * a.kv_heads + h) * kTile + r) * D + d) = x;
      } else {
        const int32_t row = item.row0 + r, i = row / a.group, g = row - i * a.group;
        const u32x2 two = {T::pack(x[0], x[1]), T::pack(x[2], x[3])};
        *reinterpret_cast<u32x2*>(a.out + (((int64_t)(item.q_begin + i) * a.kv_heads + h) * a.group + g) * D * 2 + d * 2) = two;
      }
    }
    __syncthreads();
  }
}

// A workgroup per (item of up to 128 rows, key head): 32 rows to a wavefront, 64 keys at a time, staged in LDS for all four.
// The next step's loads are under way in registers while one is worked on; the buffers alternate, and K runs half a step
// ahead of V, as their products do, so that a step has one barrier. S^T and O^T as above, in 32 x 32 pieces: a lane holds one
// row and, of 32 keys, those with bit 2 as its own half (lane / 32). K rows are 16 bytes apart in the banks (a lane reads 16
// bytes of a row of its own), V rows 64.
// The maximum that the weights are taken against grows only when a row's has outgrown it by 2^8: until then the larger weights
// (below 2^8) and sums say the same, and the rescaling of O, 64 registers at 128 columns, is left out of nearly every step.
// Bound by the instructions that two wavefronts a SIMD can have under way: the matrix unit is busy for 41 % of the cycles
// (2048 new tokens behind 13 to 30 thousand keys, 7 query heads to a key head of 128: 780 us at least and 825 in the median of 30
// launches, 860 to 910 TFLOP/s).
template <int DP>
constexpr int wide_lds() { return 2 * kStep * (DP * 2 + 16 + DP * 2 + kVPad) + (kWaves + 1) * 4; }

template <typename T, int DP, Reach REACH>
__device__ __forceinline__ void wide_item(const AttendArgs& a, const Item& item, int32_t h, char* lds) {
  constexpr int KSTEPS = DP / 16, DTILES = DP / 32;
  constexpr int KSTRIDE = DP * 2 + 16, VSTRIDE = DP * 2 + kVPad;
  constexpr int LPR = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;  // lanes to a row
  constexpr int RPW = 64 / LPR, ROUNDS = kStep / (RPW * kWaves);
  constexpr float kScaledUp = T::kScaledUp / 2, kOutgrown = 8 + kScaledUp, kUnscaled = 1.f / (1 << (int)kScaledUp);
  typedef char KStep[kStep * KSTRIDE];
  typedef char VStep[kStep * VSTRIDE];
  KStep* const k_lds = reinterpret_cast<KStep*>(lds);
  VStep* const v_lds = reinterpret_cast<VStep*>(lds + 2 * sizeof(KStep));
  int32_t* const leasts = reinterpret_cast<int32_t*>(lds + 2 * sizeof(KStep) + 2 * sizeof(VStep));
  int32_t& left_out = leasts[kWaves];
  const int32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t n = lane & 31, hi = lane >> 5, lrow = lane / LPR, lcol = lane % LPR;
  const int32_t D = a.head_dim;
  {
    const char* const heads = a.cache + (int64_t)h * D * 2;
    const int32_t my_row = wave * 32 + n;
    u32x4 q[KSTEPS] = {};
    int32_t limit = 0, token = 0, g = 0;
    if (my_row < item.rows) {
      const int32_t row = item.row0 + my_row, i = row / a.group;
      g = row - i * a.group;
      const int2 x = item.q_begin >= 0 ? make_int2(item.q_begin + i, item.limit + i) : a.l.shared_tokens[i];
      token = x.x;
      limit = clamp(x.y, 0, item.key_end);
      const char* p = a.query + (int64_t)token * a.q_stride + ((int64_t)(h * a.group + g) * D + hi * 8) * 2;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
        if (REACH == kGroupsFull || k * 16 + hi * 8 < D) q[k] = *reinterpret_cast<const u32x4*>(p + k * 32);
    }
    // the wavefront's first limit (rows that are not there have none)
    int32_t least = my_row < item.rows ? limit : INT32_MAX;
    for (int d = 16; d; d >>= 1) least = min(least, __shfl_xor(least, d));
    least = __builtin_amdgcn_readfirstlane(least);
    if (lane == 0) leasts[wave] = least;
    if (tid == 0) left_out = 0;
    __syncthreads();
    const int32_t tile_least = min(min(leasts[0], leasts[1]), min(leasts[2], leasts[3]));
    f32x16 o[DTILES] = {};
    float base = -INFINITY, l = 0;  // as in a narrow tile
    u32x4 kr[ROUNDS], vr[ROUNDS];
    uint32_t group_lo = 0, group_hi = 0;  // where the groups of 16 keys of 16 windows lie, one to a lane
    uint64_t groups = 0;                  // and which of them are there
    // Keys come in windows of 64: window w begins 32 before the item's 64 w-th key, so that what a step reads, K of the 64
    // keys from its own 32nd on and V of the 64 keys up to its own 32nd, are the windows w + 1 and w.
    const auto window = [&](int32_t w) { return item.key_begin + w * kStep - kStep / 2; };
    const auto offset_of = [&](int32_t key) { return key < item.key_begin ? -1 : key_offset(a, item.table, key, item.key_end); };
    int64_t place[ROUNDS];  // of the rows of the window that K was last asked of, by round (the same in all lanes)
    // where a round's rows lie (one row of every LPR lanes), or null where there is none to read
    const auto row_of = [&](int32_t w, int i) -> const char* {
      if constexpr (REACH == kAnyPage) {
        const int64_t off = offset_of(window(w) + i * RPW * kWaves + wave * RPW + lrow);
        return off < 0 || lcol * 8 >= D ? nullptr : heads + off + lcol * 16;
      } else {
        if (REACH == kGroups && lcol * 8 >= D) return nullptr;
        return heads + place[i] + (lrow * a.row_stride + lcol * 16);
      }
    };
    // K of a window, on its way; which of the keys are there
    const auto fetch_k = [&](int32_t w) -> uint64_t {
      uint64_t present = 0;
      const int32_t first = window(w);
      if constexpr (REACH == kAnyPage) {
        present = __ballot(offset_of(first + lane) >= 0);
      } else {
        if ((w & 15) == 0) {
          const int32_t key = first + lane * 16;
          uint64_t at = 0;  // (of what is not there: the cache's first page)
          bool have = false;
          if (key >= item.key_begin && key < item.key_end) {
            const int32_t p = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
            const int32_t id = a.kv_indices[item.table + p];
            have = id >= 0 && id < a.num_pages;
            if (have) at = (uint64_t)(uint32_t)id * a.page_stride + (uint64_t)(uint32_t)(key - p * a.page_size) * a.row_stride;
          }
          group_lo = (uint32_t)at;
          group_hi = (uint32_t)(at >> 32);
          groups = __ballot(have);
        }
        const uint32_t four = (uint32_t)(groups >> (w & 15) * 4) & 15, left = (uint32_t)(item.key_end - first);
        present = ~(uint64_t)0;
        if (four != 15 || left < kStep) {
          present = 0;
          for (int i = 0; i < 4; ++i) present |= (uint64_t)(four >> i & 1 ? 0xffffu : 0) << (i * 16);
          if (left < kStep) present &= ((uint64_t)1 << left) - 1;
        }
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
          const int32_t row0 = i * RPW * kWaves + wave * RPW, group = (w & 15) * 4 + row0 / 16;
          place[i] = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(group_hi, group) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane(group_lo, group)) + (uint32_t)(row0 % 16) * a.row_stride;
        }
      }
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        const char* from = row_of(w, i);
        if (REACH != kGroupsFull) kr[i] = u32x4{};
        if (REACH == kGroupsFull || from) kr[i] = *reinterpret_cast<const u32x4*>(from);
      }
      return present;
    };
    // V of the window that K was last asked of
    const auto fetch_v = [&](int32_t w) {
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        const char* from = row_of(w, i);
        if (REACH != kGroupsFull) vr[i] = u32x4{};
        if (REACH == kGroupsFull || from) vr[i] = *reinterpret_cast<const u32x4*>(from + a.plane);
      }
    };
    // The columns beyond head_dim are zeros, and V of keys that are not there is cleared, which K's need not be: their scores
    // are masked.
    const auto stage_k = [&](int buf) {
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i)
        if (LPR * 8 == DP || lcol * 8 < DP)
          *reinterpret_cast<u32x4*>(k_lds[buf] + (i * RPW * kWaves + wave * RPW + lrow) * KSTRIDE + lcol * 16) = kr[i];
    };
    const auto stage_v = [&](int buf, int32_t w, uint64_t present) {
      if (REACH != kAnyPage && ~present)
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i)
          if (!(present >> (i * RPW * kWaves + wave * RPW + lrow) & 1)) vr[i] = u32x4{};
      if (window(w) + kStep > tile_least) {  // a row stops in it: are there values that 0 does not cancel?
        Oddities<T> odd;
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) odd.take(vr[i]);
        if (__ballot(odd.any())) {
          left_out = 1;
#pragma unroll
          for (int i = 0; i < ROUNDS; ++i) vr[i] = finite_part<T>(vr[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i)
        if (LPR * 8 == DP || lcol * 8 < DP)
          *reinterpret_cast<u32x4*>(v_lds[buf] + (i * RPW * kWaves + wave * RPW + lrow) * VSTRIDE + lcol * 16) = vr[i];
    };

    // Pieces from LDS: 16 columns of K of 32 keys (a half of a step), 32 columns of V of 16 of them, of which the lane's are
    // 4 hi..4 hi + 3 and 8 + 4 hi..8 + 4 hi + 3.
    const auto k_piece = [&](int buf, int half, int j) {
      return *reinterpret_cast<const u32x4*>(k_lds[buf] + (half * 32 + n) * KSTRIDE + hi * 16 + j * 32);
    };
    const auto v_piece = [&](int buf, int half, int j) {
      typedef __attribute__((address_space(3))) s16x4* Lds;
      const char* from = v_lds[buf] + (half * 32 + hi * 4 + (n & 15) / 4) * VSTRIDE + ((n >> 4) * 16 + n % 4 * 4) * 2 +
                         j / DTILES * 16 * VSTRIDE + j % DTILES * 64;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(from));
      const s16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(from + 8 * VSTRIDE));
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, up);
      return u32x4{x[0], x[1], y[0], y[1]};
    };
    // the row's highest score of 32 keys, those of keys that it does not see taken out
    const auto highest = [&](f32x16& s) {
      float top = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
      return top;
    };
    const auto mask = [&](f32x16& s, float top, int32_t k0, uint32_t present) {
      if (least < k0 + 32 || ~present) {
        // the keys that the row sees, bit x for key x + 4 hi, so that a lane's are at fixed bits
        const int32_t left = clamp(limit - k0, 0, 32);
        const uint32_t sees = (left ? 0xffffffffu >> (32 - left) & present : 0) >> hi * 4;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!(sees >> (r / 4 * 8 + r % 4) & 1)) s[r] = -INFINITY;
        top = highest(s);
      }
      return max_across32(top);
    };
    // A base that has been outgrown. It is a whole number, so that what was made with the old one, the weights that wait
    // for their product among it, is scaled exactly (in f16 those that stay above 2^-21 of a weight of 1, others to 2^-32 of it).
    const auto grow = [&](float top, uint32_t* waiting) {
      if (__ballot(top * a.scale > base + kOutgrown)) {
        const float grown = fmaxf(base, __builtin_ceilf(top * a.scale) - kScaledUp);
        const float shrink = exp2_of(base - (grown == -INFINITY ? 0.f : grown));  // 0 from -inf
#pragma unroll
        for (int d = 0; d < DTILES; ++d) o[d] *= shrink;
#pragma unroll
        for (int i = 0; i < 8; ++i) waiting[i] = T::pack(T::wide(waiting[i] & 0xffffu) * shrink, T::wide(waiting[i] >> 16) * shrink);
        l *= shrink;
        base = grown;
      }
    };
    // 32 keys: their weights from the scores s, while the scores of the keys behind them and the product of the weights
    // before them, that waited, with V are on the matrix unit. The order is written out, a product with what goes on beside
    // it to a line: pieces from LDS for the products kAhead further on, half a pair of weights, the next scores' maximum.
    // A weight is rounded to the storage type for its product, off by at most half a step of itself; their sum l is of the weights
    // before that. The rest as a second product, as in a narrow tile, would cost what the matrix unit is bound by: 2048 new
    // tokens 800 us so and 1043 with both, the error against 64 bits 2.33e-3 and 1.66e-3 of the outputs' size.
    const auto take = [&](const f32x16& s, uint32_t* p, f32x16& next, float& top, const uint32_t* waiting, int buf, auto which,
                          u32x4* piece) {
      constexpr int PIECES = KSTEPS + 2 * DTILES, HALF = decltype(which)::value;
      static_assert(PIECES % (kAhead + 1) == 0, "the second half's first pieces are asked for at the end of the first's");
      const float minus = base == -INFINITY ? 0.f : -base;
      float sum[2] = {}, weight[3] = {};
      next = f32x16{};
      // a weight is used behind the next one's exponential, whose result the adder would wait for
      const auto add = [&](int r) {
        sum[r % 2] += weight[r % 3];
        asm volatile("" : "+v"(sum[r % 2]));
        if (r % 2) {
          p[r / 2] = T::pack(weight[(r + 2) % 3], weight[r % 3]);
          asm volatile("" : "+v"(p[r / 2]));
        }
      };
      const auto ask = [&](int j) {
        if (j < PIECES) piece[j % (kAhead + 1)] = j < KSTEPS ? k_piece(buf, HALF, j) : v_piece(buf, HALF, j - KSTEPS);
        else if (HALF == 0) piece[j % (kAhead + 1)] = k_piece(buf, 1, j - PIECES);
      };
      if (HALF == 0)
#pragma unroll
        for (int j = 0; j < kAhead; ++j) ask(j);
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        ask(j + kAhead);
        if (j < KSTEPS) {
          next = T::mfma(piece[j % (kAhead + 1)], q[j], next);
        } else {
          const int v = j - KSTEPS;
          const uint32_t* w = waiting + v / DTILES * 4;
          o[v % DTILES] = T::mfma(piece[j % (kAhead + 1)], u32x4{w[0], w[1], w[2], w[3]}, o[v % DTILES]);
        }
#pragma unroll
        for (int r = j * 16 / PIECES; r < (j + 1) * 16 / PIECES; ++r) {
          float y = exp2_of(__builtin_fmaf(s[r], a.scale, minus));
          asm volatile("" : "+v"(y));  // here, and not where it is used
          weight[r % 3] = y;
          if (r) add(r - 1);
        }
        if (j == PIECES - 1) top = highest(next);
        __builtin_amdgcn_sched_barrier(0);
      }
      add(15);
      l += sum[0] + sum[1];
    };
    const int32_t steps = a.num_pages > 0 ? (item.key_end - item.key_begin + kStep - 1) / kStep : 0;
    if (steps > 0) {
      int32_t k0 = item.key_begin;
      // nothing waits for the first product: zeros, and V of the keys before the first is cleared
      uint32_t p0[8], p1[8] = {};
      uint64_t before = fetch_k(0);
      fetch_v(0);
      stage_k(1);
      stage_v(0, 0, before);
      uint64_t present = fetch_k(1), coming = 0, then = 0;  // of the windows i + 1, i + 2, i + 3
      fetch_v(1);
      stage_k(0);
      if (steps > 1) coming = fetch_k(2);
      __syncthreads();
      f32x16 s0 = {}, s1;
#pragma unroll
      for (int j = 0; j < KSTEPS; ++j) s0 = T::mfma(k_piece(1, 1, j), q[j], s0);
      float top = mask(s0, highest(s0), k0, (uint32_t)(before >> 32));
      for (int32_t i = 0; i < steps; ++i, k0 += kStep) {
        const int buf = i & 1;
        u32x4 piece[kAhead + 1];
        __syncthreads();  // this step's windows are there, the last step's have been read
        stage_v(buf ^ 1, i + 1, present);
        if (i + 1 < steps) {
          stage_k(buf ^ 1);
          fetch_v(i + 2);
          if (i + 2 < steps) then = fetch_k(i + 3);
        }
        // before the other workgroup's wavefronts that stage (2048 new tokens 817 us without, 796 so)
        __builtin_amdgcn_s_setprio(1);
        grow(top, p1);
        take(s0, p0, s1, top, p1, buf, std::integral_constant<int, 0>{}, piece);
        top = mask(s1, top, k0 + 32, (uint32_t)present);
        grow(top, p0);
        take(s1, p1, s0, top, p0, buf, std::integral_constant<int, 1>{}, piece);  // (after the last step: scores of keys that are not there)
        top = mask(s0, top, k0 + kStep, (uint32_t)(present >> 32));
        __builtin_amdgcn_s_setprio(0);
        present = coming;
        coming = then;
        then = 0;
      }
      __syncthreads();
      // the last weights' product
#pragma unroll
      for (int j = 0; j < 2 * DTILES; ++j) {
        const uint32_t* w = p1 + j / DTILES * 4;
        o[j % DTILES] = T::mfma(v_piece(steps & 1, 0, j), u32x4{w[0], w[1], w[2], w[3]}, o[j % DTILES]);
      }
    }
    __syncthreads();  // (left_out is complete, and the buffers are free)
    l += __shfl_xor(l, 32);
    f32x4 probe = {};
#pragma unroll
    for (int d = 0; d < DTILES; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) probe[r % 4] = __builtin_fmaf(o[d][r], 0.f, probe[r % 4]);
    const bool mine = !finite((probe[0] + probe[1]) + (probe[2] + probe[3])) && finite(l);
    const bool some = __ballot(mine) != 0;
    if (__builtin_expect(some || left_out, 0)) {  // as above
      int32_t zero = 0;
      asm volatile("" : "+v"(zero));
      uint32_t odd[(DTILES + 1) / 2] = {};
      if (mine)
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!finite(o[d][r])) {
              odd[d / 2] |= 1u << (d % 2 * 16 + r);
              o[d][r] = 0;
            }
      const int32_t from = some ? item.key_begin
                                : item.key_begin + max((max(tile_least - item.key_begin, 0) + kStep / 2) / kStep * kStep - kStep / 2, 0);
#pragma unroll 1
      for (int32_t key = from; key < item.key_end; ++key) {
        const int64_t off = key_offset(a, item.table, key, item.key_end);
        if (off < 0 || key >= limit) continue;
        const char* row = heads + a.plane + off + hi * 8 + zero;
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (d * 32 + i * 8 + hi * 4 < D) {
              const f32x4 x = infinite_part<T>(*reinterpret_cast<const u32x2*>(row + d * 64 + i * 16));
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][i * 4 + e] += x[e];
            }
      }
#pragma unroll
      for (int d = 0; d < DTILES; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if ((odd[d / 2] >> (d % 2 * 16 + r) & 1) && o[d][r] == 0) o[d][r] = NAN;
          if (l == 0) o[d][r] = 0;
        }
    }
    const float inv = l == 0 ? 0.f : 1.f / l, lse2 = l == 0 ? -INFINITY : base + kScaledUp + __log2f(l * kUnscaled);
    if (my_row < item.rows) {
      if (item.slot >= 0) {
        const int64_t row = ((int64_t)item.slot * a.kv_heads + h) * kWide + my_row;
        if (hi == 0) a.partial_lse[1][row] = lse2;
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int32_t c = d * 32 + i * 8 + hi * 4;
            if (REACH != kGroupsFull && c >= D) continue;
            *reinterpret_cast<f32x4*>(a.partial[1] + row * D + c) =
                f32x4{o[d][i * 4] * inv, o[d][i * 4 + 1] * inv, o[d][i * 4 + 2] * inv, o[d][i * 4 + 3] * inv};
          }
      } else {
        const int64_t row = ((int64_t)token * a.kv_heads + h) * a.group + g;
        if (a.lse && hi == 0) a.lse[row] = lse2 * kLn2;
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int32_t c = d * 32 + i * 8 + hi * 4;
            if (REACH != kGroupsFull && c >= D) continue;
            *reinterpret_cast<u32x2*>(a.out + (row * D + c) * 2) =
                u32x2{T::pack(o[d][i * 4] * inv, o[d][i * 4 + 1] * inv), T::pack(o[d][i * 4 + 2] * inv, o[d][i * 4 + 3] * inv)};
          }
      }
    }
    __syncthreads();  // before the next item
  }
}

// A workgroup of a key head takes its share's items one after the other
template <typename T, int DP, Reach REACH, bool NT>
__device__ __forceinline__ void narrow_share(const AttendArgs& a, int32_t at, char* lds) {
  const int32_t group = at / a.kv_heads, h = at - group * a.kv_heads;
  const Range range = a.l.ranges[group];
  for (int32_t i = range.begin; i < range.end; ++i) narrow_item<T, DP, REACH, NT>(a, a.l.items[0][i], h, lds);
}
// As many workgroups as are on the card at once, by their registers. NT: keys by non-temporal loads, see launch_attend.
constexpr int narrow_residents(int dp) { return dp <= 64 ? 4 : dp <= 128 ? 2 : 1; }  // of a CU
template <typename T, int DP, Reach REACH, bool NT = false>
__global__ __launch_bounds__(kThreads, narrow_residents(DP)) void attend_rows_kernel(AttendArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[narrow_lds<T, DP>()];
  narrow_share<T, DP, REACH, NT>(a, blockIdx.x, lds);
}

// Steps that may have wide tiles: both kinds in one launch, side by side on the card, as the narrow ones wait for memory and
// the wide ones for the matrix units. 32 workgroups of a kind in turn: they are dealt to the 8 XCDs and there to 4 shader
// engines in rotation (8 in turn put all wide ones on half of the engines: 2048 new tokens 1218 us, 917 so). The wide items, of one key head
// after the other, are dealt to the XCDs in eight runs, so that items that read the same keys share an L2.
template <typename T, int DP, Reach REACH>
__global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) void attend_step_kernel(AttendArgs a) {
  constexpr int LDS = wide_lds<DP>() > narrow_lds<T, DP>() ? wide_lds<DP>() : narrow_lds<T, DP>();
  __shared__ __attribute__((aligned(16))) char lds[LDS];
  const int32_t narrow = a.narrow_groups, both = min(narrow, a.wide_groups) & ~31;
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
    narrow_share<T, DP, REACH, false>(a, at, lds);
    return;
  }
  const int32_t items = a.l.header->wide_items, all = items * a.kv_heads, run = (all + 7) / 8;
  for (int32_t i = at >> 3; i < run; i += a.wide_groups >> 3) {
    const int32_t x = (at & 7) * run + i;
    if (x >= all) break;
    const int32_t h = x / items;
    const Item item = a.l.items[1][x - h * items];
    if (item.rows) wide_item<T, DP, REACH>(a, item, h, lds);
  }
}

// Joins a row's partials: weights exp2(lse_c - lse). An entry of several rows, of few parts each, takes half a wavefront a row,
// its lanes over the columns; one of a single row of many parts a workgroup, the parts over the eight halves.
// Bound by the chain of loads (entry, lse, partials) at few rows, by the partials' bytes at many.
template <typename T>
__global__ __launch_bounds__(kThreads, 6) void attend_join_kernel(AttendArgs a) {
  __shared__ f32x4 sums[8][64];
  const int32_t half = threadIdx.x >> 5, column = threadIdx.x & 31;
  const Header head = *a.l.header;
  const bool shared_wide = head.shared_wide;
  const int32_t D = a.head_dim, entries = head.narrow_entries + head.wide_entries;
  for (int32_t at = blockIdx.x; at < entries * a.kv_heads; at += gridDim.x) {
    const int32_t it = at / a.kv_heads, h = at - it * a.kv_heads;
    const bool wide = it >= head.narrow_entries;
    const Entry e = a.l.entries[wide ? a.max_entries - 1 - (it - head.narrow_entries) : it];
    const int32_t own_tile = wide ? kWide : kTile, shared_tile = shared_wide ? kWide : kTile;
    const float* const own_lse = a.partial_lse[wide], * const shared_lse = a.partial_lse[shared_wide];
    const float* const own_o = a.partial[wide], * const shared_o = a.partial[shared_wide];
    const bool many = e.many;
    for (int32_t r = many ? 0 : half; r < e.rows; r += 8) {
      const int32_t row = e.row0 + r, shared_row = e.shared_row0 + r;
      const Parts sh = e.shared_row0 >= 0 ? a.l.shared_parts[shared_row / shared_tile] : Parts{};
      const int32_t own = e.parts.count, parts = own + sh.count;
      const auto row_of = [&](int32_t c) -> int64_t {  // of part c
        if (c < own) return ((int64_t)(c ? e.parts.next + c * e.parts.step : e.parts.slot) * a.kv_heads + h) * own_tile + row % own_tile;
        c -= own;
        return ((int64_t)(c ? sh.next + c * sh.step : sh.slot) * a.kv_heads + h) * shared_tile + shared_row % shared_tile;
      };
      const auto lse_of = [&](int32_t c) { return (c < own ? own_lse : shared_lse)[row_of(c)]; };
      float top = -INFINITY;
      for (int32_t c = column; c < parts; c += 32) top = fmaxf(top, lse_of(c));
      for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
      const float base = top == -INFINITY ? 0.f : top;
      float total = 0;
      for (int32_t c = column; c < parts; c += 32) total += exp2_of(lse_of(c) - base);
      for (int d = 16; d; d >>= 1) total += __shfl_xor(total, d);
      const float inv = total == 0 ? 0.f : 1.f / total;
      const int32_t i = row / a.group, g = row - i * a.group;
      const int64_t out_row = ((int64_t)(e.q_begin + i) * a.kv_heads + h) * a.group + g;
      if (a.lse && column == 0 && (!many || half == 0)) a.lse[out_row] = (total == 0 ? -INFINITY : base + __log2f(total)) * kLn2;
      const auto put = [&](int32_t d, f32x4 x) {
        x *= inv;
        *reinterpret_cast<u32x2*>(a.out + (out_row * D + d) * 2) = u32x2{T::pack(x[0], x[1]), T::pack(x[2], x[3])};
      };
      const auto sum_of = [&](int32_t d, int32_t from, int32_t step) {
        f32x4 x = {};
#pragma unroll 4
        for (int32_t c = from; c < parts; c += step)
          x += *reinterpret_cast<const f32x4*>((c < own ? own_o : shared_o) + row_of(c) * D + d) * fmaxf(exp2_of(lse_of(c) - base), kLeastWeight);
        return x;
      };
      if (!many) {
        for (int32_t d = column * 4; d < D; d += 128) put(d, sum_of(d, 0, 1));
      } else {
        for (int32_t d = column; d < D / 4; d += 32) sums[half][d] = sum_of(d * 4, half, 8);
        __syncthreads();
        for (int32_t d = threadIdx.x; d < D / 4; d += kThreads) {
          f32x4 x = {};
#pragma unroll
          for (int w = 0; w < 8; ++w) x += sums[w][d];
          put(d * 4, x);
        }
        __syncthreads();
      }
    }
  }
}

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

struct Memory {  // of an argument (which may be null)
  const void* p;
  int64_t bytes;
  bool meets(const Memory& o) const {
    return p && o.p && bytes > 0 && o.bytes > 0 && (uintptr_t)p < (uintptr_t)o.p + (uint64_t)o.bytes && (uintptr_t)o.p < (uintptr_t)p + (uint64_t)bytes;
  }
};

// The sizes that follow from the capacities: of narrow and of wide items
struct Sizes {
  int64_t groups, residents, max_items[2], max_slots[2], max_shared_tiles, max_entries;
  bool wide, join;  // can there be wide tiles, or any that are joined?
};

}  // namespace

extern "C" {

struct kvc_attention_plan {
  const int32_t *qo_indptr, *kv_indices, *kv_indptr, *kv_last_page_len;
  int64_t batch_size, num_tokens, num_kv_indices, num_heads, num_kv_heads, head_dim, page_size, shared_pages;
  int64_t narrow_rows;
  int dtype;
  float scale;
  Sizes n;
  int64_t plan_bytes, workspace_bytes;
  char* buffer;  // of kvc_attention_plan_build
};

}  // extern "C"

namespace {

constexpr int64_t kStepGroups = 1024;         // workgroups for narrow tiles of a launch that has wide ones as well
constexpr int64_t kResidents = 512;           // wide items on the card at a time
constexpr int64_t kMaxRounds = 4;             // of them in a step, where a range of keys is longer than the least
// The most rows of a request for narrow tiles, with more it is cut into wide ones: one narrow tile where there is work to
// fill the card, that is, where all rows together, over the requests' average of keys, make more than kMuchWork, else two. 32 rows
// each over 8 key heads: 64 requests of 2000 keys 125 us wide and 133 in two narrow tiles, 256 of 600 169 and 220, one of 16000 31 and 40,
// of 131000 130 and 189; one of 2000 24.8 and 23.0, four of 20 rows and 900 keys 23.1 and 17.3. (One key head, one of 131000: 44 and 29.)
constexpr int64_t kNarrowRows = 32, kMuchWork = 1 << 18;

Layout layout_of(const kvc_attention_plan& p, char* buffer, int64_t* bytes) {
  Layout l;
  int64_t at = 0;
  const auto take = [&](int64_t n) {
    char* q = buffer ? buffer + at : nullptr;
    at += round_up(n, 256);
    return q;
  };
  l.header = (Header*)take(sizeof(Header));
  l.shares = (int32_t*)take(p.shared_pages > 0 ? p.batch_size * 4 : 0);
  l.shared_tokens = (int2*)take(p.shared_pages > 0 ? p.num_tokens * 8 : 0);
  l.ranges = (Range*)take(p.n.groups * sizeof(Range));
  for (int k = 0; k < 2; ++k) l.items[k] = (Item*)take(p.n.max_items[k] * sizeof(Item));
  l.shared_parts = (Parts*)take(p.n.max_shared_tiles * sizeof(Parts));
  l.entries = (Entry*)take(p.n.max_entries * sizeof(Entry));
  if (bytes) *bytes = at;
  return l;
}

// What a step of these capacities can need. Requests with tokens are at most `requests`; those of more than `narrow_rows` rows
// are wide, the others narrow, and only narrow ones share a prefix. Tiles of a kind are at most their rows / tile and one more
// a request. A narrow tile's part in a workgroup has place tile + workgroup in the list; two parts of a workgroup that the line
// reaches need slots, and, where a prefix is shared, every tile's first part. Wide tiles cut into ranges of at least the rounds'
// share of all keys make at most the rounds' items and one more a tile. Slots are for those of two ranges or more: they have no
// more tiles than rounds' items, and no more ranges than the tables' keys hold of the least length. (Heads of 128: 20 tokens of
// 4 x 8 heads over 900 keys 1.5 MB of workspace, 256 tokens of 256 requests 8, or 188 where any request may have them all, 2048
// tokens of 7 x 4 heads behind long contexts 175.)
Sizes sizes_of(const kvc_attention_plan& p) {
  Sizes n;
  const int64_t rows = p.num_tokens * (p.num_heads / p.num_kv_heads), keys = p.num_kv_indices * p.page_size;
  const bool shared = p.shared_pages > 0;
  n.wide = rows > p.narrow_rows || (shared && wide_prefix(rows, p.shared_pages * p.page_size));
  const int64_t groups = n.wide ? kStepGroups : 256 * narrow_residents((int)p.head_dim);
  n.groups = std::min<int64_t>(kMaxGroups, std::max<int64_t>(1, groups / p.num_kv_heads));
  n.residents = std::max<int64_t>(1, kResidents / p.num_kv_heads);
  const int64_t requests = std::min(p.batch_size, p.num_tokens), of_narrow = std::min(rows, p.narrow_rows);
  const int64_t narrow_tiles = std::min(rows / kTile + requests, requests * ((of_narrow + kTile - 1) / kTile));
  const int64_t wide_tiles = rows / kWide + std::min(requests, rows / (p.narrow_rows + 1));
  const auto shared_tiles = [&](int64_t tile) { return shared ? std::min(rows, requests * of_narrow) / tile + 1 : 0; };
  const auto ranges = [](int64_t of) { return of > kMinChunk ? (of + kMinChunk - 1) / kMinChunk : 0; };
  const int64_t rounds = kMaxRounds * n.residents;
  n.max_items[0] = narrow_tiles + shared_tiles(kTile) + n.groups;
  // The line of work of the narrow tiles. It counts a request's keys once a tile (Tiles::before), or its tokens where they are
  // more than its keys; a request has as many tiles as `narrow_rows` allow, all of them where a hint made every request narrow.
  const int64_t each = kTileWork + kTile + 2, request_tokens = of_narrow / (p.num_heads / p.num_kv_heads);
  const int64_t line = (of_narrow + kTile - 1) / kTile * (keys + p.num_tokens) + narrow_tiles * each;
  n.max_slots[0] = shared ? 2 * n.groups + narrow_tiles + shared_tiles(kTile) : 2 * std::min(n.groups, line / kMinShare + 2);
  n.max_items[1] = n.wide ? wide_tiles + shared_tiles(kWide) + rounds : 0;
  n.max_slots[1] = n.wide ? std::min(rounds + std::min(wide_tiles, rounds) + shared_tiles(kWide),
                                     wide_tiles * ranges(keys) + shared_tiles(kWide) * std::max<int64_t>(ranges(p.shared_pages * p.page_size), 1))
                          : 0;
  n.max_shared_tiles = shared_tiles(kTile);
  // Where no tile can be cut none is joined. Narrow ones are cut where the line is longer than all shares of the least length,
  // or a tile as long as one, wide ones where a request has more keys than the least range.
  n.join = shared || line > kMinShare * n.groups || std::max(keys, request_tokens) + each >= kMinShare || (n.wide && keys > kMinChunk);
  n.max_entries = n.join ? rows : 0;
  return n;
}

template <typename T, int DP>
void launch_attend(const AttendArgs& a, const kvc_attention_plan& p, hipStream_t s) {
  const dim3 block(kThreads), grid((unsigned)(a.narrow_groups + a.wide_groups));
  const bool any = a.page_size % 16 != 0, full = a.head_dim == DP;
  // Keys that no cache holds, and that are read once, by non-temporal loads (decode of 256 requests, 2.2 GB: 421 and 406 us;
  // one of 131001 keys, 0.5 GB: 108 and 103; behind a shared prompt, 0.27 GB of which 16 MB are read again and again, 126
  // and 130)
  const bool nt = p.shared_pages == 0 && p.num_kv_indices * 2 * p.page_size * p.num_kv_heads * p.head_dim * 2 >= (int64_t(256) << 20);
  if (p.n.wide) {
    if (any) kvc::launch((attend_step_kernel<T, DP, kAnyPage>), grid, block, 0, s, a);
    else if (!full) kvc::launch((attend_step_kernel<T, DP, kGroups>), grid, block, 0, s, a);
    else kvc::launch((attend_step_kernel<T, DP, kGroupsFull>), grid, block, 0, s, a);
  } else {
    if (any) kvc::launch((attend_rows_kernel<T, DP, kAnyPage>), grid, block, 0, s, a);
    else if (!full) kvc::launch((attend_rows_kernel<T, DP, kGroups>), grid, block, 0, s, a);
    else if (nt) kvc::launch((attend_rows_kernel<T, DP, kGroupsFull, true>), grid, block, 0, s, a);
    else kvc::launch((attend_rows_kernel<T, DP, kGroupsFull>), grid, block, 0, s, a);
  }
}
template <typename T>
void launch_attend(const AttendArgs& a, const kvc_attention_plan& p, hipStream_t s) {
  if (p.head_dim <= 64) launch_attend<T, 64>(a, p, s);
  else if (p.head_dim <= 96) launch_attend<T, 96>(a, p, s);
  else if (p.head_dim <= 128) launch_attend<T, 128>(a, p, s);
  else launch_attend<T, 256>(a, p, s);
  if (!p.n.join) return;
  const unsigned joins = (unsigned)std::min<int64_t>(p.n.max_entries * p.num_kv_heads, 4096);
  kvc::launch((attend_join_kernel<T>), dim3(joins), dim3(kThreads), 0, s, a);
}

}  // namespace

extern "C" {

int kvc_attention_plan_create(const int32_t* qo_indptr, const int32_t* kv_indices, const int32_t* kv_indptr,
                              const int32_t* kv_last_page_len, int64_t batch_size, int64_t num_tokens,
                              int64_t num_kv_indices, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                              int64_t page_size, int64_t max_q_len, int64_t shared_pages, float sm_scale, int dtype,
                              kvc_attention_plan** out) {
  constexpr const char* fn = "kvc_attention_plan_create";
  if (!out) return fail(KVC_ERR_INVALID_ARG, "%s: null out", fn);
  *out = nullptr;
  if (dtype != KVC_DTYPE_BF16 && dtype != KVC_DTYPE_F16)
    return fail(KVC_ERR_UNSUPPORTED, "%s: dtype %d (need bf16 or f16)", fn, dtype);
  if (batch_size < 0 || num_tokens < 0 || num_kv_indices < 0 || shared_pages < 0 || max_q_len < 0)
    return fail(KVC_ERR_INVALID_ARG, "%s: negative size", fn);
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads)
    return fail(KVC_ERR_INVALID_ARG, "%s: %lld query heads are no multiple of %lld key heads", fn, (long long)num_heads,
                (long long)num_kv_heads);
  if (head_dim <= 0 || head_dim % 8 || head_dim > 256)
    return fail(KVC_ERR_UNSUPPORTED, "%s: head_dim %lld (need a multiple of 8 up to 256)", fn, (long long)head_dim);
  if (page_size <= 0 || page_size > (1 << 20))
    return fail(KVC_ERR_INVALID_ARG, "%s: page_size %lld", fn, (long long)page_size);
  if (!(sm_scale > 0) || !std::isfinite(sm_scale))
    return fail(KVC_ERR_INVALID_ARG, "%s: the scale must be positive and finite", fn);
  if (batch_size >= (1 << 24) || num_kv_indices >= (int64_t(1) << 31) || num_heads > 0xffff ||
      num_tokens * num_heads >= (int64_t(1) << 30))
    return fail(KVC_ERR_UNSUPPORTED, "%s: too many requests, pages, tokens or heads", fn);
  if (batch_size > 0 && (!qo_indptr || !kv_indptr || !kv_last_page_len || (num_kv_indices > 0 && !kv_indices)))
    return fail(KVC_ERR_INVALID_ARG, "%s: null pointer", fn);
  // more pages than the tables hold are shared by no one
  if (shared_pages > num_kv_indices || shared_pages * page_size > (1 << 30)) shared_pages = 0;
  kvc_attention_plan* p = new (std::nothrow) kvc_attention_plan{
      qo_indptr, kv_indices, kv_indptr, kv_last_page_len, batch_size, num_tokens, num_kv_indices, num_heads, num_kv_heads,
      head_dim, page_size, shared_pages, kNarrowRows, dtype, sm_scale, {}, 0, 0, nullptr};
  if (!p) return fail(KVC_ERR_HIP, "%s: out of host memory", fn);
  const int64_t rows = num_tokens * (num_heads / num_kv_heads), keys = num_kv_indices * page_size / std::max<int64_t>(batch_size, 1);
  if ((double)rows * (double)keys > (double)kMuchWork) p->narrow_rows = kTile;
  // said to have few tokens each: every request in narrow items, whatever it has, and no launch for the others
  if (max_q_len > 0 && max_q_len * (num_heads / num_kv_heads) <= p->narrow_rows) p->narrow_rows = INT32_MAX;
  p->n = sizes_of(*p);
  layout_of(*p, nullptr, &p->plan_bytes);
  for (int k = 0; k < 2; ++k) p->workspace_bytes += p->n.max_slots[k] * num_kv_heads * (k ? kWide : kTile) * (head_dim + 1) * 4;
  p->workspace_bytes = round_up(std::max<int64_t>(p->workspace_bytes, 1), 256);
  *out = p;
  return KVC_OK;
}

int64_t kvc_attention_plan_bytes(const kvc_attention_plan* plan) {
  return plan ? plan->plan_bytes : (int64_t)fail(KVC_ERR_INVALID_ARG, "kvc_attention_plan_bytes: null plan");
}
int64_t kvc_attention_workspace_bytes(const kvc_attention_plan* plan) {
  return plan ? plan->workspace_bytes : (int64_t)fail(KVC_ERR_INVALID_ARG, "kvc_attention_workspace_bytes: null plan");
}

int kvc_attention_plan_build(kvc_attention_plan* plan, void* buffer, int64_t buffer_bytes, void* stream) {
  constexpr const char* fn = "kvc_attention_plan_build";
  if (!plan) return fail(KVC_ERR_INVALID_ARG, "%s: null plan", fn);
  if (!buffer || (uintptr_t)buffer % 256 || buffer_bytes < plan->plan_bytes)
    return fail(KVC_ERR_STAGING, "%s: the plan needs %lld bytes, aligned to 256", fn, (long long)plan->plan_bytes);
  const Memory to{buffer, plan->plan_bytes};
  if (to.meets({plan->qo_indptr, (plan->batch_size + 1) * 4}) || to.meets({plan->kv_indices, plan->num_kv_indices * 4}) ||
      to.meets({plan->kv_indptr, (plan->batch_size + 1) * 4}) || to.meets({plan->kv_last_page_len, plan->batch_size * 4}))
    return fail(KVC_ERR_INVALID_ARG, "%s: the buffer overlaps the index arrays", fn);
  plan->buffer = (char*)buffer;
  if (plan->batch_size == 0 || plan->num_tokens == 0) return KVC_OK;
  PlanArgs a{plan->qo_indptr, plan->kv_indices, plan->kv_indptr, plan->kv_last_page_len, (int32_t)plan->batch_size,
             (int32_t)plan->num_tokens, (int32_t)plan->num_kv_indices, (int32_t)plan->page_size,
             (int32_t)plan->shared_pages, (int32_t)(plan->num_heads / plan->num_kv_heads), (int32_t)plan->narrow_rows,
             (int32_t)plan->n.groups, (int32_t)plan->n.residents,
             {(int32_t)plan->n.max_items[0], (int32_t)plan->n.max_items[1]}, (int32_t)plan->n.max_entries,
             layout_of(*plan, plan->buffer, nullptr)};
  hipStream_t s = (hipStream_t)stream;
  if (plan->shared_pages > 0) kvc::launch(attend_shares_kernel, dim3((unsigned)plan->batch_size), dim3(256), 0, s, a);
  kvc::launch(attend_schedule_kernel, dim3(1), dim3(1024), 0, s, a);
  KVC_HIP(hipGetLastError());
  return KVC_OK;
}

int kvc_attention_plan_run(const kvc_attention_plan* plan, const void* query, int64_t q_token_stride,
                           const void* paged_kv_cache, int64_t page_stride, int64_t num_pages, void* out, float* lse,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  constexpr const char* fn = "kvc_attention_plan_run";
  if (!plan) return fail(KVC_ERR_INVALID_ARG, "%s: null plan", fn);
  if (plan->batch_size == 0 || plan->num_tokens == 0) return KVC_OK;
  const int64_t row = plan->num_kv_heads * plan->head_dim, page = 2 * plan->page_size * row;
  if (!query || !out || !workspace || (num_pages > 0 && !paged_kv_cache))
    return fail(KVC_ERR_INVALID_ARG, "%s: null pointer", fn);
  if (num_pages < 0 || num_pages >= (int64_t(1) << 31) || page_stride < page || page_stride * 2 >= (int64_t(1) << 32))
    return fail(KVC_ERR_INVALID_ARG, "%s: bad cache geometry", fn);
  if (q_token_stride < plan->num_heads * plan->head_dim)
    return fail(KVC_ERR_INVALID_ARG, "%s: token stride smaller than a row", fn);
  if (((uintptr_t)query | (uintptr_t)paged_kv_cache | (uint64_t)q_token_stride * 2 | (uint64_t)page_stride * 2) % 16 ||
      (uintptr_t)out % 8 || (uintptr_t)lse % 4 || (uintptr_t)workspace % 256)
    return fail(KVC_ERR_INVALID_ARG, "%s: rows must be aligned to 16 bytes, the output to 8", fn);
  if (workspace_bytes < plan->workspace_bytes)
    return fail(KVC_ERR_STAGING, "%s: the workspace needs %lld bytes", fn, (long long)plan->workspace_bytes);
  if (!plan->buffer) return fail(KVC_ERR_INVALID_ARG, "%s: the plan is not built", fn);
  // A row of the query is read before the same row of the output is written, and by no one else afterwards; nothing else that
  // is read or written may share memory with what is written
  const int64_t q_row = plan->num_heads * plan->head_dim * 2;
  const bool in_place = out == query && (plan->num_tokens == 1 || q_token_stride * 2 == q_row);
  const Memory written[] = {{out, plan->num_tokens * q_row}, {lse, plan->num_tokens * plan->num_heads * 4}, {workspace, plan->workspace_bytes}};
  const Memory read[] = {{query, (plan->num_tokens - 1) * q_token_stride * 2 + q_row},
                         {paged_kv_cache, num_pages > 0 ? (num_pages - 1) * page_stride * 2 + page * 2 : 0},
                         {plan->buffer, plan->plan_bytes},
                         {plan->kv_indices, plan->num_kv_indices * 4}};
  bool apart = true;
  for (const Memory& w : written) {
    for (const Memory& r : read) apart = apart && (!w.meets(r) || (&w == written && &r == read && in_place));
    for (const Memory* x = written; x < &w; ++x) apart = apart && !w.meets(*x);
  }
  if (!apart) return fail(KVC_ERR_INVALID_ARG, "%s: what is written overlaps what is read (the output may be the query itself)", fn);
  AttendArgs a{};
  a.query = (const char*)query;
  a.cache = (const char*)paged_kv_cache;
  a.kv_indices = plan->kv_indices;
  a.out = (char*)out;
  a.lse = lse;
  float* at = (float*)workspace;
  for (int k = 0; k < 2; ++k) {
    const int64_t rows = plan->n.max_slots[k] * plan->num_kv_heads * (k ? kWide : kTile);
    a.partial[k] = at;
    at += rows * plan->head_dim;
  }
  for (int k = 0; k < 2; ++k) {
    a.partial_lse[k] = at;
    at += plan->n.max_slots[k] * plan->num_kv_heads * (k ? kWide : kTile);
  }
  a.q_stride = q_token_stride * 2;
  a.page_stride = (uint32_t)(page_stride * 2);
  a.row_stride = (uint32_t)(row * 2);
  a.plane = (uint32_t)(plan->page_size * row * 2);
  a.num_pages = (int32_t)num_pages;
  a.page_size = (int32_t)plan->page_size;
  a.page_shift = log2_exact(plan->page_size);
  a.kv_heads = (int32_t)plan->num_kv_heads;
  a.group = (int32_t)(plan->num_heads / plan->num_kv_heads);
  a.head_dim = (int32_t)plan->head_dim;
  a.narrow_groups = (int32_t)(plan->n.groups * plan->num_kv_heads);
  // (a workgroup takes further items where there are more than these)
  a.wide_groups = (int32_t)round_up(std::min<int64_t>(plan->n.max_items[1] * plan->num_kv_heads, 4096), 8);
  a.max_entries = (int32_t)plan->n.max_entries;
  a.scale = plan->scale * kLog2e;
  a.l = layout_of(*plan, plan->buffer, nullptr);
  if (plan->dtype == KVC_DTYPE_BF16) launch_attend<BF16>(a, *plan, (hipStream_t)stream);
  else launch_attend<F16>(a, *plan, (hipStream_t)stream);
  KVC_HIP(hipGetLastError());
  return KVC_OK;
}

int kvc_attention_plan_destroy(kvc_attention_plan* plan) {
  delete plan;
  return KVC_OK;
}

}  // extern "C"
