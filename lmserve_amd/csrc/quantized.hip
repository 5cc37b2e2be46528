// K/V write into the 8-bit cache, and back (gfx950).
//
// A group of 16 tokens of a head has one exponent for K and one for V, the least e with which the largest magnitude of its tokens
// is at most 448 2^e; a code is x 2^-e rounded to e4m3. As the scale is a power of two, the product is exact and the code has one
// rounding, whatever order the group's tokens come in within a call. The tokens of a group come in several calls, one at a time in decode: a call that begins
// at the group's first token begins the group anew, another one keeps e where it is enough, and where it is not, the codes that are
// there are rounded again to the new e, which changes nothing but those that get below the type's normal numbers.
//
// A workgroup's wavefronts deal with 16 tokens: a token that continues its predecessor's group belongs to that one's run, every
// other opens a run, and the wavefronts of the 16 tokens take (run, head, K or V) in turn. So decode, where every token is a run, and
// prefill, where 16 are one, have as many wavefronts at work from one launch, without a list of runs.
//   K: a lane has 8 columns of a row, 16 bytes as they come, and stores their 8 codes.
//   V: a lane has 2 columns of all tokens, 4 bytes a token, 256 bytes a wavefront, and stores 16 codes of each: the group's
//   transposition needs no LDS. A group that is continued is read, and written whole.
// Bound by HBM and the caches from some thousand tokens on (16384 tokens of 8 heads of 128, 101 MB: 20.2 to 21.9 us, 4.6 to 5.0 TB/s, and 17.8 where a
// graph writes the same rows again, which the last-level cache then holds; 131001 read back, 0.8 GB: 144 us, 5.6 TB/s), by launch and the chain of slots,
// rows and exponents below (256 single tokens, each of which has a group of V read and written whole, 7.7 us in a graph, 6.5 over the same rows; one token 4.0).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "common.h"
#include "device.h"
#include "kvcache.h"
#include "q8.h"

namespace {

using namespace kvc;
using namespace kvc::q8;

constexpr int kThreads = 256, kWavesPerGroup = kThreads / 64;
constexpr int kChunk = 16;  // tokens of a workgroup
// Rows beyond so many bytes go past the caches. What is read back: stores past them (8 heads of 128, 8192 tokens, 32 MiB of rows, 10.7 us without and
// 9.4 so, 32768 43.4 and 31.2, 131001 158 and 144); what is written: loads (32768 tokens, 128 MiB of rows, 42.6 us without and 36.7 so, 65536 82
// and 69; 16384 18.6 and 20.9, whose rows a projection before them leaves in the caches). The codes are stored plainly, through the
// caches they cost 23 us at 16384.
constexpr int64_t kReadPastBytes = int64_t(32) << 20, kWritePastBytes = int64_t(128) << 20;

struct Args {
  char *key, *value;  // rows, read or written
  int64_t k_stride, v_stride;  // bytes
  char* cache;
  const void* slots;  // or null: the page table's arrays
  const int32_t *batch_indices, *positions, *kv_indices, *kv_indptr;
  int64_t num_tokens, num_slots;
  int32_t slot_bytes, batch_size, num_kv_indices, num_pages, page_size, page_shift;
  int32_t heads, dim;
  uint32_t splits, page_stride, group_stride;
};

// A token's place in the cache, page * page_size + entry, or -1: none
__device__ __forceinline__ int64_t slot_of(const Args& a, int64_t t) {
  if (t < 0 || t >= a.num_tokens) return -1;
  if (a.slots) {
    const int64_t s = a.slot_bytes == 8 ? reinterpret_cast<const int64_t*>(a.slots)[t] : reinterpret_cast<const int32_t*>(a.slots)[t];
    return s >= 0 && s < a.num_slots ? s : -1;
  }
  const int32_t b = a.batch_indices[t], p = a.positions[t];
  if (b < 0 || b >= a.batch_size || p < 0) return -1;
  const int32_t in_table = a.page_shift >= 0 ? p >> a.page_shift : p / a.page_size;
  const int32_t begin = a.kv_indptr[b];
  const int64_t i = (int64_t)begin + in_table;
  if (begin < 0 || i >= a.kv_indptr[b + 1] || i >= a.num_kv_indices) return -1;
  const int32_t page = a.kv_indices[i];
  if (page < 0 || page >= a.num_pages) return -1;
  return (int64_t)page * a.page_size + (p - in_table * a.page_size);
}

struct Run {  // tokens of a call that lie one behind another in a group
  char* group;
  int64_t token;       // the first
  int32_t first, end;  // and their places in the group
};

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  for (int d = 32; d; d >>= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)x, d);
    x = x > y ? x : y;
  }
  return x;
}

// The largest magnitude of a wavefront's finite 16-bit values; whether there are others
template <typename T, int N>
__device__ __forceinline__ float largest(const uint32_t (&words)[N], bool& odd) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 top = {};
#pragma unroll
  for (int i = 0; i < N; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, words[i] & 0x7fff7fffu));
  uint32_t one = wave_max(top[0] > top[1] ? top[0] : top[1]);
  odd = one >= T::kExponent;
  if (odd) {
    one = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int s = 0; s < 32; s += 16) {
        const uint32_t x = words[i] >> s & 0x7fffu;
        if (x < T::kExponent && x > one) one = x;
      }
    one = wave_max(one);
  }
  return T::wide(one);
}

// The group's exponent, stored, when tokens up to `top` join those before `first`, which had `had`; how far it has grown
__device__ __forceinline__ int32_t grow(const Run& r, int32_t had, float top, int32_t& grown) {
  const int32_t need = exponent_of(top);
  had = r.first == 0 ? 0 : min(max(had, kLeast + kBias), kMost + kBias);
  grown = r.first && need > had ? need - had : 0;
  return max(need, had);
}

// Codes of a group that has grown by 2^n, rounded again (exact up to there: codes are numbers of f16); NaN stays
__device__ __forceinline__ uint32_t rescaled(uint32_t codes, int32_t n) {
  const float scale = power_of((uint32_t)(kBias + min(n, 64)));
  const uint32_t lo = F16::from_codes<false>(codes, 1.f), hi = F16::from_codes<true>(codes, 1.f);
  const uint32_t c = F16::to_codes<true>(hi, scale, F16::to_codes<false>(lo, scale, 0));
  return c & ~nan_codes(c);
}

// Codes of 4 values, two to a word; an infinity or NaN is the positive NaN
template <typename T>
__device__ __forceinline__ uint32_t codes_of(uint32_t x, uint32_t y, float scale, bool odd) {
  const uint32_t c = T::template to_codes<true>(y, scale, T::template to_codes<false>(x, scale, 0));
  return odd ? c & ~nan_codes(c) : c;
}

// LPR: lanes to a row of 16-byte vectors
template <typename T, int LPR>
struct Head {
  static constexpr int RPP = 64 / LPR, PASSES = kGroup / RPP;
  static constexpr int TPL = LPR == 8 ? 8 : 16;         // tokens of a lane's columns of V
  static constexpr int COLUMNS = LPR == 32 ? 2 : 1;     // pairs of columns of a lane
  static constexpr int WORDS = TPL / 4;

  template <bool PAST>
  static __device__ __forceinline__ void write_k(const Args& a, const Run& r, int32_t h, int32_t lane) {
    const int32_t row = lane / LPR, col = lane % LPR, D = a.dim;
    const bool there = col * 8 < D;
    const char* from = a.key + r.token * a.k_stride + ((int64_t)h * D + col * 8) * 2;
    char* const to = r.group + h * kGroup * D + col / 2 * 64 + col % 2 * 8;
    uint8_t* const exponent = reinterpret_cast<uint8_t*>(r.group + 2 * kGroup * a.heads * D + 2 * h);
    const int32_t had = *exponent;
    uint32_t x[PASSES * 4] = {};
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int32_t t = p * RPP + row;
      if (there && t >= r.first && t < r.end) {
        const u32x4 v = get<PAST, u32x4>(from + (t - r.first) * a.k_stride);
#pragma unroll
        for (int w = 0; w < 4; ++w) x[p * 4 + w] = v[w];
      }
    }
    bool odd;
    int32_t grown;
    const float top = largest<T>(x, odd);
    const int32_t e = grow(r, had, top, grown);
    const float scale = power_of(e);
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int32_t t = p * RPP + row;
      u32x2* const tile = reinterpret_cast<u32x2*>(to + t / 4 * (4 * D) + t % 4 * 16);
      if (!there || t >= r.end) continue;
      if (t >= r.first) {
        *tile = u32x2{codes_of<T>(x[p * 4], x[p * 4 + 1], scale, odd), codes_of<T>(x[p * 4 + 2], x[p * 4 + 3], scale, odd)};
      } else if (grown) {
        const u32x2 c = *tile;
        *tile = u32x2{rescaled(c[0], grown), rescaled(c[1], grown)};
      }
    }
    if (lane == 0) *exponent = (uint8_t)e;
  }

  template <bool PAST>
  static __device__ __forceinline__ void write_v(const Args& a, const Run& r, int32_t h, int32_t lane) {
    const int32_t D = a.dim, t0 = TPL == 8 ? lane / 32 * 8 : 0, pair = TPL == 8 ? lane % 32 : lane;
    const char* from = a.value + r.token * a.v_stride + ((int64_t)h * D + pair * 2) * 2;
    char* const to = r.group + kGroup * a.heads * D + (int64_t)h * kGroup * D + pair * 2 * kGroup + t0;
    uint8_t* const exponent = reinterpret_cast<uint8_t*>(r.group + 2 * kGroup * a.heads * D + 2 * h + 1);
    const int32_t had = *exponent;
    const bool whole = r.first == 0 && r.end == kGroup;
    uint32_t x[COLUMNS * TPL] = {}, old[COLUMNS][2][WORDS] = {};
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c)
      if ((c * 64 + pair) * 2 < D) {
        if (whole) {
#pragma unroll
          for (int i = 0; i < TPL; ++i) x[c * TPL + i] = get<PAST, uint32_t>(from + (t0 + i) * a.v_stride + c * 256);
        } else {
#pragma unroll
          for (int i = 0; i < TPL; ++i)
            if (t0 + i >= r.first && t0 + i < r.end)
              x[c * TPL + i] = get<PAST, uint32_t>(from + (t0 + i - r.first) * a.v_stride + c * 256);
#pragma unroll
          for (int d = 0; d < 2; ++d) load(reinterpret_cast<const uint32_t*>(to + c * 128 * kGroup + d * kGroup), old[c][d]);
        }
      }
    bool odd;
    int32_t grown;
    const float top = largest<T>(x, odd);
    const int32_t e = grow(r, had, top, grown);
    const float scale = power_of(e);
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) {
      if ((c * 64 + pair) * 2 >= D) continue;
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        uint32_t now[WORDS];
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
          const uint32_t* y = x + c * TPL + w * 4;
          const auto two = [&](int i) { return __builtin_amdgcn_perm(y[i + 1], y[i], d ? 0x07060302u : 0x05040100u); };
          now[w] = codes_of<T>(two(0), two(2), scale, odd);
          if (!whole) {
            const uint32_t before = bytes_below(r.first, t0 + w * 4), until = bytes_below(r.end, t0 + w * 4);
            const uint32_t kept = grown ? rescaled(old[c][d][w], grown) : old[c][d][w];
            now[w] = (kept & before) | (now[w] & until & ~before) | (old[c][d][w] & ~until);
          }
        }
        store(reinterpret_cast<uint32_t*>(to + c * 128 * kGroup + d * kGroup), now);
      }
    }
    if (lane == 0) *exponent = (uint8_t)e;
  }

  static __device__ __forceinline__ void load(const uint32_t* p, uint32_t (&v)[WORDS]) {
    if constexpr (WORDS == 4) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(p);
      for (int i = 0; i < 4; ++i) v[i] = x[i];
    } else {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p);
      v[0] = x[0], v[1] = x[1];
    }
  }
  static __device__ __forceinline__ void store(uint32_t* p, const uint32_t (&v)[WORDS]) {
    if constexpr (WORDS == 4) *reinterpret_cast<u32x4*>(p) = u32x4{v[0], v[1], v[2], v[3]};
    else *reinterpret_cast<u32x2*>(p) = u32x2{v[0], v[1]};
  }
  template <bool PAST, typename V>
  static __device__ __forceinline__ void put(char* p, V v) {
    if constexpr (PAST) st_through_nt(p, v);
    else *reinterpret_cast<V*>(p) = v;
  }
  template <bool PAST, typename V>
  static __device__ __forceinline__ V get(const char* p) {
    if constexpr (PAST) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    else return *reinterpret_cast<const V*>(p);
  }

  static __device__ __forceinline__ float scale_at(const char* exponent) {
    return power_of(max((uint32_t)*reinterpret_cast<const uint8_t*>(exponent), 1u));
  }

  template <bool PAST>
  static __device__ __forceinline__ void read_k(const Args& a, const Run& r, int32_t h, int32_t lane) {
    const int32_t row = lane / LPR, col = lane % LPR, D = a.dim;
    if (col * 8 >= D) return;
    const char* const from = r.group + h * kGroup * D + col / 2 * 64 + col % 2 * 8;
    char* to = a.key + r.token * a.k_stride + ((int64_t)h * D + col * 8) * 2;
    const float by = scale_at(r.group + 2 * kGroup * a.heads * D + 2 * h);
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int32_t t = p * RPP + row;
      if (t < r.first || t >= r.end) continue;
      const u32x2 c = *reinterpret_cast<const u32x2*>(from + t / 4 * (4 * D) + t % 4 * 16);
      put<PAST>(to + (t - r.first) * a.k_stride,
                u32x4{T::template from_codes<false>(c[0], by), T::template from_codes<true>(c[0], by), T::template from_codes<false>(c[1], by),
                      T::template from_codes<true>(c[1], by)});
    }
  }

  template <bool PAST>
  static __device__ __forceinline__ void read_v(const Args& a, const Run& r, int32_t h, int32_t lane) {
    const int32_t D = a.dim, t0 = TPL == 8 ? lane / 32 * 8 : 0, pair = TPL == 8 ? lane % 32 : lane;
    char* to = a.value + r.token * a.v_stride + ((int64_t)h * D + pair * 2) * 2;
    const char* const from = r.group + kGroup * a.heads * D + (int64_t)h * kGroup * D + pair * 2 * kGroup + t0;
    const float by = scale_at(r.group + 2 * kGroup * a.heads * D + 2 * h + 1);
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) {
      if ((c * 64 + pair) * 2 >= D) continue;
      uint32_t x[2][WORDS];
#pragma unroll
      for (int d = 0; d < 2; ++d) load(reinterpret_cast<const uint32_t*>(from + c * 128 * kGroup + d * kGroup), x[d]);
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        // tokens 2 i and 2 i + 1 of both columns
        const uint32_t column[2][2] = {{T::template from_codes<false>(x[0][w], by), T::template from_codes<true>(x[0][w], by)},
                                       {T::template from_codes<false>(x[1][w], by), T::template from_codes<true>(x[1][w], by)}};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t t = t0 + w * 4 + i;
          if (t >= r.first && t < r.end)
            put<PAST>(to + (t - r.first) * a.v_stride + c * 256,
                      (uint32_t)__builtin_amdgcn_perm(column[1][i / 2], column[0][i / 2], i % 2 ? 0x07060302u : 0x05040100u));
        }
      }
    }
  }
};

enum Way : int { kWrite, kWritePast, kRead, kReadPast };
template <typename T, int LPR, Way WAY>
__global__ __launch_bounds__(kThreads) void rows_kernel(Args a) {
  const int32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  // The workgroups of 16 tokens on one XCD, of 8 that take such runs of workgroups in turn (16384 tokens written 19.7 us in the plain order, 18.1 so)
  const uint32_t turn = 8 * a.splits, whole = gridDim.x / turn * turn, in = blockIdx.x / 8;
  const bool dealt = blockIdx.x < whole;
  const int64_t chunk = dealt ? in / a.splits * 8 + blockIdx.x % 8 : blockIdx.x / a.splits;
  const int32_t split = dealt ? in % a.splits : blockIdx.x % a.splits;
  const int32_t waves = a.splits * kWavesPerGroup;
  // the 16 tokens are lanes 1 to 16; the one before them, and those behind them that their groups may reach
  const int64_t slot = lane < 2 * kChunk ? slot_of(a, chunk * kChunk - 1 + lane) : -1;
  const int64_t before = __shfl_up((long long)slot, 1);
  const bool follows = lane > 0 && slot >= 0 && slot % kGroup != 0 && slot == before + 1;
  const uint32_t continues = (uint32_t)__ballot(follows);
  uint32_t opens = (uint32_t)__ballot(lane >= 1 && lane <= kChunk && slot >= 0 && !follows);
  const int32_t tasks = __popc(opens) * a.heads * 2;
  int32_t at = 0;
  for (int32_t i = split * kWavesPerGroup + wave; i < tasks; i += waves) {
    const int32_t run = i / (2 * a.heads), rest = i - run * 2 * a.heads;
    for (; at < run; ++at) opens &= opens - 1;
    const int32_t first = __builtin_ctz(opens);
    const int64_t s = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(slot >> 32), first) << 32 |
                                (uint32_t)__builtin_amdgcn_readlane((int)slot, first));
    const int64_t page = a.page_shift >= 0 ? s >> a.page_shift : s / a.page_size;
    const int32_t entry = (int32_t)(s - page * a.page_size);
    Run r;
    r.group = a.cache + page * a.page_stride + (int64_t)(entry / kGroup) * a.group_stride;
    r.token = chunk * kChunk - 1 + first;
    r.first = entry % kGroup;
    r.end = r.first + 1 + __builtin_ctz(~(continues >> (first + 1)));
    constexpr bool PAST = WAY == kWritePast || WAY == kReadPast;
    if constexpr (WAY >= kRead) {
      if (rest & 1) Head<T, LPR>::template read_v<PAST>(a, r, rest >> 1, lane);
      else Head<T, LPR>::template read_k<PAST>(a, r, rest >> 1, lane);
    } else {
      if (rest & 1) Head<T, LPR>::template write_v<PAST>(a, r, rest >> 1, lane);
      else Head<T, LPR>::template write_k<PAST>(a, r, rest >> 1, lane);
    }
  }
}

template <typename T, Way WAY>
void launch_rows(const Args& a, unsigned grid, hipStream_t s) {
  if (a.dim <= 64) kvc::launch((rows_kernel<T, 8, WAY>), dim3(grid), dim3(kThreads), 0, s, a);
  else if (a.dim <= 128) kvc::launch((rows_kernel<T, 16, WAY>), dim3(grid), dim3(kThreads), 0, s, a);
  else kvc::launch((rows_kernel<T, 32, WAY>), dim3(grid), dim3(kThreads), 0, s, a);
}

int check_geometry(const char* fn, int64_t heads, int64_t dim, int64_t page_size) {
  if (heads <= 0 || heads > 0xffff) return fail(KVC_ERR_INVALID_ARG, "%s: %lld heads", fn, (long long)heads);
  if (dim <= 0 || dim % 16 || dim > 256)
    return fail(KVC_ERR_UNSUPPORTED, "%s: head_dim %lld (an 8-bit cache needs a multiple of 16 up to 256)", fn, (long long)dim);
  if (page_size <= 0 || page_size % kGroup || page_size > (1 << 20))
    return fail(KVC_ERR_UNSUPPORTED, "%s: page_size %lld (an 8-bit cache needs a multiple of 16)", fn, (long long)page_size);
  if (page_size / kGroup * group_bytes(heads, dim) >= int64_t(1) << 32)
    return fail(KVC_ERR_UNSUPPORTED, "%s: pages of 4 GiB and more", fn);
  return KVC_OK;
}

struct Index {
  const void* slots;
  int slot_bytes;
  const int32_t *batch_indices, *positions, *kv_indices, *kv_indptr;
  int64_t batch_size, num_kv_indices;
};

int run_rows(const char* fn, bool read, const void* key, const void* value, void* cache, const Index& x, int64_t num_tokens,
             int64_t heads, int64_t dim, int64_t page_size, int64_t k_stride, int64_t v_stride, int64_t page_stride, int64_t num_pages,
             int dtype, void* stream) {
  if (const int rc = check_geometry(fn, heads, dim, page_size)) return rc;
  if (dtype != KVC_DTYPE_BF16 && dtype != KVC_DTYPE_F16) return fail(KVC_ERR_UNSUPPORTED, "%s: dtype %d (need bf16 or f16)", fn, dtype);
  if (num_tokens < 0 || num_pages < 0 || num_pages >= (int64_t(1) << 31) || x.batch_size < 0 || x.num_kv_indices < 0 ||
      x.batch_size >= (int64_t(1) << 31) || x.num_kv_indices >= (int64_t(1) << 31))
    return fail(KVC_ERR_INVALID_ARG, "%s: bad size", fn);
  const int64_t page = page_size / kGroup * group_bytes(heads, dim), row = heads * dim;
  if (page_stride < page || page_stride >= (int64_t(1) << 32))
    return fail(KVC_ERR_INVALID_ARG, "%s: page_stride %lld (pages have %lld bytes)", fn, (long long)page_stride, (long long)page);
  if (k_stride < row || v_stride < row) return fail(KVC_ERR_INVALID_ARG, "%s: token stride smaller than a row", fn);
  if (x.slots && x.slot_bytes != 4 && x.slot_bytes != 8) return fail(KVC_ERR_UNSUPPORTED, "%s: slot_bytes %d", fn, x.slot_bytes);
  if (num_tokens == 0 || num_pages == 0) return KVC_OK;
  if (!key || !value || !cache || (!x.slots && (!x.batch_indices || !x.positions || !x.kv_indptr || (x.num_kv_indices > 0 && !x.kv_indices))))
    return fail(KVC_ERR_INVALID_ARG, "%s: null pointer", fn);
  if (((uintptr_t)key | (uintptr_t)value | (uintptr_t)cache | (uint64_t)k_stride * 2 | (uint64_t)v_stride * 2 | (uint64_t)page_stride) % 16)
    return fail(KVC_ERR_INVALID_ARG, "%s: rows and pages must be aligned to 16 bytes", fn);
  const Memory rows[] = {{key, ((num_tokens - 1) * k_stride + row) * 2}, {value, ((num_tokens - 1) * v_stride + row) * 2}};
  const Memory pages{cache, (num_pages - 1) * page_stride + page};
  const Memory index[] = {{x.slots, num_tokens * x.slot_bytes}, {x.batch_indices, num_tokens * 4}, {x.positions, num_tokens * 4},
                          {x.kv_indices, x.num_kv_indices * 4}, {x.kv_indptr, (x.batch_size + 1) * 4}};
  bool apart = !rows[0].meets(pages) && !rows[1].meets(pages);
  if (read && rows[0].meets(rows[1])) {  // slices of the same rows lie side by side
    const int64_t d = (int64_t)(((uintptr_t)value - (uintptr_t)key) / 2) % k_stride, ahead = d < 0 ? d + k_stride : d;
    apart = apart && k_stride == v_stride && ahead >= row && k_stride - ahead >= row;
  }
  for (const Memory& m : index) apart = apart && (read ? !m.meets(rows[0]) && !m.meets(rows[1]) : !m.meets(pages));
  if (!apart) return fail(KVC_ERR_INVALID_ARG, "%s: what is written overlaps what is read", fn);
  const int64_t chunks = (num_tokens + kChunk - 1) / kChunk;
  // As many wavefronts for 16 tokens as their runs can use, from 2 for a head (one run, K and V) up to 32 (16 runs), 4096 in all as far as that
  // allows (8 heads of 128: 256 requests' tokens 6.7 us, 7.5 with 2048; 4 heads, 2048 tokens of four requests 5.2, 4.3 with 2048 and 6.5 with 8192).
  const int64_t waves = std::min(std::max<int64_t>(4096 / chunks, 2 * heads), 2 * heads * kChunk);
  const int64_t splits = (waves + kWavesPerGroup - 1) / kWavesPerGroup;
  if (chunks * splits >= (int64_t(1) << 31)) return fail(KVC_ERR_UNSUPPORTED, "%s: too many tokens", fn);
  Args a{(char*)key, (char*)value, k_stride * 2, v_stride * 2, (char*)cache, x.slots, x.batch_indices, x.positions, x.kv_indices, x.kv_indptr,
         num_tokens, num_pages * page_size, x.slot_bytes, (int32_t)x.batch_size, (int32_t)x.num_kv_indices, (int32_t)num_pages,
         (int32_t)page_size, log2_exact(page_size), (int32_t)heads, (int32_t)dim, (uint32_t)splits, (uint32_t)page_stride,
         (uint32_t)group_bytes(heads, dim)};
  const unsigned grid = (unsigned)(chunks * splits);
  hipStream_t s = (hipStream_t)stream;
  const bool bf16 = dtype == KVC_DTYPE_BF16, past = num_tokens * row * 4 >= (read ? kReadPastBytes : kWritePastBytes);
  switch (read ? past ? kReadPast : kRead : past ? kWritePast : kWrite) {
    case kWrite: bf16 ? launch_rows<BF16, kWrite>(a, grid, s) : launch_rows<F16, kWrite>(a, grid, s); break;
    case kWritePast: bf16 ? launch_rows<BF16, kWritePast>(a, grid, s) : launch_rows<F16, kWritePast>(a, grid, s); break;
    case kRead: bf16 ? launch_rows<BF16, kRead>(a, grid, s) : launch_rows<F16, kRead>(a, grid, s); break;
    case kReadPast: bf16 ? launch_rows<BF16, kReadPast>(a, grid, s) : launch_rows<F16, kReadPast>(a, grid, s); break;
  }
  KVC_HIP(hipGetLastError());
  return KVC_OK;
}

}  // namespace

extern "C" {

int64_t kvc_q8_page_bytes(int64_t num_kv_heads, int64_t head_dim, int64_t page_size) {
  if (const int rc = check_geometry("kvc_q8_page_bytes", num_kv_heads, head_dim, page_size)) return rc;
  return page_size / kGroup * group_bytes(num_kv_heads, head_dim);
}

int kvc_reshape_and_cache_q8(const void* key, const void* value, void* kv_cache, const void* slot_mapping, int slot_bytes,
                             int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim, int64_t page_size, int64_t key_token_stride,
                             int64_t value_token_stride, int64_t page_stride, int64_t num_pages, int dtype, void* stream) {
  if (num_tokens > 0 && !slot_mapping) return fail(KVC_ERR_INVALID_ARG, "kvc_reshape_and_cache_q8: null pointer");
  return run_rows("kvc_reshape_and_cache_q8", false, key, value, kv_cache, {slot_mapping, slot_bytes, nullptr, nullptr, nullptr, nullptr, 0, 0},
                  num_tokens, num_kv_heads, head_dim, page_size, key_token_stride, value_token_stride, page_stride, num_pages, dtype, stream);
}

int kvc_append_paged_kv_cache_q8(const void* append_key, const void* append_value, const int32_t* batch_indices, const int32_t* positions,
                                 void* paged_kv_cache, const int32_t* kv_indices, const int32_t* kv_indptr,
                                 const int32_t* kv_last_page_len, int64_t nnz, int64_t batch_size, int64_t num_kv_indices,
                                 int64_t num_kv_heads, int64_t head_dim, int64_t page_size, int64_t key_token_stride,
                                 int64_t value_token_stride, int64_t page_stride, int64_t num_pages, int dtype, void* stream) {
  (void)kv_last_page_len;
  return run_rows("kvc_append_paged_kv_cache_q8", false, append_key, append_value, paged_kv_cache,
                  {nullptr, 0, batch_indices, positions, kv_indices, kv_indptr, batch_size, num_kv_indices}, nnz, num_kv_heads, head_dim,
                  page_size, key_token_stride, value_token_stride, page_stride, num_pages, dtype, stream);
}

int kvc_read_cache_q8(const void* kv_cache, const void* slot_mapping, int slot_bytes, void* key, void* value, int64_t num_tokens,
                      int64_t num_kv_heads, int64_t head_dim, int64_t page_size, int64_t key_token_stride, int64_t value_token_stride,
                      int64_t page_stride, int64_t num_pages, int dtype, void* stream) {
  if (num_tokens > 0 && !slot_mapping) return fail(KVC_ERR_INVALID_ARG, "kvc_read_cache_q8: null pointer");
  return run_rows("kvc_read_cache_q8", true, key, value, (void*)kv_cache, {slot_mapping, slot_bytes, nullptr, nullptr, nullptr, nullptr, 0, 0},
                  num_tokens, num_kv_heads, head_dim, page_size, key_token_stride, value_token_stride, page_stride, num_pages, dtype, stream);
}

int kvc_read_paged_kv_cache_q8(const int32_t* batch_indices, const int32_t* positions, const void* paged_kv_cache, const int32_t* kv_indices,
                               const int32_t* kv_indptr, const int32_t* kv_last_page_len, void* key, void* value, int64_t nnz,
                               int64_t batch_size, int64_t num_kv_indices, int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                               int64_t key_token_stride, int64_t value_token_stride, int64_t page_stride, int64_t num_pages, int dtype,
                               void* stream) {
  (void)kv_last_page_len;
  return run_rows("kvc_read_paged_kv_cache_q8", true, key, value, (void*)paged_kv_cache,
                  {nullptr, 0, batch_indices, positions, kv_indices, kv_indptr, batch_size, num_kv_indices}, nnz, num_kv_heads, head_dim,
                  page_size, key_token_stride, value_token_stride, page_stride, num_pages, dtype, stream);
}

}  // extern "C"
