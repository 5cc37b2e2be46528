// Causal attention over the 8-bit cache (gfx950): the tiles of the step's layout (attention.hip lays it out and joins the parts).
//
// A key's codes c and its group's exponents ek, ev: k = c 2^ek, v = c 2^ev. The matrix instructions take 16 bits, and every code is a
// number of bf16 and of f16, so nothing is rounded on the way to them:
//   the scores are those of the codes, and 2^ek goes with the softmax's scale into the exponent's multiply-add: a lane's scores
//   are of one group, so that is one register;
//   V's codes are the product's as they are, and 2^ev goes with the weights: a weight is exp2(score - base) 2^(ev - E) there, and O in units of
//   2^(base + E). base and E are a row's own: base follows its highest score, base + E the greatest score + ev of the keys that it sees. So
//   what a row does not see has no part in its units, and a weight is rounded as a part of the row's largest term, weight times group's size.
// The weights are f16, scaled up as in the 16-bit kernels, whatever the query's type. base and E are whole numbers, so what has been summed is scaled exactly.
//
// The keys are permuted: which row of the matrix instruction's A a key is does not matter, and with
//   row 4 g + r of the i-th product = token 4 i + r of group g        (16 rows, 4 groups, products i = 0..3)
//   row 8 j + 4 g + r = token 4 j + r of group g                      (32 rows, 2 groups)
// a lane's scores come out as the 16 tokens of one group in order, which is what its weights have to be beside V's columns as the cache
// holds them. So V needs no transposition, and a narrow tile no LDS before its end.

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "attention.h"
#include "device.h"
#include "q8.h"

namespace {

using namespace kvc;
using namespace kvc::attn;
using namespace kvc::q8;

constexpr float kLowest = -1000;  // E before the row's first key
// What ev - E is held to. At most kFar: E is raised to the greatest ev of the keys that the row sees less that, however small their weights. At least
// kNear: what f16 holds of a weight ends long before, and the sum, in fp32, keeps weights from 2^-62 on. From kLag down a base is looked after by itself.
constexpr int32_t kNear = -64, kFar = 100, kLag = -40;
// From here on a base is too large to have ev - E added to it in fp32
constexpr float kHuge = 1 << 22;
constexpr int kVPad = 16;  // bytes between a wide item's columns of V in LDS

// The code below keeps the lanes of a wavefront together: what differs between lanes is selected, loads go to an address that is there for
// every lane, and an item is in scalar registers. With registers of every kind in use (heads of 256) the compiler saves vector registers at the end of
// a region that some lanes skipped, before it lets these lanes in again: they lose what was saved.
__device__ __forceinline__ Item uniform(const Item& x) {
  const auto one = [](int32_t v) { return __builtin_amdgcn_readfirstlane(v); };
  return Item{one(x.q_begin), one(x.row0), one(x.rows), one(x.table), one(x.key_begin), one(x.key_end), one(x.slot), one(x.limit)};
}

// 8 codes as 8 numbers, times a power of two
template <typename T>
__device__ __forceinline__ u32x4 widen(uint32_t lo, uint32_t hi, float by) {
  return u32x4{T::template from_codes<false>(lo, by), T::template from_codes<true>(lo, by), T::template from_codes<false>(hi, by),
               T::template from_codes<true>(hi, by)};
}
// What the scores of a group of K are scaled by. A product beyond fp32's normal numbers would make 0 * inf or -inf * 0 of scores that are
// 0 or masked; at their ends it has the same weights, as scores of that size are equal, or infinitely apart, in fp32.
__device__ __forceinline__ float score_scale(float scale, uint32_t ek) {
  return __builtin_amdgcn_fmed3f(scale * power_of(ek), 1.17549435e-38f, 3.402823466e38f);
}
// Is a key before `end` (of an item that has keys), and on a page of the cache? Where its group lies (that of what is not there: at the cache's beginning)
__device__ __forceinline__ bool find_group(const AttendArgs& a, int32_t table, int32_t key, int32_t end, uint64_t& at) {
  const int32_t k = min(max(key, 0), end - 1);
  const int32_t p = a.page_shift >= 0 ? k >> a.page_shift : k / a.page_size;
  const int32_t page = a.kv_indices[table + p];
  const bool there = key >= 0 && key < end && page >= 0 && page < a.num_pages;
  const uint32_t in = there ? (uint32_t)(k - p * a.page_size) / kGroup : 0;
  at = (uint64_t)(uint32_t)(there ? page : 0) * a.page_stride + (uint64_t)in * a.group_stride;
  return there;
}

template <bool NT, typename V>
__device__ __forceinline__ V load(const char* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
  else return *reinterpret_cast<const V*>(p);
}

// NaN among V's codes of 4 tokens, which a weight of 0 does not cancel, taken out
__device__ __forceinline__ uint32_t without_nan(uint32_t codes) { return codes & ~((nan_codes(codes) >> 7) * 0xffu); }
// Is the code of a token of a column NaN?
__device__ __forceinline__ bool is_nan(const char* column, int32_t token) { return (column[token] & 0x7f) == 0x7f; }

// ---- narrow items: up to 16 rows, a wavefront takes 64 keys at once ----------------------------------------------------
// A lane (n = lane % 16, quad = lane / 16) reads, in 16-byte loads,
//   of K the columns 64 s + 16 quad.. of token 4 i + n % 4 of group n / 4: two operands of the product i,
//   of V the column 16 d + n of group quad: 16 tokens, two operands,
// and holds the scores and weights of row n and group quad.
// Bound by HBM where there are many keys: decode of 256 requests, 1.13 GB of codes, 182 us (6.2 TB/s; the 16-bit cache 400), one
// request of 131001 keys 45 to 63; by the chain of item, pages, keys and the joining of wavefronts where there are few: 900 keys of one
// request 6.7 us. Two workgroups a CU by their registers (three, with 45 of them spilled, are slower); asking for the next item's
// record, pages, queries and keys ahead cost more in code and registers than it hid (one request of 900 keys 6.7 to 7.3 us, one of 32000 keys 26.6 to 29.2).
// f16 queries have their weights in two parts, as over 16 bits; with bf16 outputs the rest of an f16 weight, 2^-12 of it, is below their rounding.
template <int DP>
constexpr int narrow_lds() { return kWaves * kTile * (DP + 4) * 4 + kWaves * kTile * 12; }

template <typename T, int DP, bool FULL, bool NT>
struct Narrow {
  static constexpr int KS = DP / 64, DTILES = DP / 16;
  u32x4 k[4][KS], v[DTILES];
  uint32_t exps;        // of the lane's group
  int32_t avail;        // its tokens that are the item's
  // where the next 16 blocks' groups lie, one to a lane: block (L / 4), group L % 4
  uint32_t at_lo, at_hi;
  uint64_t there;
  const char *k_at, *v_at;

  __device__ __forceinline__ void look_up(const AttendArgs& a, const Item& item, int32_t k0, int32_t lane) {
    uint64_t at;
    there = __ballot(find_group(a, item.table, k0 + (lane >> 2) * (kWaves * kStep) + (lane & 3) * kGroup, item.key_end, at));
    at_lo = (uint32_t)at;
    at_hi = (uint32_t)(at >> 32);
  }
  __device__ __forceinline__ const char* place(const char* base, int32_t group) const {
    const uint32_t lo = (uint32_t)__shfl((int)at_lo, group), hi = (uint32_t)__shfl((int)at_hi, group);
    return base + (int64_t)((uint64_t)hi << 32 | lo);
  }
  // The (it mod 16)-th block of those that were looked up: its places, K and exponents
  __device__ __forceinline__ void load_k(const AttendArgs& a, const Item& item, int32_t h, int32_t k0, int32_t it, int32_t lane) {
    const int32_t n = lane & 15, quad = lane >> 4, D = a.head_dim, first = (it & 15) * 4;
    k_at = place(a.cache + (int64_t)h * kGroup * D + quad * 64 + n % 4 * 16, first + n / 4);
    v_at = place(a.cache, first + quad);
    avail = there >> (first + quad) & 1 ? min(max(item.key_end - k0 - quad * kGroup, 0), kGroup) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        // (columns that the head does not have meet zeros of the query: any number will do, but no NaN)
        const bool have = FULL || s * 64 + quad * 16 < D;
        const u32x4 x = load<NT, u32x4>(k_at + i * 4 * (FULL ? DP : D) + (have ? s * 256 : -quad * 64));
        k[i][s] = have ? x : u32x4{};
      }
    exps = *reinterpret_cast<const uint16_t*>(v_at + a.exponents + 2 * h);
  }
  __device__ __forceinline__ void load_v(const AttendArgs& a, int32_t h, int32_t lane) {
    const int32_t D = a.head_dim;
    const char* from = v_at + a.plane + (int64_t)h * kGroup * D + (lane & 15) * 16;
#pragma unroll
    for (int d = 0; d < DTILES; ++d) {
      if (!FULL) v[d] = u32x4{};
      if (FULL || d * 16 < D) v[d] = load<NT, u32x4>(from + d * 256);
    }
  }
};

template <typename T, int DP, bool FULL, bool NT>
__device__ __forceinline__ void narrow_item(const AttendArgs& a, const Item& given, int32_t h, char* lds) {
  const Item item = uniform(given);
  typedef Narrow<T, DP, FULL, NT> Block;
  constexpr int KS = Block::KS, DTILES = Block::DTILES, OSTRIDE = DP + 4, STEP = kWaves * kStep;
  constexpr bool kRest = std::is_same<T, F16>::value;
  constexpr float kScaledUp = F16::kScaledUp, kOutgrown = kScaledUp + 1, kUnscaled = 1.f / (1 << (int)kScaledUp);
  float(*const stats)[3][kTile] = reinterpret_cast<float(*)[3][kTile]>(lds + kWaves * kTile * OSTRIDE * 4);
  const int32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t n = lane & 15, quad = lane >> 4, D = a.head_dim;
  float* const my_o = reinterpret_cast<float*>(lds) + wave * kTile * OSTRIDE;

  u32x4 q[KS][2] = {};
  f32x4 o[DTILES] = {};
  float base = -INFINITY, l = 0;  // weights are exp2(score * scale - base)
  float E = kLowest;              // O is in units of 2^(base + E)
  int32_t limit = 0, odd_from = INT32_MAX;
  {
    const int32_t row = item.row0 + min(n, item.rows - 1), i = row / a.group, g = row - i * a.group;  // (rows that are not there: the last)
    const int2 x = item.q_begin >= 0 ? make_int2(item.q_begin + i, item.limit + i) : a.l.shared_tokens[i];
    limit = n < item.rows ? clamp(x.y, 0, item.key_end) : 0;
    const char* p = a.query + (int64_t)x.x * a.q_stride + (int64_t)(h * a.group + g) * D * 2;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const bool have = FULL || s * 64 + quad * 16 < D;
        const u32x4 y = *reinterpret_cast<const u32x4*>(p + (have ? s * 128 + quad * 32 : 0) + half * 16);
        q[s][half] = have ? y : u32x4{};
      }
  }
  int32_t k0 = item.key_begin + wave * kStep;
  if (k0 < item.key_end && a.num_pages > 0) {
    Block b;
    b.look_up(a, item, k0, lane);
    b.load_k(a, item, h, k0, 0, lane);
    b.load_v(a, h, lane);
    for (int32_t it = 1;; ++it, k0 += STEP) {
      const bool more = k0 + STEP < item.key_end;
      f32x4 s[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          s[i] = T::mfma(widen<T>(b.k[i][c][0], b.k[i][c][1], 1.f), q[c][0], s[i]);
          s[i] = T::mfma(widen<T>(b.k[i][c][2], b.k[i][c][3], 1.f), q[c][1], s[i]);
        }
      const int32_t avail = b.avail, first = k0 + quad * kGroup;
      const int32_t ek = avail ? (int32_t)(b.exps & 255) : kBias;
      const float ev = (float)(b.exps >> 8);
      if (more) {
        if ((it & 15) == 0) b.look_up(a, item, k0 + STEP, lane);
        b.load_k(a, item, h, k0 + STEP, it, lane);
      }
      // does a row stop inside the block, or the item?
      const int32_t sees = min(max(limit - first, 0), avail);
      const bool ragged = __ballot(n < item.rows && sees < avail) != 0;
      if (ragged || __ballot(avail < kGroup)) {
#pragma unroll
        for (int j = 0; j < kGroup; ++j)
          if (j >= sees) s[j / 4][j % 4] = -INFINITY;
        uint32_t odd = 0;
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            b.v[d][w] &= bytes_below(avail, w * 4);
            odd |= nan_codes(b.v[d][w]);
          }
        if (ragged && __ballot(odd != 0)) {
          odd_from = min(odd_from, k0);
#pragma unroll
          for (int d = 0; d < DTILES; ++d)
#pragma unroll
            for (int w = 0; w < 4; ++w) b.v[d][w] = without_nan(b.v[d][w]);
        }
      }
      const float scale = score_scale(a.scale, ek);
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][r]);
      const float mine = top * scale;  // of the lane's group
      top = max_across32(max_across16(mine));
      const float grown = fmaxf(base, __builtin_ceilf(top) - kScaledUp);
      const float from = grown == -INFINITY ? 0.f : grown;
      const float by_weight = exp2_of(base - from);  // 0 from -inf
      E = fmaxf(E + (base - from), kLowest);  // O's units stay (or it comes to nothing below)
      base = grown;
      const float need = (mine == -INFINITY ? 3 * kLowest : ev) - E + fmaxf(mine - from, kOutgrown - kFar);
      if (__ballot(need > kOutgrown)) {
        const float up = fmaxf(__builtin_ceilf(max_across32(max_across16(need))) - kScaledUp, 0.f), shrink = exp2_of(-up);
#pragma unroll
        for (int d = 0; d < DTILES; ++d) o[d] *= shrink;
        E += up;
      }
      const float t = fminf(fmaxf(ev - E, kNear), kFar);
      float by = scale, minus = t - from;
      if (__ballot(__builtin_fabsf(from) > kHuge)) {
#pragma unroll
        for (int j = 0; j < kGroup; ++j) s[j / 4][j % 4] = __builtin_fmaf(s[j / 4][j % 4], scale, -from);
        by = 1, minus = t;
      }
      u32x4 p[2], rest[2];
      float sum = 0;
#pragma unroll
      for (int j = 0; j < kGroup; j += 2) {
        const float x = exp2_of(__builtin_fmaf(s[j / 4][j % 4], by, minus));
        const float y = exp2_of(__builtin_fmaf(s[j / 4][j % 4 + 1], by, minus));
        const uint32_t two = F16::pack(x, y);
        p[j / 8][j % 8 / 2] = two;
        if (kRest) rest[j / 8][j % 8 / 2] = F16::pack(x - F16::wide(two & 0xffffu), y - F16::wide(two >> 16));
        sum += x + y;
      }
      l = l * by_weight + sum * exp2_of(-t);
#pragma unroll
      for (int d = 0; d < DTILES; ++d) {
        const u32x4 lo = widen<F16>(b.v[d][0], b.v[d][1], 1.f), hi = widen<F16>(b.v[d][2], b.v[d][3], 1.f);
        o[d] = F16::mfma(lo, p[0], o[d]);
        o[d] = F16::mfma(hi, p[1], o[d]);
        if (kRest) {
          o[d] = F16::mfma(lo, rest[0], o[d]);
          o[d] = F16::mfma(hi, rest[1], o[d]);
        }
      }
      if (!more) break;
      b.load_v(a, h, lane);
    }
  }
  // the sum over the four quads' keys
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  // NaN of V that were left out, where rows stop, go to the rows that see them
  if (__builtin_expect(odd_from < item.key_end, 0)) {
    for (int32_t b0 = odd_from; b0 < item.key_end; b0 += STEP)
#pragma unroll 1
      for (int32_t key = b0; key < min(b0 + kStep, item.key_end); ++key) {
        uint64_t at;
        const bool sees = find_group(a, item.table, key, item.key_end, at) && key < limit;
        const char* column = a.cache + at + a.plane + ((int64_t)h * D + quad * 4) * kGroup;
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
          if (FULL || d * 16 < D)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d][e] = is_nan(column + (d * 16 + e) * kGroup, key % kGroup) & sees ? NAN : o[d][e];
      }
  }
  // over the wavefronts (the four quads have the same)
  stats[wave][0][n] = base;
  stats[wave][1][n] = l;
  __syncthreads();
  float top = -INFINITY, all_l = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][0][n]);
  const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all_l += stats[w][1][n] * exp2_of(stats[w][0][n] - from);
  const float weight = exp2_of(base - from) * (all_l == 0 ? 0.f : 1.f / all_l);
#pragma unroll
  for (int d = 0; d < DTILES; ++d) {
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = l == 0 ? 0.f : __builtin_ldexpf(o[d][e] * weight, (int32_t)E - kBias);
    *reinterpret_cast<f32x4*>(my_o + n * OSTRIDE + d * 16 + quad * 4) = x;
  }
  if (wave == 0 && quad == 0 && n < item.rows) {
    const float lse2 = all_l == 0 ? -INFINITY : from + kScaledUp + __log2f(all_l * kUnscaled);
    if (item.slot >= 0) {
      a.partial_lse[0][partial_row(item.slot, a.kv_heads, h, kTile, n)] = lse2;
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
    for (int w = 0; w < kWaves; ++w) x += *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(lds) + (w * kTile + r) * OSTRIDE + d);
    if (item.slot >= 0) {
      *reinterpret_cast<f32x4*>(a.partial[0] + partial_row(item.slot, a.kv_heads, h, kTile, r) * D + d) = x;
    } else {
      const int32_t row = item.row0 + r, i = row / a.group, g = row - i * a.group;
      *reinterpret_cast<u32x2*>(a.out + (((int64_t)(item.q_begin + i) * a.kv_heads + h) * a.group + g) * D * 2 + d * 2) =
          u32x2{T::pack(x[0], x[1]), T::pack(x[2], x[3])};
    }
  }
  __syncthreads();  // before the next item
}

// ---- wide items: up to 128 rows, a workgroup takes 64 keys at once ------------------------------------------------------
// As the wide tiles over 16 bits (attention.hip): 32 rows to a wavefront, K half a step ahead of V, one barrier a step. What is
// staged in LDS is 16 bits: K as the query's type, its rows permuted, V as f16 columns, so a group is converted once for
// all four wavefronts; a wavefront converts the group of the window that is its own number.
// V's columns lie in LDS as the product takes them, so it reads them whole, without the transposing read.
// Heads of 64 have three workgroups a CU (a step of 3 chunks and 60 single tokens 62 us with two, 182 registers, 57 with three, 168 and 24 to 28 bytes spilled).
// Bound as over 16 bits, by what two wavefronts a SIMD have under way: 2048 new tokens behind 13 to 30 thousand keys 773 to 860 us from card to
// card (16 bits: 770 to 820), 830 to 925 TFLOP/s.
template <int DP>
constexpr int wide_lds() { return 2 * kStep * (DP * 2 + 16) + 2 * DP * (kStep * 2 + kVPad) + (kWaves + 1) * 4; }

struct Window {  // of 64 keys
  uint64_t present;  // which are there
  uint64_t exps;     // its groups' exponents, 16 bits each
};

template <typename T, int DP, bool FULL>
__device__ __forceinline__ void wide_item(const AttendArgs& a, const Item& given, int32_t h, char* lds) {
  const Item item = uniform(given);
  constexpr int KSTEPS = DP / 16, DTILES = DP / 32, ROUNDS = (DP + 63) / 64;
  constexpr int KSTRIDE = DP * 2 + 16, VSTRIDE = kStep * 2 + kVPad;
  constexpr float kScaledUp = F16::kScaledUp / 2, kOutgrown = 8 + kScaledUp, kUnscaled = 1.f / (1 << (int)kScaledUp);
  typedef char KStep[kStep * KSTRIDE];
  typedef char VStep[DP * VSTRIDE];
  KStep* const k_lds = reinterpret_cast<KStep*>(lds);
  VStep* const v_lds = reinterpret_cast<VStep*>(lds + 2 * sizeof(KStep));
  int32_t* const leasts = reinterpret_cast<int32_t*>(lds + 2 * sizeof(KStep) + 2 * sizeof(VStep));
  int32_t& left_out = leasts[kWaves];
  const int32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t n = lane & 31, hi = lane >> 5, D = FULL ? DP : a.head_dim;
  const char* const heads = a.cache + (int64_t)h * kGroup * D;
  const int32_t my_row = wave * 32 + n;
  u32x4 q[KSTEPS] = {};
  int32_t limit = 0, token = 0, g = 0;
  {
    const int32_t row = item.row0 + min(my_row, item.rows - 1), i = row / a.group;  // (rows that are not there: the last)
    g = row - i * a.group;
    const int2 x = item.q_begin >= 0 ? make_int2(item.q_begin + i, item.limit + i) : a.l.shared_tokens[i];
    token = x.x;
    limit = my_row < item.rows ? clamp(x.y, 0, item.key_end) : 0;
    const char* p = a.query + (int64_t)token * a.q_stride + ((int64_t)(h * a.group + g) * D + hi * 8) * 2;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k)
      if (FULL || k * 16 < D) q[k] = *reinterpret_cast<const u32x4*>(p + k * 32);
  }
  // the wavefront's first limit (rows that are not there have none)
  int32_t least = my_row < item.rows ? limit : INT32_MAX;
  for (int d = 16; d; d >>= 1) least = min(least, __shfl_xor(least, d));
  least = __builtin_amdgcn_readfirstlane(least);
  leasts[wave] = least;
  left_out = 0;
  if (!FULL)  // the columns of K beyond head_dim: zeros, as the query's are
    for (int32_t x = tid; x < 2 * kStep * ((DP - D) / 8); x += kThreads) {
      const int32_t row = x / ((DP - D) / 8), c = x - row * ((DP - D) / 8);
      *reinterpret_cast<u32x4*>(lds + row * KSTRIDE + (D + c * 8) * 2) = u32x4{};
    }
  __syncthreads();
  const int32_t tile_least = min(min(leasts[0], leasts[1]), min(leasts[2], leasts[3]));
  f32x16 o[DTILES] = {};
  float base = -INFINITY, l = 0;  // as in a narrow tile
  // The sum of the weights as they went into the product, rounded: what O is divided by with f16 outputs, as a row of few keys then keeps what their weights'
  // roundings have in common (chunks of 5 to 50 tokens from their first key on: up to 1.63 times the plain form's error without, 1.46 so; a step of 3 chunks
  // and 60 single tokens 57.0 and 59.5 us). Beside bf16's rounding there is no difference.
  constexpr bool kRounded = std::is_same<T, F16>::value;
  float rounded = 0;
  int32_t E = (int32_t)kLowest, least_E = E, most_E = E;  // (of the wavefront's rows that see keys)
  bool huge = false;
  u32x4 kr[ROUNDS], vr[ROUNDS];
  // where the groups of 16 windows lie, one to a lane, which of them are there, their exponents
  uint32_t group_lo = 0, group_hi = 0, group_exps = 0;
  uint64_t groups = 0;
  const char* place = nullptr;  // of the wavefront's group of the window that K was last asked of
  // Keys come in windows of 64: window w begins 32 before the item's 64 w-th key, so that what a step reads, K of the 64
  // keys from its own 32nd on and V of the 64 keys up to its own 32nd, are the windows w + 1 and w.
  const auto window = [&](int32_t w) { return item.key_begin + w * kStep - kStep / 2; };
  // the lane's 16-byte pieces of a group's K or V (where there are fewer than lanes, the last one more than once)
  const auto piece_of = [&](int i) { return FULL && DP % 64 == 0 ? lane + i * 64 : min(lane + i * 64, D - 1); };
  // K of a window, on its way
  const auto fetch_k = [&](int32_t w) -> Window {
    const int32_t first = window(w);
    if ((w & 15) == 0) {
      const int32_t key = first + lane * kGroup;
      uint64_t at;
      const bool there = find_group(a, item.table, key < item.key_begin ? -1 : key, item.key_end, at);
      groups = __ballot(there);
      group_lo = (uint32_t)at;
      group_hi = (uint32_t)(at >> 32);
      const uint32_t exps = *reinterpret_cast<const uint16_t*>(a.cache + at + a.exponents + 2 * h);
      group_exps = there ? exps : kBias << 8 | kBias;
    }
    const uint32_t four = (uint32_t)(groups >> (w & 15) * 4) & 15, left = (uint32_t)(item.key_end - first);
    Window x;
    x.present = ~(uint64_t)0;
    if (four != 15 || left < kStep) {
      x.present = 0;
      for (int i = 0; i < 4; ++i) x.present |= (uint64_t)(four >> i & 1 ? 0xffffu : 0) << (i * 16);
      if (left < kStep) x.present &= ((uint64_t)1 << left) - 1;
    }
    x.exps = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t e = (uint32_t)__builtin_amdgcn_readlane((int)group_exps, (w & 15) * 4 + i);
      x.exps |= (uint64_t)e << (i * 16);
    }
    place = heads + (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)group_hi, (w & 15) * 4 + wave) << 32 |
                              (uint32_t)__builtin_amdgcn_readlane((int)group_lo, (w & 15) * 4 + wave));
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) kr[i] = *reinterpret_cast<const u32x4*>(place + piece_of(i) * 16);
    return x;
  };
  // V of the window that K was last asked of
  const auto fetch_v = [&]() {
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) vr[i] = *reinterpret_cast<const u32x4*>(place + a.plane + piece_of(i) * 16);
  };
  const auto stage_k = [&](int buf) {
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      // a piece is 16 columns of a token; the tokens' rows are those of the matrix instruction
      const int32_t x = piece_of(i), four = x / (D / 4), in = x - four * (D / 4);
      char* const to = k_lds[buf] + ((wave >> 1) * 32 + four * 8 + (wave & 1) * 4 + (in & 3)) * KSTRIDE + (in >> 2) * 32;
      *reinterpret_cast<u32x4*>(to) = widen<T>(kr[i][0], kr[i][1], 1.f);
      *reinterpret_cast<u32x4*>(to + 16) = widen<T>(kr[i][2], kr[i][3], 1.f);
    }
  };
  const auto stage_v = [&](int buf, int32_t w, const Window& x) {
    const uint32_t mine = (uint32_t)(x.present >> wave * 16) & 0xffffu;
    if (mine != 0xffffu) {  // tokens that are not there
      const int32_t avail = __builtin_popcount(mine);
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) vr[i][j] &= bytes_below(avail, j * 4);
    }
    if (window(w) + kStep > tile_least) {  // a row stops in it: are there NaN, which a weight of 0 does not cancel?
      uint32_t odd = 0;
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= nan_codes(vr[i][j]);
      if (__ballot(odd != 0)) {
        left_out = 1;
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) vr[i][j] = without_nan(vr[i][j]);
      }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      char* const to = v_lds[buf] + piece_of(i) * VSTRIDE + wave * 32;
      *reinterpret_cast<u32x4*>(to) = widen<F16>(vr[i][0], vr[i][1], 1.f);
      *reinterpret_cast<u32x4*>(to + 16) = widen<F16>(vr[i][2], vr[i][3], 1.f);
    }
  };

  // Pieces from LDS: 16 columns of K of 32 keys (a half of a step); of 32 columns of V 8 tokens of the lane's group
  const auto k_piece = [&](int buf, int half, int j) {
    return *reinterpret_cast<const u32x4*>(k_lds[buf] + (half * 32 + n) * KSTRIDE + hi * 16 + j * 32);
  };
  const auto v_piece = [&](int buf, int half, int j) {
    return *reinterpret_cast<const u32x4*>(v_lds[buf] + (j % DTILES * 32 + n) * VSTRIDE + half * 64 + hi * 32 + j / DTILES * 16);
  };
  // the exponents of the lane's group of a half of a window; the scale of its scores
  const auto exps_of = [&](const Window& x, int half) {
    const uint32_t two = (uint32_t)(x.exps >> half * 32);
    return hi ? two >> 16 : two & 0xffffu;
  };
  const auto scale_of = [&](uint32_t exps) { return score_scale(a.scale, exps & 255); };
  const auto evs_of = [&](const Window& x, int half) {
    const uint32_t two = (uint32_t)(x.exps >> half * 32);
    return make_int2(two >> 8 & 255, two >> 24);
  };
  const auto highest = [&](f32x16& s) {
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    return top;
  };
  // the highest score of the lane's group of 32 keys, scaled, those of keys that the row does not see taken out
  const auto mask = [&](f32x16& s, float top, float scale, int32_t k0, uint32_t present) {
    if (least < k0 + 32 || ~present) {
      const int32_t left = clamp(limit - k0 - hi * 16, 0, 16);
      const uint32_t sees = ((1u << left) - 1) & (hi ? present >> 16 : present);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!(sees >> r & 1)) s[r] = -INFINITY;
      top = highest(s);
    }
    return top * scale;
  };
  // Units of O that have been outgrown, and with them the base, as over 16 bits. (The base may be outgrown by more, as its weights stay in
  // fp32: by kOutgrown - kLag, while no ev is further below E than that.) The exponents of the weights to come, s * scale + minus, in
  // which they are scaled by 2^(ev - E); what their sum is scaled back by. `evs` are those of both groups.
  const auto grow = [&](f32x16& s, float& scale, float mine, int32_t ev, int2 evs, uint32_t* waiting, float& minus) {
    const float need = mine - base + (float)(ev - E);
    if (__ballot(need > kOutgrown) || max(evs.x, evs.y) - least_E > kFar || min(evs.x, evs.y) - most_E < kLag) {
      const float top = max_across32(mine), grown = top > base + kOutgrown ? __builtin_ceilf(top) - kScaledUp : base;
      const float by = base - (grown == -INFINITY ? 0.f : grown);  // -inf from -inf
      l *= exp2_of(by);
      if (kRounded) rounded *= exp2_of(by);
      E = max(E + (int32_t)fmaxf(by, kLowest), (int32_t)kLowest);  // O's units stay (or it comes to nothing here)
      base = grown;
      const float above = max_across32(mine == -INFINITY ? mine : fmaxf(mine - base, kOutgrown - kFar) + (float)(ev - E));
      const float up = above > kOutgrown ? __builtin_ceilf(above) - kScaledUp : 0.f, shrink = exp2_of(-up);
#pragma unroll
      for (int d = 0; d < DTILES; ++d) o[d] *= shrink;
#pragma unroll
      for (int i = 0; i < 8; ++i) waiting[i] = F16::pack(F16::wide(waiting[i] & 0xffffu) * shrink, F16::wide(waiting[i] >> 16) * shrink);
      E += (int32_t)up;
      int32_t x = limit > item.key_begin ? E : INT32_MAX, y = limit > item.key_begin ? E : INT32_MIN / 2;
      for (int d = 16; d; d >>= 1) x = min(x, __shfl_xor(x, d)), y = max(y, __shfl_xor(y, d));
      least_E = __builtin_amdgcn_readfirstlane(x);
      most_E = __builtin_amdgcn_readfirstlane(y);
      huge = __ballot(__builtin_fabsf(base) > kHuge && base != -INFINITY);
    }
    const int32_t t = clamp(ev - E, kNear, kFar);
    const float from = base == -INFINITY ? 0.f : base;
    minus = (float)t - from;
    if (__builtin_expect(huge, 0)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], scale, -from);
      scale = 1;
      minus = (float)t;
    }
    return __uint_as_float((uint32_t)(kBias - t) << 23);
  };
  // 32 keys: their weights from the scores s, while the scores of the keys behind them and the product of the weights
  // before them, that waited, with V are on the matrix unit, in the order of attention.hip.
  const auto take = [&](const f32x16& s, float scale, float minus, float back, uint32_t* p, f32x16& next, float& top, const uint32_t* waiting, int buf, auto which,
                        u32x4* piece) {
    constexpr int PIECES = KSTEPS + 2 * DTILES, HALF = decltype(which)::value;
    static_assert(PIECES % (kAhead + 1) == 0, "the second half's first pieces are asked for at the end of the first's");
    float sum[2] = {}, weight[3] = {}, used = 0;
    next = f32x16{};
    // a weight is used behind the next one's exponential, whose result the adder would wait for
    const auto add = [&](int r) {
      sum[r % 2] += weight[r % 3];
      asm volatile("" : "+v"(sum[r % 2]));
      if (r % 2) {
        p[r / 2] = F16::pack(weight[(r + 2) % 3], weight[r % 3]);
        asm volatile("" : "+v"(p[r / 2]));
        if (kRounded) used = F16::sum(p[r / 2], used);
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
        o[v % DTILES] = F16::mfma(piece[j % (kAhead + 1)], u32x4{w[0], w[1], w[2], w[3]}, o[v % DTILES]);
      }
#pragma unroll
      for (int r = j * 16 / PIECES; r < (j + 1) * 16 / PIECES; ++r) {
        float y = exp2_of(__builtin_fmaf(s[r], scale, minus));
        asm volatile("" : "+v"(y));  // here, and not where it is used
        weight[r % 3] = y;
        if (r) add(r - 1);
      }
      if (j == PIECES - 1) top = highest(next);
      __builtin_amdgcn_sched_barrier(0);
    }
    add(15);
    const float all = sum[0] + sum[1];
    l = __builtin_fmaf(all, back, l);
    // (where they are further off than numbers of f16 are rounded, 2^(ev - E) has scaled them to below f16's: values that count for nothing, weights that do)
    if (kRounded) rounded = __builtin_fmaf(__builtin_fabsf(used - all) <= all * (1.f / 2048) ? used : all, back, rounded);
  };
  const int32_t steps = a.num_pages > 0 ? (item.key_end - item.key_begin + kStep - 1) / kStep : 0;
  if (steps > 0) {
    int32_t k0 = item.key_begin;
    // nothing waits for the first product: zeros, and V of the keys before the first is cleared
    uint32_t p0[8], p1[8] = {};
    const Window before = fetch_k(0);
    fetch_v();
    stage_k(1);
    stage_v(0, 0, before);
    Window now = fetch_k(1), coming = {}, then = {};  // the windows i + 1, i + 2, i + 3
    fetch_v();
    stage_k(0);
    if (steps > 1) coming = fetch_k(2);
    __syncthreads();
    f32x16 s0 = {}, s1;
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j) s0 = T::mfma(k_piece(1, 1, j), q[j], s0);
    uint32_t exps0 = exps_of(before, 1);
    int2 evs0 = evs_of(before, 1);
    float scale0 = scale_of(exps0);
    float top = mask(s0, highest(s0), scale0, k0, (uint32_t)(before.present >> 32));
    for (int32_t i = 0; i < steps; ++i, k0 += kStep) {
      const int buf = i & 1;
      u32x4 piece[kAhead + 1];
      __syncthreads();  // this step's windows are there, the last step's have been read
      stage_v(buf ^ 1, i + 1, now);
      if (i + 1 < steps) {
        stage_k(buf ^ 1);
        fetch_v();
        if (i + 2 < steps) then = fetch_k(i + 3);
      }
      // before the other workgroup's wavefronts that stage
      __builtin_amdgcn_s_setprio(1);
      float minus;
      const float back0 = grow(s0, scale0, top, (int32_t)(exps0 >> 8), evs0, p1, minus);
      take(s0, scale0, minus, back0, p0, s1, top, p1, buf, std::integral_constant<int, 0>{}, piece);
      const uint32_t exps1 = exps_of(now, 0);
      float scale1 = scale_of(exps1);
      top = mask(s1, top, scale1, k0 + 32, (uint32_t)now.present);
      const float back1 = grow(s1, scale1, top, (int32_t)(exps1 >> 8), evs_of(now, 0), p0, minus);
      take(s1, scale1, minus, back1, p1, s0, top, p0, buf, std::integral_constant<int, 1>{}, piece);  // (after the last step: scores of keys that are not there)
      exps0 = exps_of(now, 1);
      evs0 = evs_of(now, 1);
      scale0 = scale_of(exps0);
      top = mask(s0, top, scale0, k0 + kStep, (uint32_t)(now.present >> 32));
      __builtin_amdgcn_s_setprio(0);
      now = coming;
      coming = then;
    }
    __syncthreads();
    // the last weights' product
#pragma unroll
    for (int j = 0; j < 2 * DTILES; ++j) {
      const uint32_t* w = p1 + j / DTILES * 4;
      o[j % DTILES] = F16::mfma(v_piece(steps & 1, 0, j), u32x4{w[0], w[1], w[2], w[3]}, o[j % DTILES]);
    }
  }
  __syncthreads();  // (left_out is complete, and the buffers are free)
  l += __shfl_xor(l, 32);
  if (kRounded) rounded += __shfl_xor(rounded, 32);
  if (__builtin_expect(left_out, 0)) {  // as above
    const int32_t from = item.key_begin + max((max(tile_least - item.key_begin, 0) + kStep / 2) / kStep * kStep - kStep / 2, 0);
#pragma unroll 1
    for (int32_t key = from; key < item.key_end; ++key) {
      uint64_t at;
      const bool sees = find_group(a, item.table, key, item.key_end, at) && key < limit;
      const char* column = heads + at + a.plane;
      int32_t last = D - 1, mine = hi * 4;
      asm volatile("" : "+s"(last), "+v"(mine));  // here, and not for all columns ahead of the items
#pragma unroll
      for (int d = 0; d < DTILES; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int32_t c = d * 32 + r / 4 * 8 + mine + r % 4;  // (of columns beyond the head's: any of its own)
          o[d][r] = is_nan(column + (FULL ? c : min(c, last)) * kGroup, key % kGroup) & sees ? NAN : o[d][r];
        }
    }
  }
  const float inv = l == 0 ? 0.f : 1.f / (kRounded ? rounded : l), lse2 = l == 0 ? -INFINITY : base + kScaledUp + __log2f(l * kUnscaled);
  if (my_row < item.rows) {
    const auto four = [&](int d, int i) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = l == 0 ? 0.f : __builtin_ldexpf(o[d][i * 4 + e] * inv, E - kBias);
      return x;
    };
    if (item.slot >= 0) {
      const int64_t row = partial_row(item.slot, a.kv_heads, h, kWide, my_row);
      if (hi == 0) a.partial_lse[1][row] = lse2;
#pragma unroll
      for (int d = 0; d < DTILES; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t c = d * 32 + i * 8 + hi * 4;
          if (!FULL && d * 32 + i * 8 >= D) continue;
          *reinterpret_cast<f32x4*>(a.partial[1] + row * D + c) = four(d, i);
        }
    } else {
      const int64_t row = ((int64_t)token * a.kv_heads + h) * a.group + g;
      if (a.lse && hi == 0) a.lse[row] = lse2 * kLn2;
#pragma unroll
      for (int d = 0; d < DTILES; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t c = d * 32 + i * 8 + hi * 4;
          if (!FULL && d * 32 + i * 8 >= D) continue;
          const f32x4 x = four(d, i);
          *reinterpret_cast<u32x2*>(a.out + (row * D + c) * 2) = u32x2{T::pack(x[0], x[1]), T::pack(x[2], x[3])};
        }
    }
  }
  __syncthreads();  // before the next item
}

template <typename T, int DP, bool FULL, bool NT>
__global__ __launch_bounds__(kThreads, q8_narrow_residents(DP)) void rows_kernel(AttendArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[narrow_lds<DP>()];
  take_share(a, blockIdx.x, [&](const Item& item, int32_t h) { narrow_item<T, DP, FULL, NT>(a, item, h, lds); });
}
template <typename T, int DP, bool FULL>
__global__ __launch_bounds__(kThreads, DP <= 64 && FULL ? 3 : DP <= 128 ? 2 : 1) void step_kernel(AttendArgs a) {
  constexpr int LDS = wide_lds<DP>() > narrow_lds<DP>() ? wide_lds<DP>() : narrow_lds<DP>();
  __shared__ __attribute__((aligned(16))) char lds[LDS];
  take_step<true>(a, [&](const Item& item, int32_t h) { narrow_item<T, DP, FULL, false>(a, item, h, lds); },
                  [&](const Item& item, int32_t h) { wide_item<T, DP, FULL>(a, item, h, lds); });
}

template <typename T, int DP>
void launch_tiles(const AttendArgs& a, bool wide, bool nt, hipStream_t s) {
  const dim3 block(kThreads), grid((unsigned)(a.narrow_groups + (wide ? a.wide_groups : 0)));
  const bool full = a.head_dim == DP;
  if (wide) {
    if (full) kvc::launch((step_kernel<T, DP, true>), grid, block, 0, s, a);
    else kvc::launch((step_kernel<T, DP, false>), grid, block, 0, s, a);
  } else {
    if (!full) kvc::launch((rows_kernel<T, DP, false, false>), grid, block, 0, s, a);
    else if (nt) kvc::launch((rows_kernel<T, DP, true, true>), grid, block, 0, s, a);
    else kvc::launch((rows_kernel<T, DP, true, false>), grid, block, 0, s, a);
  }
}
template <typename T>
void launch_tiles(const AttendArgs& a, bool wide, bool nt, hipStream_t s) {
  if (a.head_dim <= 64) launch_tiles<T, 64>(a, wide, nt, s);
  else if (a.head_dim <= 128) launch_tiles<T, 128>(a, wide, nt, s);
  else launch_tiles<T, 256>(a, wide, nt, s);
}

}  // namespace

namespace kvc {
namespace attn {

void launch_q8(const AttendArgs& a, bool f16, bool wide, bool past_the_caches, hipStream_t s) {
  if (f16) launch_tiles<F16>(a, wide, past_the_caches, s);
  else launch_tiles<BF16>(a, wide, past_the_caches, s);
}

}  // namespace attn
}  // namespace kvc
