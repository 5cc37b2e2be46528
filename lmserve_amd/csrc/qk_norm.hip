// Norms of queries and keys, head by head, with the rotation and the K/V write in the same pass (gfx950).
//
// For a head x of Q or K with the weight w of its kind:
//   y = x w / sqrt(mean(x^2) + eps),   then the rotation of y's first rotary_dim lanes as the plain rotation does it;
// fp32 throughout, one rounding at the end. The rotated key and the value go straight to the token's cache slot.
// A workgroup belongs to one token. A head is a group of lanes (a power of two, so that groups do not cross wavefronts);
// a lane holds both halves of its rotation pairs, 16 bytes each, so that norm and rotation need nothing of each other's lanes
// but the sum of squares, a few DPP steps within the group. V heads ride along as copies.

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "common.h"
#include "device.h"
#include "kvcache.h"

namespace {

using kvc::fail;
using kvc::log2_exact;
using kvc::u32x4;

// ---- storage types: 16 bytes to and from fp32 ------------------------------------------------------------------------
struct BF16 {
  typedef uint16_t Word;
  static constexpr int kBytes = 2;
  static __device__ __forceinline__ float wide(Word w) { return __uint_as_float((uint32_t)w << 16); }
  static __device__ __forceinline__ Word narrow(float f) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  }
};
struct F16 {
  typedef uint16_t Word;
  static constexpr int kBytes = 2;
  static __device__ __forceinline__ float wide(Word w) { return __half2float(__ushort_as_half(w)); }
  static __device__ __forceinline__ Word narrow(float f) { return __half_as_ushort(__float2half_rn(f)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return (uint32_t)narrow(lo) | (uint32_t)narrow(hi) << 16; }
};
struct F32 {
  typedef uint32_t Word;
  static constexpr int kBytes = 4;
  static __device__ __forceinline__ float wide(Word w) { return __uint_as_float(w); }
  static __device__ __forceinline__ Word narrow(float f) { return __float_as_uint(f); }
};
template <typename T>
struct Vec {
  static constexpr int kN = 16 / T::kBytes;
  static __device__ __forceinline__ void widen(u32x4 v, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kN == 8) {
        f[2 * i] = T::wide((uint16_t)(v[i] & 0xffffu));
        f[2 * i + 1] = T::wide((uint16_t)(v[i] >> 16));
      } else {
        f[i] = __uint_as_float(v[i]);
      }
    }
  }
  static __device__ __forceinline__ u32x4 narrow(const float* f) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kN == 8) v[i] = T::pack(f[2 * i], f[2 * i + 1]);
      else v[i] = __float_as_uint(f[i]);
    }
    return v;
  }
};

struct NormArgs {
  const char *query, *key, *value;
  const char *q_weight, *k_weight;
  char *query_out, *key_out;  // key_out may be null when a cache takes the key
  const void* positions;
  const char* cos_sin_cache;
  int64_t max_position;
  char *key_cache, *value_cache;  // null: no cache
  const void* slot_mapping;
  const int32_t *batch_indices, *kv_indices, *kv_indptr;  // batch_indices non-null: page-table addressing
  int64_t batch_size, num_kv_indices;
  int64_t block_size, cache_block_stride, cache_slot_stride, num_cache_blocks;  // strides in bytes
  int64_t q_token_stride, k_token_stride, v_token_stride, qo_token_stride, ko_token_stride;  // bytes
  float eps, inv_dim;
  int32_t num_heads, num_kv_heads, head_dim, rotary_dim;
  int32_t pairs, vecs;  // 16-byte vectors: of one half of the rotation, of a head
  int32_t pos_bytes, slot_bytes, bs_shift;
};

enum Addressing : int { kNoCache, kSlots, kPages };

__device__ __forceinline__ int64_t entry_of(const void* array, int bytes, int64_t t) {
  return bytes == 4 ? (int64_t) reinterpret_cast<const int32_t*>(array)[t] : reinterpret_cast<const int64_t*>(array)[t];
}

// Byte offset of the token's slot in a cache plane, or -1 where the write skips the token. The same for all lanes.
template <Addressing ADDR, bool FAST>
__device__ __forceinline__ int64_t slot_offset(const NormArgs& a, int64_t t, int64_t pos) {
  if constexpr (ADDR == kNoCache) return -1;
  int64_t block = -1, off = 0;
  if constexpr (ADDR == kPages) {
    const int64_t b = a.batch_indices[t];
    const bool known = b >= 0 && b < a.batch_size;
    const int64_t at = known ? b : 0, begin = a.kv_indptr[at], end = a.kv_indptr[at + 1];
    const int64_t page = FAST ? pos >> a.bs_shift : pos / a.block_size;
    off = pos - page * a.block_size;
    const int64_t i = begin + page;
    const bool ok = known && i >= 0 && i < end && i < a.num_kv_indices;
    const int64_t id = a.kv_indices[ok ? i : 0];
    if (ok) block = id;
  } else {
    const int64_t s = FAST ? reinterpret_cast<const int64_t*>(a.slot_mapping)[t] : entry_of(a.slot_mapping, a.slot_bytes, t);
    if (s >= 0) {
      block = FAST ? s >> a.bs_shift : s / a.block_size;
      off = s - block * a.block_size;
    }
  }
  if (block < 0 || block >= a.num_cache_blocks) return -1;
  return block * a.cache_block_stride + off * a.cache_slot_stride;
}

// The sum over groups of W lanes, the same bits in all of them
template <int CTRL>
__device__ __forceinline__ float plus_dpp(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int W>
__device__ __forceinline__ float group_sum(float x) {
  if constexpr (W >= 2) x = plus_dpp<0xb1>(x);    // quad_perm 1,0,3,2
  if constexpr (W >= 4) x = plus_dpp<0x4e>(x);    // quad_perm 2,3,0,1
  if constexpr (W >= 8) x = plus_dpp<0x141>(x);   // row_half_mirror
  if constexpr (W >= 16) x = plus_dpp<0x140>(x);  // row_mirror
  if constexpr (W >= 32) x += __shfl_xor(x, 16);
  if constexpr (W >= 64) x += __shfl_xor(x, 32);
  return x;
}

typedef u32x4 __attribute__((aligned(2))) u32x4_at_any_element;  // a table or weight that is a view
__device__ __forceinline__ u32x4 ld16_any(const char* p) { return *reinterpret_cast<const u32x4_at_any_element*>(p); }

// Rows of aligned 16-byte vectors. W lanes to a head.
// Bound by HBM where tokens are many: 16384 of (32 + 2 x 8) heads of 128 in bf16, 0.71 GB, take 119 us (5.95 TB/s); few of them
// by the launch and loads one behind the other, position, then cos/sin: one token 2.6 us, 256 tokens 3.8.
template <typename T, Addressing ADDR, bool FAST, int W, bool PAST>
__global__ __launch_bounds__(256) void norm_rotate_kernel(NormArgs a) {
  constexpr int N = Vec<T>::kN, E = T::kBytes;
  const int64_t t = blockIdx.x;
  const int32_t lane = blockIdx.y * blockDim.x + threadIdx.x;
  const int32_t h = lane / W, j = lane % W;
  const int32_t hq = a.num_heads, hk = hq + a.num_kv_heads, heads = ADDR == kNoCache ? hk : hk + a.num_kv_heads;
  const int64_t pos = FAST ? (int64_t) reinterpret_cast<const int32_t*>(a.positions)[t] : entry_of(a.positions, a.pos_bytes, t);
  const bool is_q = h < hq, is_v = h >= hk;
  const bool turns = j < a.pairs;
  const int32_t v0 = turns ? j : 2 * j, v1 = turns ? j + a.pairs : v0 + 1;  // (2 pairs + 2 (j - pairs) = 2 j)
  const bool some = h < heads && v0 < a.vecs, both = h < heads && v1 < a.vecs;
  const int64_t head_off = (int64_t)(h - (is_q ? 0 : is_v ? hk : hq)) * a.head_dim * E;
  const char* in = (is_q ? a.query + t * a.q_token_stride : is_v ? a.value + t * a.v_token_stride : a.key + t * a.k_token_stride) + head_off;
  u32x4 x0 = {}, x1 = {};
  if (some) x0 = *reinterpret_cast<const u32x4*>(in + v0 * 16);
  if (both) x1 = *reinterpret_cast<const u32x4*>(in + v1 * 16);
  if (pos < 0 || pos >= a.max_position) return;  // no cos/sin row: the token is left alone
  const char* weight = is_q ? a.q_weight : a.k_weight;
  u32x4 w0 = {}, w1 = {}, c0 = {}, c1 = {}, s0 = {}, s1 = {};
  if (!is_v) {
    if (some) w0 = ld16_any(weight + v0 * 16);
    if (both) w1 = ld16_any(weight + v1 * 16);
    if (turns) {
      const char* row = a.cos_sin_cache + pos * (2 * a.rotary_dim * E);
      c0 = ld16_any(row + v0 * 16);
      c1 = ld16_any(row + v1 * 16);
      s0 = ld16_any(row + a.rotary_dim * E + v0 * 16);
      s1 = ld16_any(row + a.rotary_dim * E + v1 * 16);
    }
  }
  const int64_t slot = slot_offset<ADDR, FAST>(a, t, pos);
  float x[2][N];
  Vec<T>::widen(x0, x[0]);
  Vec<T>::widen(x1, x[1]);
  float sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) sum += x[0][i] * x[0][i] + x[1][i] * x[1][i];
  sum = group_sum<W>(sum);
  if (!some) return;
  if (!is_v) {
    const float r = 1.f / sqrtf(sum * a.inv_dim + a.eps);
    float w[2][N], c[2][N], s[2][N];
    Vec<T>::widen(w0, w[0]);
    Vec<T>::widen(w1, w[1]);
    Vec<T>::widen(c0, c[0]);
    Vec<T>::widen(c1, c[1]);
    Vec<T>::widen(s0, s[0]);
    Vec<T>::widen(s1, s[1]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y0 = x[0][i] * r * w[0][i], y1 = x[1][i] * r * w[1][i];
      x[0][i] = turns ? __builtin_fmaf(y0, c[0][i], -(y1 * s[0][i])) : y0;
      x[1][i] = turns ? __builtin_fmaf(y1, c[1][i], y0 * s[1][i]) : y1;
    }
    x0 = Vec<T>::narrow(x[0]);
    x1 = Vec<T>::narrow(x[1]);
  }
  const auto put = [&](char* row) {
    u32x4 *to0 = reinterpret_cast<u32x4*>(row + head_off + v0 * 16), *to1 = reinterpret_cast<u32x4*>(row + head_off + v1 * 16);
    if constexpr (PAST) {
      __builtin_nontemporal_store(x0, to0);
      if (both) __builtin_nontemporal_store(x1, to1);
    } else {
      *to0 = x0;
      if (both) *to1 = x1;
    }
  };
  if (is_q) put(a.query_out + t * a.qo_token_stride);
  else if (!is_v && a.key_out) put(a.key_out + t * a.ko_token_stride);
  if (ADDR != kNoCache && !is_q && slot >= 0) put((is_v ? a.value_cache : a.key_cache) + slot);
}

// All other rows (odd heads, unaligned rows): a wavefront to a head, an element or a pair to a lane at a time, read once for the sum and again, from
// the first-level cache, for the product. A lane reads again only what it alone writes, so that the output may be the input.
template <typename T, Addressing ADDR>
__global__ __launch_bounds__(256) void norm_rotate_element_kernel(NormArgs a) {
  typedef typename T::Word Word;
  constexpr int E = T::kBytes;
  const int64_t t = blockIdx.x;
  const int32_t lane = threadIdx.x & 63, h = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int32_t hq = a.num_heads, hk = hq + a.num_kv_heads, heads = ADDR == kNoCache ? hk : hk + a.num_kv_heads;
  const int64_t pos = entry_of(a.positions, a.pos_bytes, t);
  if (h >= heads || pos < 0 || pos >= a.max_position) return;
  const int64_t slot = slot_offset<ADDR, false>(a, t, pos);
  const bool is_q = h < hq, is_v = h >= hk;
  const int64_t head_off = (int64_t)(h - (is_q ? 0 : is_v ? hk : hq)) * a.head_dim * E;
  const Word* in = reinterpret_cast<const Word*>(
      (is_q ? a.query + t * a.q_token_stride : is_v ? a.value + t * a.v_token_stride : a.key + t * a.k_token_stride) + head_off);
  const Word* weight = reinterpret_cast<const Word*>(is_q ? a.q_weight : a.k_weight);
  const Word* cos = reinterpret_cast<const Word*>(a.cos_sin_cache + pos * (2 * (int64_t)a.rotary_dim * E));
  const Word* sin = cos + a.rotary_dim;
  char* row = is_v ? nullptr : is_q ? a.query_out + t * a.qo_token_stride : a.key_out ? a.key_out + t * a.ko_token_stride : nullptr;
  Word* out = reinterpret_cast<Word*>(row ? row + head_off : nullptr);
  Word* cached = ADDR != kNoCache && !is_q && slot >= 0
                     ? reinterpret_cast<Word*>((is_v ? a.value_cache : a.key_cache) + slot + head_off) : nullptr;
  const auto put = [&](int32_t i, Word w) {
    if (out) out[i] = w;
    if (cached) cached[i] = w;
  };
  if (is_v) {
    for (int32_t i = lane; i < a.head_dim; i += 64) put(i, in[i]);
    return;
  }
  float sum = 0;
  for (int32_t i = lane; i < a.head_dim; i += 64) {
    const float x = T::wide(in[i]);
    sum += x * x;
  }
  const float r = 1.f / sqrtf(group_sum<64>(sum) * a.inv_dim + a.eps);
  const int32_t half = a.rotary_dim / 2;
  for (int32_t i = lane; i < a.head_dim - half; i += 64) {
    if (i < half) {
      const float y0 = T::wide(in[i]) * r * T::wide(weight[i]);
      const float y1 = T::wide(in[i + half]) * r * T::wide(weight[i + half]);
      put(i, T::narrow(__builtin_fmaf(y0, T::wide(cos[i]), -(y1 * T::wide(sin[i])))));
      put(i + half, T::narrow(__builtin_fmaf(y1, T::wide(cos[i + half]), y0 * T::wide(sin[i + half]))));
    } else {
      const int32_t e = i + half;
      put(e, T::narrow(T::wide(in[e]) * r * T::wide(weight[e])));
    }
  }
}

template <typename T, Addressing ADDR, bool FAST, bool PAST>
void launch_vector(const NormArgs& a, int lanes, dim3 grid, dim3 block, hipStream_t s) {
  switch (lanes) {
    case 1: kvc::launch((norm_rotate_kernel<T, ADDR, FAST, 1, PAST>), grid, block, 0, s, a); break;
    case 2: kvc::launch((norm_rotate_kernel<T, ADDR, FAST, 2, PAST>), grid, block, 0, s, a); break;
    case 4: kvc::launch((norm_rotate_kernel<T, ADDR, FAST, 4, PAST>), grid, block, 0, s, a); break;
    case 8: kvc::launch((norm_rotate_kernel<T, ADDR, FAST, 8, PAST>), grid, block, 0, s, a); break;
    case 16: kvc::launch((norm_rotate_kernel<T, ADDR, FAST, 16, PAST>), grid, block, 0, s, a); break;
    case 32: kvc::launch((norm_rotate_kernel<T, ADDR, FAST, 32, PAST>), grid, block, 0, s, a); break;
    default: kvc::launch((norm_rotate_kernel<T, ADDR, FAST, 64, PAST>), grid, block, 0, s, a); break;
  }
}

template <typename T, Addressing ADDR>
void launch_norm(const NormArgs& a, bool vector, int64_t tokens, hipStream_t s) {
  const int heads = a.num_heads + (ADDR == kNoCache ? 1 : 2) * a.num_kv_heads;
  if (!vector) {
    kvc::launch((norm_rotate_element_kernel<T, ADDR>), dim3((unsigned)tokens, (unsigned)((heads + 3) / 4)), dim3(256), 0, s, a);
    return;
  }
  // Outputs past the caches where the last-level one would not hold them till they are read, and where they are few (what is
  // written ends the launch later than the stores do). With the attention that reads them behind it, a layer of 32 + 2 x 8
  // heads of 128 takes, plain and past the caches: 256 tokens (3 MB) 135 and 132 us, 2048 (25 MB) 46.6 and 47.3, 8192 (101 MB) 162
  // and 169, 16384 (201 MB) 328 and 330; the launch by itself 2048 tokens 9.7 and 8.1, 16384 134 and 119 (loads too: 119).
  const int64_t written = tokens * heads * a.head_dim * T::kBytes;
  const bool past = written < (int64_t(8) << 20) || written >= (int64_t(128) << 20);
  int lanes = 1;
  while (2 * lanes < a.vecs) lanes *= 2;
  const int64_t all = (int64_t)heads * lanes;
  // (a token's heads in one workgroup of up to 1024: 2048 tokens 8.9 us for 8.2, 256 tokens and one 0.1 us less)
  const unsigned threads = (unsigned)std::min<int64_t>(256, (all + 63) / 64 * 64);
  const dim3 grid((unsigned)tokens, (unsigned)((all + threads - 1) / threads)), block(threads);
  const bool fast = a.pos_bytes == 4 && (ADDR == kNoCache || a.bs_shift >= 0) && (ADDR != kSlots || a.slot_bytes == 8);
  if (!fast) launch_vector<T, ADDR, false, false>(a, lanes, grid, block, s);
  else if (past) launch_vector<T, ADDR, true, true>(a, lanes, grid, block, s);
  else launch_vector<T, ADDR, true, false>(a, lanes, grid, block, s);
}

template <typename T>
void launch_norm(const NormArgs& a, bool vector, int64_t tokens, hipStream_t s) {
  if (!a.key_cache) launch_norm<T, kNoCache>(a, vector, tokens, s);
  else if (a.batch_indices) launch_norm<T, kPages>(a, vector, tokens, s);
  else launch_norm<T, kSlots>(a, vector, tokens, s);
}

struct Rows {  // of one tensor: bytes
  const char* p;
  int64_t stride, row;
};
// May `out` be written while `in` is read? Where they lie apart, where they are the same rows (`same`: of one kind, a lane
// owns what it reads), or where they are different columns of one matrix.
bool may_write(const Rows& out, const Rows& in, int64_t tokens, bool same) {
  if (!out.p || !in.p) return true;
  const __int128 o = (uintptr_t)out.p, i = (uintptr_t)in.p;
  if (o >= i + (__int128)(tokens - 1) * in.stride + in.row || i >= o + (__int128)(tokens - 1) * out.stride + out.row) return true;
  if (out.stride != in.stride && tokens > 1) return false;
  if (o == i) return same;
  const int64_t stride = tokens > 1 ? out.stride : int64_t(1) << 60;
  const int64_t apart = (int64_t)(o > i ? (o - i) % stride : stride - (i - o) % stride);
  return apart >= in.row && apart + out.row <= stride;
}

struct Cache {
  void *key_cache, *value_cache;
  const void* slot_mapping;
  int slot_bytes;
  const int32_t *batch_indices, *kv_indices, *kv_indptr;
  int64_t batch_size, num_kv_indices, block_size, cache_block_stride, cache_slot_stride, num_cache_blocks;  // elements
};

int run_norm(const char* fn, const void* query, const void* key, const void* value, const void* q_weight, const void* k_weight,
             float eps, void* query_out, void* key_out, const void* positions, int pos_bytes, const void* cos_sin_cache,
             int64_t max_position, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim,
             int64_t q_ts, int64_t k_ts, int64_t v_ts, int64_t qo_ts, int64_t ko_ts, int dtype, const Cache* c, void* stream) {
  if (dtype != KVC_DTYPE_BF16 && dtype != KVC_DTYPE_F16 && dtype != KVC_DTYPE_F32)
    return fail(KVC_ERR_UNSUPPORTED, "%s: dtype %d (need bf16, f16 or f32)", fn, dtype);
  const int E = dtype == KVC_DTYPE_F32 ? 4 : 2;
  if (tokens < 0 || heads < 0 || kv_heads < 0 || head_dim <= 0 || rotary_dim < 0 || max_position < 0)
    return fail(KVC_ERR_INVALID_ARG, "%s: negative size", fn);
  if (rotary_dim > head_dim || (rotary_dim & 1))
    return fail(KVC_ERR_INVALID_ARG, "%s: rotary_dim %lld must be even and <= head_dim %lld", fn, (long long)rotary_dim,
                (long long)head_dim);
  if (!(eps > 0) || !std::isfinite(eps)) return fail(KVC_ERR_INVALID_ARG, "%s: eps must be positive and finite", fn);
  if (pos_bytes != 4 && pos_bytes != 8) return fail(KVC_ERR_UNSUPPORTED, "%s: pos_bytes=%d (need 4 or 8)", fn, pos_bytes);
  if (tokens > 0x7fffffffll || heads + 2 * kv_heads > 0xffffll || head_dim > 0xffffll)
    return fail(KVC_ERR_UNSUPPORTED, "%s: too many tokens or heads, or heads too wide", fn);
  if (tokens == 0 || heads + kv_heads == 0) return KVC_OK;
  if (!query || !key || !query_out || !positions || (!cos_sin_cache && rotary_dim) || !q_weight || !k_weight)
    return fail(KVC_ERR_INVALID_ARG, "%s: null pointer", fn);
  if (!c && !key_out) return fail(KVC_ERR_INVALID_ARG, "%s: no destination for the key", fn);
  const int64_t q_row = heads * head_dim, k_row = kv_heads * head_dim;
  if (q_ts < q_row || qo_ts < q_row || k_ts < k_row || (key_out && ko_ts < k_row))
    return fail(KVC_ERR_INVALID_ARG, "%s: token stride smaller than a row", fn);
  NormArgs a{};
  a.query = (const char*)query;
  a.key = (const char*)key;
  a.value = (const char*)value;
  a.q_weight = (const char*)q_weight;
  a.k_weight = (const char*)k_weight;
  a.query_out = (char*)query_out;
  a.key_out = (char*)key_out;
  a.positions = positions;
  a.cos_sin_cache = (const char*)cos_sin_cache;
  a.max_position = max_position;
  a.q_token_stride = q_ts * E;
  a.k_token_stride = k_ts * E;
  a.v_token_stride = v_ts * E;
  a.qo_token_stride = qo_ts * E;
  a.ko_token_stride = ko_ts * E;
  a.eps = eps;
  a.inv_dim = 1.f / (float)head_dim;
  a.num_heads = (int32_t)heads;
  a.num_kv_heads = (int32_t)kv_heads;
  a.head_dim = (int32_t)head_dim;
  a.rotary_dim = (int32_t)rotary_dim;
  a.pos_bytes = pos_bytes;
  uint64_t align = (uintptr_t)query | (uintptr_t)key | (uintptr_t)query_out | (uintptr_t)key_out | (uint64_t)a.q_token_stride |
                   (uint64_t)a.k_token_stride | (uint64_t)a.qo_token_stride | (uint64_t)(key_out ? a.ko_token_stride : 0);
  const Rows in_q{a.query, a.q_token_stride, q_row * E}, in_k{a.key, a.k_token_stride, k_row * E},
      in_v{c ? a.value : nullptr, a.v_token_stride, k_row * E}, out_q{a.query_out, a.qo_token_stride, q_row * E},
      out_k{a.key_out, a.ko_token_stride, k_row * E};
  bool apart = may_write(out_q, in_q, tokens, true) && may_write(out_q, in_k, tokens, false) && may_write(out_q, in_v, tokens, false) &&
               may_write(out_k, in_q, tokens, false) && may_write(out_k, in_k, tokens, true) && may_write(out_k, in_v, tokens, false) &&
               may_write(out_k, out_q, tokens, false);
  if (c) {
    if (!value || !c->key_cache || !c->value_cache) return fail(KVC_ERR_INVALID_ARG, "%s: null value/cache pointer", fn);
    if (v_ts < k_row) return fail(KVC_ERR_INVALID_ARG, "%s: value token stride smaller than a row", fn);
    if (c->block_size <= 0 || c->num_cache_blocks < 0 || c->cache_block_stride < 0 || c->cache_slot_stride < k_row)
      return fail(KVC_ERR_INVALID_ARG, "%s: bad cache geometry", fn);
    if (c->batch_indices) {
      if (!c->kv_indices || !c->kv_indptr || c->batch_size < 0 || c->num_kv_indices < 0)
        return fail(KVC_ERR_INVALID_ARG, "%s: bad page-table arguments", fn);
      if (pos_bytes != 4) return fail(KVC_ERR_UNSUPPORTED, "%s: page-table addressing takes int32 positions", fn);
    } else {
      if (!c->slot_mapping) return fail(KVC_ERR_INVALID_ARG, "%s: null slot_mapping", fn);
      if (c->slot_bytes != 4 && c->slot_bytes != 8)
        return fail(KVC_ERR_UNSUPPORTED, "%s: slot_bytes=%d (need 4 or 8)", fn, c->slot_bytes);
    }
    a.key_cache = (char*)c->key_cache;
    a.value_cache = (char*)c->value_cache;
    a.slot_mapping = c->slot_mapping;
    a.slot_bytes = c->slot_bytes;
    a.batch_indices = c->batch_indices;
    a.kv_indices = c->kv_indices;
    a.kv_indptr = c->kv_indptr;
    a.batch_size = c->batch_size;
    a.num_kv_indices = c->num_kv_indices;
    a.block_size = c->block_size;
    a.bs_shift = log2_exact(c->block_size);
    a.cache_block_stride = c->cache_block_stride * E;
    a.cache_slot_stride = c->cache_slot_stride * E;
    a.num_cache_blocks = c->num_cache_blocks;
    align |= (uintptr_t)value | (uint64_t)a.v_token_stride | (uintptr_t)c->key_cache | (uintptr_t)c->value_cache |
             (uint64_t)a.cache_block_stride | (uint64_t)a.cache_slot_stride;
    if (c->num_cache_blocks > 0)
      for (const char* plane : {a.key_cache, a.value_cache}) {
        const __int128 end = (__int128)(c->num_cache_blocks - 1) * a.cache_block_stride + (__int128)(c->block_size - 1) * a.cache_slot_stride + k_row * E;
        for (const Rows& r : {in_q, in_k, in_v, out_q, out_k}) {
          const __int128 p = (uintptr_t)plane, x = (uintptr_t)r.p;
          if (r.p && x < p + end && p < x + (__int128)(tokens - 1) * r.stride + r.row) apart = false;
        }
      }
    if (c->batch_indices && (c->batch_size == 0 || c->num_kv_indices == 0)) a.key_cache = nullptr;  // every token is skipped
  }
  // nor may what is written, rows and cache planes, share memory with the arrays beside the rows
  const auto span = [&](const Rows& r) { return r.p ? (__int128)(tokens - 1) * r.stride + r.row : (__int128)0; };
  const __int128 plane = c && c->num_cache_blocks > 0
                             ? (__int128)(c->num_cache_blocks - 1) * a.cache_block_stride + (__int128)(c->block_size - 1) * a.cache_slot_stride + k_row * E
                             : (__int128)0;
  struct Memory {
    const void* p;
    __int128 bytes;
  };
  const Memory written[] = {{a.query_out, span(out_q)}, {a.key_out, span(out_k)}, {c ? c->key_cache : nullptr, plane}, {c ? c->value_cache : nullptr, plane}};
  const Memory arrays[] = {{q_weight, head_dim * E}, {k_weight, head_dim * E}, {positions, tokens * pos_bytes},
                           {cos_sin_cache, (__int128)max_position * 2 * rotary_dim * E},
                           {c ? c->slot_mapping : nullptr, c ? tokens * c->slot_bytes : 0}, {c ? c->batch_indices : nullptr, tokens * 4},
                           {c ? c->kv_indices : nullptr, c ? (__int128)c->num_kv_indices * 4 : 0}, {c ? c->kv_indptr : nullptr, c ? (__int128)(c->batch_size + 1) * 4 : 0}};
  for (const Memory& w : written)
    for (const Memory& r : arrays)
      if (w.p && r.p && (uintptr_t)w.p < (uintptr_t)r.p + r.bytes && (uintptr_t)r.p < (uintptr_t)w.p + w.bytes) apart = false;
  if (!apart)
    return fail(KVC_ERR_INVALID_ARG, "%s: an output overlaps an input or another output (only a whole output on its own input's rows may)", fn);
  const int n = 16 / E;
  const bool vector = align % 16 == 0 && (rotary_dim / 2) % n == 0 && (head_dim - rotary_dim) % n == 0 && head_dim % n == 0 &&
                      head_dim / n <= 128 && head_dim > 0;
  a.pairs = (int32_t)(rotary_dim / 2 / n);
  a.vecs = (int32_t)(head_dim / n);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == KVC_DTYPE_BF16) launch_norm<BF16>(a, vector, tokens, s);
  else if (dtype == KVC_DTYPE_F16) launch_norm<F16>(a, vector, tokens, s);
  else launch_norm<F32>(a, vector, tokens, s);
  KVC_HIP(hipGetLastError());
  return KVC_OK;
}

}  // namespace

extern "C" {

int kvc_qk_norm_rotary_pos_emb(const void* query, const void* key, const void* query_weight, const void* key_weight, float eps,
                               const void* positions, int pos_bytes, const void* cos_sin_cache, int64_t max_position,
                               int64_t num_tokens, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t rotary_dim,
                               int64_t q_token_stride, int64_t k_token_stride, void* query_out, void* key_out,
                               int64_t qo_token_stride, int64_t ko_token_stride, int dtype, void* stream) {
  return run_norm("kvc_qk_norm_rotary_pos_emb", query, key, nullptr, query_weight, key_weight, eps, query_out, key_out, positions,
                  pos_bytes, cos_sin_cache, max_position, num_tokens, num_heads, num_kv_heads, head_dim, rotary_dim,
                  q_token_stride, k_token_stride, 0, qo_token_stride, ko_token_stride, dtype, nullptr, stream);
}

int kvc_qk_norm_rotary_pos_emb_and_cache(const void* query, const void* key, const void* value, const void* query_weight,
                                         const void* key_weight, float eps, const void* positions, int pos_bytes,
                                         const void* cos_sin_cache, int64_t max_position, int64_t num_tokens, int64_t num_heads,
                                         int64_t num_kv_heads, int64_t head_dim, int64_t rotary_dim, int64_t q_token_stride,
                                         int64_t k_token_stride, int64_t v_token_stride, void* query_out, void* key_out,
                                         int64_t qo_token_stride, int64_t ko_token_stride, void* key_cache, void* value_cache,
                                         const void* slot_mapping, int slot_bytes, int64_t block_size, int64_t cache_block_stride,
                                         int64_t cache_slot_stride, int64_t num_cache_blocks, int dtype, void* stream) {
  const Cache c{key_cache, value_cache, slot_mapping, slot_bytes, nullptr, nullptr, nullptr, 0, 0,
                block_size, cache_block_stride, cache_slot_stride, num_cache_blocks};
  return run_norm("kvc_qk_norm_rotary_pos_emb_and_cache", query, key, value, query_weight, key_weight, eps, query_out, key_out,
                  positions, pos_bytes, cos_sin_cache, max_position, num_tokens, num_heads, num_kv_heads, head_dim, rotary_dim,
                  q_token_stride, k_token_stride, v_token_stride, qo_token_stride, ko_token_stride, dtype, &c, stream);
}

int kvc_qk_norm_rotary_pos_emb_and_append_paged(const void* query, const void* key, const void* value, const void* query_weight,
                                                const void* key_weight, float eps, const int32_t* batch_indices,
                                                const int32_t* positions, const void* cos_sin_cache, int64_t max_position,
                                                int64_t nnz, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                                                int64_t rotary_dim, int64_t q_token_stride, int64_t k_token_stride,
                                                int64_t v_token_stride, void* query_out, void* key_out, int64_t qo_token_stride,
                                                int64_t ko_token_stride, void* paged_kv_cache, const int32_t* kv_indices,
                                                const int32_t* kv_indptr, int64_t batch_size, int64_t num_kv_indices,
                                                int64_t page_size, int64_t page_stride, int64_t num_pages, int dtype, void* stream) {
  constexpr const char* fn = "kvc_qk_norm_rotary_pos_emb_and_append_paged";
  if (nnz > 0 && !batch_indices) return fail(KVC_ERR_INVALID_ARG, "%s: null batch_indices", fn);
  if (num_kv_heads < 0 || head_dim <= 0 || page_size <= 0) return fail(KVC_ERR_INVALID_ARG, "%s: bad H/D/page_size", fn);
  const int64_t row = num_kv_heads * head_dim;
  if (page_stride < 2 * page_size * row)
    return fail(KVC_ERR_INVALID_ARG, "%s: page_stride %lld < 2*page_size*H*D", fn, (long long)page_stride);
  const int E = dtype == KVC_DTYPE_F32 ? 4 : 2;
  const Cache c{paged_kv_cache, paged_kv_cache ? (char*)paged_kv_cache + page_size * row * E : nullptr, nullptr, 0,
                batch_indices, kv_indices, kv_indptr, batch_size, num_kv_indices, page_size, page_stride, row, num_pages};
  return run_norm(fn, query, key, value, query_weight, key_weight, eps, query_out, key_out, positions, 4, cos_sin_cache,
                  max_position, nnz, num_heads, num_kv_heads, head_dim, rotary_dim, q_token_stride, k_token_stride,
                  v_token_stride, qo_token_stride, ko_token_stride, dtype, &c, stream);
}

}  // extern "C"
