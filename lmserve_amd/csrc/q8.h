// The 8-bit cache: groups of 16 tokens.
//
// A page is page_size / 16 groups. A group holds the codes (e4m3: 4 bits of exponent, 3 of mantissa) of K and V and their
// exponents, padded to whole 128 bytes, the lines of the caches:
//   K [head][token / 4][dim / 16][token % 4][dim % 16], V [head][dim][token], exponents [head][K, V] plus 127.
// Both are laid as the matrix instruction of the attention takes them, 16 bytes a lane: K as rows of 16 columns, V as columns
// of 16 tokens, so that no lane's codes have to be exchanged with another's, and the 4 groups that a wavefront takes at once lie
// in pieces of 256 bytes for every load.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "types.h"

namespace kvc {
namespace q8 {

constexpr int kGroup = 16;               // tokens of a group
constexpr int kBias = 127;               // of a stored exponent
// Exponents. With a score's scale from 2^-26 to 2^8 / log2(e) the product with 2^e is a normal fp32; the attention holds others to those.
constexpr int kLeast = -100, kMost = 120;

inline int64_t plane_bytes(int64_t heads, int64_t dim) { return kGroup * heads * dim; }
inline int64_t group_bytes(int64_t heads, int64_t dim) { return (2 * plane_bytes(heads, dim) + 2 * heads + 127) / 128 * 128; }

// 2^(stored - kBias) of a stored exponent of at least 1
__device__ __forceinline__ float power_of(uint32_t stored) { return __uint_as_float(stored << 23); }

// The stored form of the least exponent with which magnitudes up to `top` are at most 448 = 1.75 * 2^8
__device__ __forceinline__ int32_t exponent_of(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int32_t e = (int32_t)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return e < kLeast + kBias ? kLeast + kBias : e > kMost + kBias ? kMost + kBias : e;
}

// Where a code is NaN: bit 7 of its byte
__device__ __forceinline__ uint32_t nan_codes(uint32_t codes) { return ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// The bytes of those of 4 codes, from token `first` on, that are among tokens [0, n)
__device__ __forceinline__ uint32_t bytes_below(int32_t n, int32_t first) {
  const int32_t left = n - first;
  return left <= 0 ? 0u : left >= 4 ? ~0u : (1u << left * 8) - 1u;
}

}  // namespace q8
}  // namespace kvc
