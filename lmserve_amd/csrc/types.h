// Vectors and the 16-bit storage types of the kernels that compute.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "device.h"

namespace kvc {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

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
  // e4m3 codes, two at a time, from and to the lower or upper half of a word: times, and divided by, a power of two, rounded once. (An infinity becomes NaN.)
  template <bool UPPER>
  static __device__ __forceinline__ uint32_t from_codes(uint32_t codes, float by) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, by, UPPER));
  }
  template <bool UPPER>
  static __device__ __forceinline__ uint32_t to_codes(uint32_t two, float scale, uint32_t old) {
    typedef short s2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(__builtin_bit_cast(s2, old), __builtin_bit_cast(b2, two), scale, UPPER));
  }
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
  template <bool UPPER>
  static __device__ __forceinline__ uint32_t from_codes(uint32_t codes, float by) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, by, UPPER));
  }
  template <bool UPPER>
  static __device__ __forceinline__ uint32_t to_codes(uint32_t two, float scale, uint32_t old) {
    typedef short s2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(__builtin_bit_cast(s2, old), __builtin_bit_cast(h2, two), scale, UPPER));
  }
  // the two numbers of a word, and x
  static __device__ __forceinline__ float sum(uint32_t two, float x) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, two), h2{1, 1}, x, false);
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
template <typename T>
__device__ __forceinline__ u32x4 finite_part(u32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = ((v[i] & T::kExponent) == T::kExponent ? 0 : v[i] & 0xffffu) | ((v[i] >> 16 & T::kExponent) == T::kExponent ? 0 : v[i] & 0xffff0000u);
  return v;
}

}  // namespace kvc
