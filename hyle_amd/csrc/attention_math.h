// attention_math.h -- matrix-unit operands, the packing of weights and the constants that the attention kernels share.
#pragma once

#include <type_traits>

#include "attention.h"

namespace hyle_hip {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kSlack = 8.0f;

template <class T> __device__ __forceinline__ f32x16 product(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (std::is_same<T, BF16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <class T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, BF16>::value) return pack_bf16x2(lo, hi);
  else {
    const f32x2 in = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(in, f16x2));
  }
}
// 4 rows of 16 elements each, a lane of 16 its column: rows at `lane % 16 / 4`, 8 bytes at `lane % 4`.
__device__ __forceinline__ uint2 read_transposed(const unsigned char *at) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at));
}

// Bits set where a vector holds an infinity or NaN.
template <class C> __device__ __forceinline__ uint32_t no_numbers(u32x4 words) {
  uint32_t found = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (std::is_same<C, E4M3>::value) {
      const uint32_t low = words[w] & 0x7F7F7F7Fu;  // NaN alone, all ones
      found |= (low + 0x01010101u) & 0x80808080u;
    } else {
      constexpr uint32_t kExponent = std::is_same<C, BF16>::value ? 0x7F80u : 0x7C00u;
      found |= (uint32_t)((words[w] & kExponent) == kExponent) | (uint32_t)(((words[w] >> 16) & kExponent) == kExponent);
    }
  }
  return found;
}
template <class C> __device__ __forceinline__ u32x4 numbers_only(u32x4 words) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (std::is_same<C, E4M3>::value) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (((words[w] >> (8 * e)) & 0x7Fu) == 0x7Fu) words[w] &= ~(0xFFu << (8 * e));
    } else {
      constexpr uint32_t kExponent = std::is_same<C, BF16>::value ? 0x7F80u : 0x7C00u;
      if ((words[w] & kExponent) == kExponent) words[w] &= 0xFFFF0000u;
      if (((words[w] >> 16) & kExponent) == kExponent) words[w] &= 0x0000FFFFu;
    }
  }
  return words;
}

}  // namespace hyle_hip
