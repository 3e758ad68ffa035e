// cache_types.h -- the elements of caches narrower than the tokens: e4m3, and 4 bits with a scale to 32 elements.
//
// In 4 bits (the microscaling format of the Open Compute Project): an element is a sign, two exponent bits and one of mantissa (0, 0.5, 1,
// 1.5, 2, 3, 4, 6), 32 neighbours along the depth share a scale 2^(byte - 127); byte 255 makes all of them NaN.  A page's rows of one head
// and side are one run of bytes: the codes [page, depth / 2], the first of two elements in the low bits, then the scales [page, depth / 32],
// so that the codes of a row are whole 16-byte vectors, one to a scale.
// The scale is the power of two two below the largest element's, doubled where that element's significand is over 1.75: then it lies
// within [3.5, 7] scales, and nothing is further from its code than half of the step that it lies in (without the doubling, elements
// between 7 and 8 scales would be off by up to 2 where the step is 2).  It is clamped to 2^-127 and 2^125 (2^13 for f16 tokens), so
// that 6 scales are a number of the tokens' type; what is beyond becomes the nearest end.
#pragma once

#include <type_traits>

#include "device_common.h"
#include "kernels.h"

namespace hyle_hip {

struct E4M3 {};
template <> struct Traits<E4M3> {
  static constexpr int kSize = 1;
  static __device__ __forceinline__ float load(const void *p, size_t i) {
    return __builtin_amdgcn_cvt_f32_fp8((int)static_cast<const uint8_t *>(p)[i], 0);
  }
};

// Nearest-even e4m3 of four values.  The converter gives NaN beyond its largest number, so those are brought to it first.
__device__ __forceinline__ float within_e4m3(float x) { return x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f); }
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(within_e4m3(a), within_e4m3(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(within_e4m3(c), within_e4m3(d), w, true);
}

struct MX4 {};
constexpr int kMx4Block = 32;  // elements to a scale

// A scale as f32.  (2^-127 is a subnormal number; byte 255, whose elements are NaN, is NaN.)
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
  return bits_f32(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}
__device__ __forceinline__ float mx4_level(uint32_t code) {
  const uint32_t size = code & 7u;
  const float v = size < 2 ? 0.5f * (float)size : bits_f32((126u + (size >> 1)) << 23 | (size & 1u) << 22);
  return (code & 8u) != 0 ? -v : v;
}
// Element i of a row by the addresses of its codes and scales.
__device__ __forceinline__ float mx4_element(const unsigned char *codes, const unsigned char *scales, int i) {
  return mx4_level((uint32_t)(codes[i >> 1] >> (4 * (i & 1))) & 15u) * mx4_scale(scales[i / kMx4Block]);
}
// The scale byte of a block by the bits of its largest magnitude: 255 where it holds an infinity or NaN.
template <class T> __device__ __forceinline__ uint32_t mx4_byte(uint32_t largest) {
  if (largest >= 0x7F800000u) return 255u;
  const int byte = (int)((largest + 0x1FFFFFu) >> 23) - 2;
  return (uint32_t)min(max(byte, 0), std::is_same<T, F16>::value ? 127 + 13 : 127 + 125);
}
// The reciprocal of a scale that mx4_byte gave, exact.
__device__ __forceinline__ float mx4_inverse(uint32_t byte) { return byte == 255 ? 1.0f : bits_f32((254u - byte) << 23); }
// Eight elements, divided by their scale, as codes: nearest, ties to the even code, beyond 6 the end.  (The converter has these rules; a
// scale of 1 leaves them alone.)
__device__ __forceinline__ uint32_t mx4_codes(const float (&x)[8]) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], 1.0f, 3);
}

// Eight elements of a lane, four neighbouring lanes of a quad to a block: their codes, and the block's scale byte.
template <class T> __device__ __forceinline__ uint32_t mx4_of_quad(const float (&x)[8], uint32_t *byte) {
  uint32_t largest = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) largest = max(largest, f32_bits(x[e]) & 0x7FFFFFFFu);
  largest = max(largest, (uint32_t)dpp_move<kDppSwap1>((int)largest));
  largest = max(largest, (uint32_t)dpp_move<kDppSwap2>((int)largest));
  *byte = mx4_byte<T>(largest);
  const float inverse = mx4_inverse(*byte);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = x[e] * inverse;
  return mx4_codes(y);
}
// A whole block by one thread, `load(e)` its elements, to bytes at any address.
template <class T, class Load> __device__ __forceinline__ void mx4_store_block(Load load, unsigned char *codes, unsigned char *scale) {
  uint32_t largest = 0;
  for (int e = 0; e < kMx4Block; ++e) largest = max(largest, f32_bits(load(e)) & 0x7FFFFFFFu);
  const uint32_t byte = mx4_byte<T>(largest);
  const float inverse = mx4_inverse(byte);
  for (int g = 0; g < kMx4Block / 8; ++g) {
    float y[8];
    for (int e = 0; e < 8; ++e) y[e] = load(8 * g + e) * inverse;
    const uint32_t w = mx4_codes(y);
    for (int k = 0; k < 4; ++k) codes[4 * g + k] = (unsigned char)(w >> (8 * k));
  }
  *scale = (unsigned char)byte;
}

}  // namespace hyle_hip
