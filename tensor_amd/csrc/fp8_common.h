// Device-side building blocks of the norm and the 8-bit operators (gfx950, wave64).
//
// 8 bits are e4m3: a sign, four bits of exponent with bias 7, three of fraction, no infinities, NaN at 0x7F and 0xFF,
// values up to 448.  A block of 128 columns of a row shares a scale s = max(a / 448, 2^-126), a the largest
// magnitude of its finite values, and holds the codes nearest to the fp32 quotient value / s, ties to the even one; what is
// not finite has the NaN code, so that whatever is summed with it is NaN, as it would be without the codes.
#pragma once

#include "gguf_common.h"
#include "fp8_launch.h"

namespace tensor_fp8 {

using tensor_gguf::float4_t;
using tensor_gguf::half8_t;
typedef float float8_t __attribute__((ext_vector_type(8)));

constexpr float kLargest = 448.0f;
constexpr float kSmallestScale = 0x1p-126f;
constexpr float kInfinity = __builtin_inff();

// A row in chunks of 8 columns, one for a lane.  The last chunk of a row whose width is no multiple of 8 begins where
// eight columns are left, and its first `skip` values are the chunk's before it; past the row, skip is 8 or more.
// (Loads so stay one instruction each, whatever the width; rows then have any alignment, which they take.)
struct Chunk {
  int at, skip, count;  // first column loaded, values to leave out, values there
  __device__ __forceinline__ Chunk(int column, int width) {
    at = max(min(column, width - 8), 0);
    skip = column - at;
    count = min(width, 8);
  }
  __device__ __forceinline__ bool has(int e) const { return e >= skip && e < count; }
  __device__ __forceinline__ bool whole() const { return skip == 0 && count == 8; }
};

template <typename T>
__device__ __forceinline__ float8_t load8(const T* p, int count) {
  typedef T Values __attribute__((ext_vector_type(8)));
  Values v;
  if (count == 8) {
    __builtin_memcpy(&v, p, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = p[min(e, count - 1)];
  }
  return __builtin_convertvector(v, float8_t);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, float8_t v, const Chunk& chunk) {
  typedef T Values __attribute__((ext_vector_type(8)));
  const Values to = __builtin_convertvector(v, Values);
  if (chunk.whole()) {
    __builtin_memcpy(p, &to, sizeof(to));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (chunk.has(e)) p[e] = to[e];
  }
}

// A block's scale from this lane's 8 values of it; the block is 16 lanes next to each other.
__device__ __forceinline__ float block_scale(float8_t v, const Chunk& chunk) {
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float size = fabsf(v[e]);
    if (chunk.has(e) && size < kInfinity) top = fmaxf(top, size);
  }
#pragma unroll
  for (int step = 8; step > 0; step >>= 1) top = fmaxf(top, __shfl_xor(top, step));
  return fmaxf(top / kLargest, kSmallestScale);
}

// v / scale as codes, stored.  q = v (1 / scale) is off by up to 1.5 units of its last place, which turns ties; what it leaves,
// q scale - v, is exact or a bit short, and taken back times 1 / scale it makes q the quotient but for an error of 2^-22 units.
// That shows only where the quotient is as near to the middle of two fp32 values, and in a code only where one of the
// two is a tie of codes: of all scales' and ties' fractions there are 255 such pairs of value and scale, and q is rounded rightly
// in each.  (What is left of the smallest values would pass below fp32: blocks of small scales are divided 2^64 up.)  An infinite
// value leaves infinity - infinity, which is the NaN that its code is.
__device__ __forceinline__ void store_codes(uint8_t* p, float8_t v, float scale, const Chunk& chunk) {
  if (scale < 0x1p-90f) {
    scale *= 0x1p64f;
    v *= 0x1p64f;
  }
  const float inverse = 1.0f / scale;
  uint32_t words[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    int word = 0;
    float q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float size = v[4 * half + e], near = size * inverse;
      q[e] = __builtin_fmaf(-__builtin_fmaf(near, scale, -size), inverse, near);
    }
    word = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], word, false);
    word = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], word, true);
    words[half] = (uint32_t)word;
  }
  if (chunk.whole()) {
    __builtin_memcpy(p, words, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (chunk.has(e)) p[e] = (uint8_t)(words[e / 4] >> (8 * (e % 4)));
  }
}

}  // namespace tensor_fp8
