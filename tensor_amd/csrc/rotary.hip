// Rotary positions of queries and keys, with or without the store of keys and values into a paged
// cache, one launch:
//   (a, b) -> (a c - b s, b c + a s), c and s the cosine and sine of the token's position times the
//   pair's frequency, for the leading `rotated` dimensions of every head; pairs are dimensions
//   (p, p + rotated / 2) or (2 p, 2 p + 1); the inverse rotation takes -s (the rotation is orthogonal:
//   it is also the gradient of the forward one).
// c and s come from a table of fp32 values, built once in 64 bits: positions reach 10^5 and more, where
// a product in 32 bits is off by 0.004 radians, and every layer of a model reads the same rows.
//
// Bound by memory: each value is read and written once.  A thread moves 16 values of one head (two
// 16-byte loads and stores in fp16), a workgroup one token's heads or a share of them, so the position, the
// slot and the table row are uniform and the table's lines stay in the caches for all heads.  8192 tokens of 32 + 8 + 8
// heads of 128 in fp16 (206 MB) are turned and stored in 41 us, 5.0 TB/s; 4093 tokens of 32 + 8 heads in fp32 (169 MB) are
// turned in 35.6 us, 4.7 TB/s (a copy of 2 GiB moves 5.0).  Calls of a few tokens are the launch, 4.2 us.
#include "gguf_common.h"
#include "paged_launch.h"

namespace tensor_paged {
namespace {

using tensor_gguf::half2_from_fp32;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
  if constexpr (sizeof(T) == 2) {
    const tensor_gguf::half8_t h = *reinterpret_cast<const tensor_gguf::half8_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
  } else {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = make_uint4(half2_from_fp32(v[0], v[1]), half2_from_fp32(v[2], v[3]),
                                              half2_from_fp32(v[4], v[5]), half2_from_fp32(v[6], v[7]));
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// VECTOR: units of 16 values (dim and rotated multiples of 16); else units of one pair, or of one
// value past the rotated dimensions, which any size takes (8192 tokens: 41 us and 92; 8 tokens: 4.5 and 5.3).
template <typename In, typename Out, bool INTERLEAVED, bool VECTOR>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a, int units, int threads) {
  const int token = blockIdx.x, work = blockIdx.y * threads + threadIdx.x;
  const int pairs = a.rotated / 2;
  const int heads = a.heads + a.kv + (a.v ? a.kv : 0);
  const int index = work / units, unit = work - index * units;
  if (index >= heads) return;
  // the head's input and output rows: a query's, a key's or a value's (the last two in the cache)
  const bool query = index < a.heads, value = index >= a.heads + a.kv;
  const int head = query ? index : index - a.heads - (value ? a.kv : 0);
  const In* x = static_cast<const In*>(query ? a.q : value ? a.v : a.k) +
                ((size_t)token * (query ? a.heads : a.kv) + head) * a.dim;
  Out* out;
  if (query || !a.v) {
    out = static_cast<Out*>(query ? a.q_out : a.k_out) + ((size_t)token * (query ? a.heads : a.kv) + head) * a.dim;
  } else {
    const int slot = a.slots[token];
    const int page = slot >> a.page_shift, place = slot & ((1 << a.page_shift) - 1);
    if (slot < 0 || page >= a.pages) return;  // a token without a place: nothing is stored
    out = static_cast<Out*>(value ? a.v_out : a.k_out) +
          ((((size_t)page * a.kv + head) << a.page_shift) + place) * a.dim;
  }
  // a position before the table is padding, whose row is zeros; past it there are no angles: NaN
  const int position = a.positions[token];
  const bool inside = position >= 0 && position < a.reach;
  const float outside = position < 0 ? 0.0f : __builtin_nanf("");
  const float* row = a.angles + (size_t)(inside ? position : 0) * a.rotated;
  const float sign = a.inverse ? -1.0f : 1.0f;
  if constexpr (VECTOR && INTERLEAVED) {
    // 16 bytes at a time, the lanes of a head next to each other: a store then fills whole lines (4093 tokens of 40
    // heads in fp32: 35.6 us, 38.6 with 64 bytes of each lane together)
    constexpr int CH = 16 / sizeof(In), COUNT = 16 / CH;
    typedef In Chunk __attribute__((ext_vector_type(CH)));
    typedef Out ChunkOut __attribute__((ext_vector_type(CH)));
    typedef float Half __attribute__((ext_vector_type(CH / 2)));
    Chunk v[COUNT];
    Half c[COUNT], s[COUNT];
#pragma unroll
    for (int k = 0; k < COUNT; ++k) {
      const int i = CH * (unit + units * k);
      v[k] = *reinterpret_cast<const Chunk*>(x + i);
      if (!value && i < a.rotated) {
        c[k] = *reinterpret_cast<const Half*>(row + i / 2);
        s[k] = *reinterpret_cast<const Half*>(row + pairs + i / 2) * sign;
      } else {
        c[k] = 1.0f;
        s[k] = 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < COUNT; ++k) {
      const int i = CH * (unit + units * k);
      const bool turned = !value && i < a.rotated;
      ChunkOut to;
#pragma unroll
      for (int e = 0; e < CH; e += 2) {
        const float x0 = (float)v[k][e], x1 = (float)v[k][e + 1], ce = c[k][e / 2], se = s[k][e / 2];
        const float lo = turned ? x0 * ce - x1 * se : x0, hi = turned ? x1 * ce + x0 * se : x1;
        to[e] = (Out)(value || inside ? lo : outside);
        to[e + 1] = (Out)(value || inside ? hi : outside);
      }
      *reinterpret_cast<ChunkOut*>(out + i) = to;
    }
  } else if constexpr (VECTOR) {
    const bool turned = !value && unit < pairs / 8;
    const int i = turned ? 8 * unit : 16 * unit;
    const int j = turned ? i + pairs : i + 8;
    float v[16];
    load8(x + i, v);
    load8(x + j, v + 8);
    if (turned) {
      float c[8], s[8];
      load8(row + 8 * unit, c);
      load8(row + pairs + 8 * unit, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float se = s[e] * sign, x0 = v[e], x1 = v[e + 8];
        v[e] = x0 * c[e] - x1 * se;
        v[e + 8] = x1 * c[e] + x0 * se;
      }
    }
    if (!value && !inside) {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = outside;
    }
    store8(out + i, v);
    store8(out + j, v + 8);
  } else {
    if (unit >= pairs || value) {
      // past the pairs: one value a unit (a value row has one per unit from 0, two per unit below `pairs`)
      const int i = unit < pairs ? 2 * unit : unit + pairs;
      out[i] = (Out)(value || inside ? (float)x[i] : outside);
      if (unit < pairs) out[i + 1] = (Out)(float)x[i + 1];
      return;
    }
    const int i = INTERLEAVED ? 2 * unit : unit, j = INTERLEAVED ? i + 1 : i + pairs;
    const float x0 = (float)x[i], x1 = (float)x[j], c = row[unit], s = row[pairs + unit] * sign;
    out[i] = (Out)(inside ? x0 * c - x1 * s : outside);
    out[j] = (Out)(inside ? x1 * c + x0 * s : outside);
  }
}

template <typename In, typename Out>
hipError_t launch_typed(const RotaryArgs& a, hipStream_t stream) {
  const bool vector = a.dim % 16 == 0 && a.rotated % 16 == 0;
  const int units = vector ? a.dim / 16 : a.dim - a.rotated / 2;
  const int64_t work = (int64_t)units * (a.heads + a.kv + (a.v ? a.kv : 0));
  const int64_t shares = (work + 255) / 256;
  if (shares > 65535) return hipErrorInvalidValue;
  const int threads = (int)((work + shares - 1) / shares + 63) / 64 * 64;  // whole waves, even shares
  const dim3 grid(a.tokens, (unsigned)((work + threads - 1) / threads));
#define LAUNCH(I, V) \
  hipLaunchKernelGGL((rotary_kernel<In, Out, I, V>), grid, dim3(threads), 0, stream, a, units, threads)
  if (a.interleaved) {
    if (vector) LAUNCH(true, true); else LAUNCH(true, false);
  } else {
    if (vector) LAUNCH(false, true); else LAUNCH(false, false);
  }
#undef LAUNCH
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t stream) {
  if (a.in_f32) return a.out_f32 ? launch_typed<float, float>(a, stream) : launch_typed<float, _Float16>(a, stream);
  return a.out_f32 ? launch_typed<_Float16, float>(a, stream) : launch_typed<_Float16, _Float16>(a, stream);
}

}  // namespace tensor_paged
