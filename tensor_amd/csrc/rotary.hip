// Rotary positions of queries and keys, with or without the store of keys and values into a paged
// cache, one launch:
//   (a, b) -> (a c - b s, b c + a s), c and s the cosine and sine of the token's position times the
//   pair's frequency, for the leading `rotated` dimensions of every head; pairs are dimensions
//   (p, p + rotated / 2) or (2 p, 2 p + 1); the inverse takes -s: the transposed map, the gradient of the forward one
//   whatever c and s, and its inverse where c^2 + s^2 = 1.
// c and s come from a table of fp32 values, built once in 64 bits: positions reach 10^5 and more, where
// a product in 32 bits is off by 0.004 radians, and every layer of a model reads the same rows.
//
// Bound by memory: each value is read and written once.  A thread moves 16 values of one head, 16
// bytes at a time, a workgroup one token's heads or a share of them, so the position, the
// slot and the table row are uniform and the table's lines stay in the caches for all heads.  8192 tokens of 32 + 8 + 8
// heads of 128 in fp16 (206 MB) are turned and stored in 40.4 us, 5.1 TB/s; 4093 tokens of 32 + 8 heads in fp32 (169 MB) are
// turned in 35.6 us, 4.7 TB/s (a copy of 2 GiB moves 5.0).  Calls of a few tokens are the launch, 4.2 us.
#include "gguf_common.h"
#include "paged_launch.h"

namespace tensor_paged {
namespace {

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
    // The same: units below `whole` take 8 pairs, in chunks among the others' of the first halves and the second ones;
    // those from it on share what is not turned (4093 tokens of 40 heads in fp32: 33.3 us, 35.4 with 32 bytes of each
    // lane together; half of each head turned: 35.2 and 38.4; 8192 stored in fp16: 40.4 and 41.8).
    constexpr int CH = 16 / sizeof(In), COUNT = 16 / CH, HALF = COUNT / 2;
    typedef In Chunk __attribute__((ext_vector_type(CH)));
    typedef Out ChunkOut __attribute__((ext_vector_type(CH)));
    typedef float Floats __attribute__((ext_vector_type(CH)));
    const int whole = value ? 0 : pairs / 8;
    const bool turned = unit < whole;
    const int i = turned ? CH * unit : 16 * whole + CH * (unit - whole), apart = CH * (turned ? whole : units - whole);
    const int second = turned ? pairs : HALF * apart;  // from a chunk to that HALF chunks later
    Chunk v[COUNT];
    Floats c[HALF], s[HALF];
#pragma unroll
    for (int k = 0; k < HALF; ++k) {
      v[k] = *reinterpret_cast<const Chunk*>(x + i + apart * k);
      v[k + HALF] = *reinterpret_cast<const Chunk*>(x + i + apart * k + second);
      if (turned) {
#pragma unroll
        for (int e = 0; e < CH; e += 4) {
          const float4 cos = *reinterpret_cast<const float4*>(row + i + apart * k + e);
          const float4 sin = *reinterpret_cast<const float4*>(row + pairs + i + apart * k + e);
          c[k][e] = cos.x; c[k][e + 1] = cos.y; c[k][e + 2] = cos.z; c[k][e + 3] = cos.w;
          s[k][e] = sin.x; s[k][e + 1] = sin.y; s[k][e + 2] = sin.z; s[k][e + 3] = sin.w;
        }
      } else {
        c[k] = 1.0f;
        s[k] = 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < HALF; ++k) {
      ChunkOut lo, hi;
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        const float x0 = (float)v[k][e], x1 = (float)v[k + HALF][e], se = s[k][e] * sign;
        const float a0 = turned ? x0 * c[k][e] - x1 * se : x0, a1 = turned ? x1 * c[k][e] + x0 * se : x1;
        lo[e] = (Out)(value || inside ? a0 : outside);
        hi[e] = (Out)(value || inside ? a1 : outside);
      }
      *reinterpret_cast<ChunkOut*>(out + i + apart * k) = lo;
      *reinterpret_cast<ChunkOut*>(out + i + apart * k + second) = hi;
    }
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

bool in_vectors(const RotaryArgs& a) { return a.dim % 16 == 0 && a.rotated % 16 == 0; }
int units_of(const RotaryArgs& a) { return in_vectors(a) ? a.dim / 16 : a.dim - a.rotated / 2; }
int64_t work_of(const RotaryArgs& a) { return (int64_t)units_of(a) * (a.heads + a.kv + (a.v ? a.kv : 0)); }

template <typename In, typename Out>
hipError_t launch_typed(const RotaryArgs& a, hipStream_t stream) {
  const bool vector = in_vectors(a);
  const int units = units_of(a), threads = rotary_threads(a);
  const int64_t work = work_of(a);
  if ((work + 255) / 256 > 65535) return hipErrorInvalidValue;
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

int rotary_threads(const RotaryArgs& a) {
  const int64_t work = work_of(a), shares = (work + 255) / 256;
  return (int)((work + shares - 1) / shares + 63) / 64 * 64;  // whole waves, even shares
}

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t stream) {
  if (a.in_f32) return a.out_f32 ? launch_typed<float, float>(a, stream) : launch_typed<float, _Float16>(a, stream);
  return a.out_f32 ? launch_typed<_Float16, float>(a, stream) : launch_typed<_Float16, _Float16>(a, stream);
}

}  // namespace tensor_paged
