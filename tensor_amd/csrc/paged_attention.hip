// Attention over a paged key/value cache, behind a prefix that all requests share (the mathematics and the
// arguments: tensor_paged_attention_v1 in tensor_hip.h; how the work is shared out: paged_plan.h).
//
// One pass over the keys with the running maximum m and sum l of each row's softmax: a tile of scores
// S^T = K Q^T (keys x rows) leaves the matrix cores with each lane holding scores of one row, so the softmax is
// in-lane but for one or two exchanges, and the weights are the B operand of O^T += V^T P^T as they
// are (the sum over keys takes them in any order, V^T's operand in the same).  K and V tiles go to LDS by
// DMA, V^T comes out of it by transposing reads; chunks of 16 bytes are swizzled by row so that both reads
// spread over the banks.
#include "gguf_common.h"
#include "paged_launch.h"
#include "paged_plan.h"

namespace tensor_paged {
namespace {

using tensor_gguf::float4_t;
using tensor_gguf::half2_from_fp32;
using tensor_gguf::half8_t;
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr int kThreads = 64 * kWaves;

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__host__ __device__ inline Extents extents_of(const AttentionArgs& a) {
  return extents(a.tokens, a.requests, a.heads, a.kv, a.page_shift, a.columns, a.prefix_columns);
}
__device__ inline Request request_of(const AttentionArgs& a, const Extents& e, int b) {
  return b == a.requests ? prefix_request(e, a.offsets[b], *a.prefix_length)
                         : own_request(e, a.offsets[b], a.offsets[b + 1], a.lengths[b]);
}

__device__ const uint4 zeros[1] = {};

// 16 bytes a lane from global memory to LDS, lane l to dst + 16 l (dst the same in the whole wave).
// Written as assembly: the compiler makes every LDS read wait for all such loads in flight, of
// other buffers too; the waits here are written out where a stage is read.  (Nothing else here uses m0.)
__device__ __forceinline__ void dma16(const void* src, const void* dst) {
  const uint32_t at = (uint32_t)(uintptr_t)(const void __attribute__((address_space(3)))*)dst;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(uniform((int)at)), "v"(src) : "memory");
}

__device__ __forceinline__ half4_t read_transposed(const _Float16* p) {
  typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
      (fp16x4 __attribute__((address_space(3)))*)p));
}

__device__ __forceinline__ half8_t join(half4_t a, half4_t b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The 16-byte chunk at which a row of a staged tile keeps chunk c: fragment reads of keys take one
// chunk of eight consecutive rows at a time, transposed reads of values two chunks of four rows.
template <int D>
__device__ __forceinline__ int key_chunk(int row, int c) { return c ^ (row & (D / 8 - 1)); }
template <int D>
__device__ __forceinline__ int value_chunk(int row, int c) { return c ^ (2 * (row & (D / 16 - 1))); }

constexpr float kInfinity = __builtin_inff();
// The running maximum is raised (and the sums rescaled) only where a score passes it by this many
// powers of two: weights stay below 2^8 in fp16, and most tiles rescale nothing.
constexpr float kLazy = 8.0f;

// One key head of the cache behind a page list.  A wave holds a window of 64 entries of the list, one in
// each lane, so that a lookup is a lane exchange and the list's loads are rare.
template <int D>
struct Keys {
  const _Float16 *k, *v;
  const int32_t* list;
  int pages, kv, head, shift, bound;  // bound: keys past it are not there
  int first, window, ahead;           // list entry of lane 0, this lane's page (-1: none), the next window's
  __device__ Keys(const AttentionArgs& a, int head, const int32_t* list, int bound)
      : k(static_cast<const _Float16*>(a.k_cache)), v(static_cast<const _Float16*>(a.v_cache)), list(list), pages(a.pages),
        kv(a.kv), head(head), shift(a.page_shift), bound(bound) {}
  __device__ __forceinline__ int entry(int index) const {
    const int p = ((int64_t)index << shift) < bound ? list[index] : -1;
    return (unsigned)p < (unsigned)pages ? p : -1;  // an entry that is no page of the cache hides its keys
  }
  // windows from the one of key `from` on, a tile's first: a tile's entries are in one window
  __device__ __forceinline__ void begin(int from) {
    first = from >> shift;
    window = entry(first + (int)(threadIdx.x & 63));
    ahead = entry(first + 64 + (int)(threadIdx.x & 63));
  }
  __device__ __forceinline__ void reach(int from) {
    if (from >> shift < first + 64) return;
    first += 64;
    window = ahead;
    ahead = entry(first + 64 + (int)(threadIdx.x & 63));
  }
  // the page of a key within the window, -1 for none
  __device__ __forceinline__ int page(int key) const {
    const int p = __shfl(window, (key >> shift) - first);
    return key < bound ? p : -1;
  }
  // 64 bits: a cache passes 2^32 values
  __device__ __forceinline__ size_t at(int page, int key) const {
    return ((((size_t)(unsigned)page * kv + head) << shift) + (key & ((1 << shift) - 1))) * D;
  }
};

// The softmax of one tile of scores against the running maximum: s becomes the weights; returns
// whether the sums have to be scaled by alpha.
template <int N>
__device__ __forceinline__ bool weights(float* s, float top, float& m, float& l, float& alpha, float c) {
  bool raise = (top - m) * c > kLazy || (m == -kInfinity && top > -kInfinity);
  alpha = 1.0f;
  const bool any = __any(raise);
  if (any) {
    const float next = fmaxf(m, top);
    alpha = m == -kInfinity ? 0.0f : exp2f((m - next) * c);
    m = next;
    l *= alpha;
  }
  const float mc = m == -kInfinity ? 0.0f : m * c;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = __builtin_amdgcn_exp2f(s[i] * c - mc);
    sum += s[i];
  }
  l += sum;
  return any;
}

// Where some rows of a tile do not see a key, its weight of 0 would still turn a value that is not
// finite into NaN in those rows.  Such values are cleared in the staged tile (this lane's 16 bytes; true if
// there were any) and added to the rows that see them when the segment is done.
__device__ __forceinline__ bool clear_odd(_Float16* at) {
  uint4 w = *reinterpret_cast<uint4*>(at);
  const uint32_t top = ((w.x & 0x7C007C00u) + 0x04000400u) | ((w.y & 0x7C007C00u) + 0x04000400u) |
                       ((w.z & 0x7C007C00u) + 0x04000400u) | ((w.w & 0x7C007C00u) + 0x04000400u);
  if (!(top & 0x80008000u)) return false;
  uint32_t* word = &w.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t set = (((word[i] & 0x7C007C00u) + 0x04000400u) >> 15) & 0x00010001u;
    word[i] &= ~((set << 16) - set);
  }
  *reinterpret_cast<uint4*>(at) = w;
  return true;
}
__device__ __forceinline__ void add_odd(half4_t v, float* o) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float value = (float)v[i];
    if (!(fabsf(value) < kInfinity)) o[i] += value;
  }
}

__device__ __forceinline__ half8_t pack8(const float* s) {
  const uint4 v = make_uint4(half2_from_fp32(s[0], s[1]), half2_from_fp32(s[2], s[3]), half2_from_fp32(s[4], s[5]),
                             half2_from_fp32(s[6], s[7]));
  return __builtin_bit_cast(half8_t, v);
}

// One segment of a wide item: up to 128 rows, 32 a wave, against key tiles [t0, t1).
template <int D>
__device__ __forceinline__ void wide_segment(const AttentionArgs& a, const Extents& x, const Request& r, const Segment& seg,
                                             const int32_t* pages, float* slot, bool whole, _Float16* lds) {
  constexpr int CH = D / 8, RPW = kWideKeys / kWaves, RPI = 512 / D, N = RPW / RPI;
  constexpr int MAT = kWideKeys * D;  // values of one staged matrix
  constexpr int DB = D / 32, AHEAD = 4;
  const int lane = threadIdx.x & 63, wr = uniform(threadIdx.x >> 6);
  const int half = lane >> 5;
  const int row = wr * 32 + (lane & 31), ti = row / x.share, j = row - ti * x.share, i = seg.tile * x.per + ti;
  const bool live = ti < x.per && i < r.count;
  const int ti_first = uniform(wr * 32 / x.share), i_first = seg.tile * x.per + ti_first;
  const bool wave_live = ti_first < x.per && i_first < r.count;
  const int i_last = min(r.count, (seg.tile + 1) * x.per) - 1;
  const int bound = r.prefix ? r.keys : min(r.keys, r.behind + i_last + 1);
  const int limit = r.prefix ? r.keys : r.behind + (live ? i : i_first) + 1;
  const int full = r.prefix ? r.keys : r.behind + i_first + 1;  // keys that every row of this wave sees
  const float c = a.scale * 1.44269504088896340736f;

  half8_t q[D / 16];
  {
    const _Float16* src = static_cast<const _Float16*>(a.q) +
        ((size_t)(r.first + (live ? i : seg.tile * x.per)) * a.heads + seg.head * x.share + (live ? j : 0)) * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) q[kk] = *reinterpret_cast<const half8_t*>(src + 16 * kk + 8 * half);
  }
  Keys<D> keys(a, seg.head, pages, bound);

  // this wave's 16 rows of a tile, K and V, to LDS (a key that is not there: zeros); returns which of the
  // tile's 64 keys are there
  auto stage = [&](int t, _Float16* dst) {
    const int from = t * kWideKeys;
    keys.reach(from);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r0 = wr * RPW + n * RPI, kr = r0 + lane / CH, p = keys.page(from + kr);
      const size_t at = keys.at(p, from + kr);
      dma16(p < 0 ? (const void*)zeros : keys.k + at + 8 * key_chunk<D>(kr, lane % CH), dst + r0 * D);
      dma16(p < 0 ? (const void*)zeros : keys.v + at + 8 * value_chunk<D>(kr, lane % CH), dst + MAT + r0 * D);
    }
    return __ballot(keys.page(from + lane) >= 0);
  };
  float16_t o[DB] = {};
  float m = -kInfinity, l = 0.0f;

  auto compute = [&](int t, uint64_t seen, const _Float16* ks) {
    const _Float16* vs = ks + MAT;
    float s[2][16];
    {
      float16_t acc[2] = {};
      auto fragment = [&](int n) {
        const int kr = 32 * (n & 1) + (lane & 31);
        return *reinterpret_cast<const half8_t*>(ks + kr * D + 8 * key_chunk<D>(kr, 2 * (n >> 1) + half));
      };
      half8_t k[AHEAD];  // reads stay AHEAD of their products
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) k[n] = fragment(n);
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        __builtin_amdgcn_sched_barrier(0);
        acc[n & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[n % AHEAD], q[n >> 1], acc[n & 1], 0, 0, 0);
        if (n + AHEAD < D / 8) k[n % AHEAD] = fragment(n + AHEAD);
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = acc[kb][e];
    }
    // lane: row lane % 32, keys 32 kb + 8 (e / 4) + 4 half + e % 4
    const int first = t * kWideKeys;
    const bool hidden = first + kWideKeys > full;
    if (hidden || ~seen) {
      // this lane's keys counted from 4 half: what it sees of them as bits
      const int sees = limit - first - 4 * half;
      const uint64_t left = seen >> (4 * half);
      const uint64_t bits = sees <= 0 ? 0 : sees >= 64 ? left : left & ((1ull << sees) - 1);
      const uint32_t word[2] = {(uint32_t)bits, (uint32_t)(bits >> 32)};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!(word[kb] & (1u << (8 * (e / 4) + e % 4)))) s[kb][e] = -kInfinity;
    }
    float top = s[0][0];
#pragma unroll
    for (int e = 1; e < 32; ++e) top = fmaxf(top, s[e / 16][e % 16]);
    top = fmaxf(top, __shfl_xor(top, 32));
    float alpha;
    if (weights<32>(s[0], top, m, l, alpha, c)) {
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
    }
    half8_t p[2][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      p[kb][0] = pack8(&s[kb][0]);
      p[kb][1] = pack8(&s[kb][8]);
    }
    __builtin_amdgcn_sched_barrier(0);  // keeps the second product's reads behind the scores: registers
    // a transposed read gives lane d of 16 four keys' values: rows of four, 16 dimensions of each
    auto values = [&](int n) {
      const int r0 = 16 * (n / DB) + 4 * half + ((lane & 15) >> 2);
      const int chunk = value_chunk<D>(r0, 4 * (n % DB) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1));
      const _Float16* at = vs + r0 * D + 8 * chunk + 4 * (lane & 1);
      return join(read_transposed(at), read_transposed(at + 8 * D));
    };
    half8_t v[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) v[n] = values(n);
#pragma unroll
    for (int n = 0; n < 4 * DB; ++n) {
      __builtin_amdgcn_sched_barrier(0);
      o[n % DB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[n % AHEAD], p[n / DB / 2][n / DB % 2], o[n % DB], 0, 0, 0);
      if (n + AHEAD < 4 * DB) v[n % AHEAD] = values(n + AHEAD);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  // tiles from `clear` on hold keys that some row of the workgroup does not see
  const int clear = r.prefix ? 0x7FFFFFFF : r.behind + seg.tile * x.per + 1;
  bool odd = false;
  keys.begin(seg.t0 * kWideKeys);
  __syncthreads();  // the tiles' place is free
  uint64_t seen = stage(seg.t0, lds);
  for (int t = seg.t0; t < seg.t1; ++t) {
    _Float16* const here = lds + ((t - seg.t0) & 1) * 2 * MAT;
    // this wave's rows have landed; after the barrier everyone's, and the other stage is free
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if ((t + 1) * kWideKeys > clear) {
#pragma unroll
      for (int n = 0; n < N; ++n) odd |= clear_odd(here + MAT + (wr * RPW + n * RPI) * D + 8 * lane);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const uint64_t now = seen;
    if (t + 1 < seg.t1) seen = stage(t + 1, lds + ((t + 1 - seg.t0) & 1) * 2 * MAT);
    if (wave_live) compute(t, now, here);
  }
  l += __shfl_xor(l, 32);
  if (__syncthreads_or(odd)) {
    for (int key = max(seg.t0, max(clear, 0) / kWideKeys) * kWideKeys; key < min(seg.t1 * kWideKeys, bound); ++key) {
      const int page = keys.entry(key >> x.page_shift);
      if (page < 0 || key >= limit) continue;
      const _Float16* v = keys.v + keys.at(page, key) + 4 * half;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float part[4] = {o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
          add_odd(*reinterpret_cast<const half4_t*>(v + 32 * db + 8 * g), part);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[db][4 * g + e] = part[e];
        }
    }
  }
  if (!live) return;
  const float norm = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float4 v = make_float4(o[db][e] * norm, o[db][e + 1] * norm, o[db][e + 2] * norm, o[db][e + 3] * norm);
      const int d = 32 * db + 2 * e + 4 * half;
      if (whole) {
        _Float16* out = static_cast<_Float16*>(a.out) + ((size_t)(r.first + i) * a.heads + seg.head * x.share + j) * D + d;
        *reinterpret_cast<uint2*>(out) = make_uint2(half2_from_fp32(v.x, v.y), half2_from_fp32(v.z, v.w));
      } else {
        *reinterpret_cast<float4*>(slot + 2 * kWideRows + (size_t)row * D + d) = v;
      }
    }
  if (!whole && half == 0) {
    slot[row] = m;
    slot[kWideRows + row] = l;
  }
}

// One segment of a narrow item by one wave: up to 16 rows against key tiles [t0, t1).
template <int D>
__device__ __forceinline__ void narrow_segment(const AttentionArgs& a, const Extents& x, const Request& r, const Segment& seg,
                                               const int32_t* pages, float* slot, bool whole, _Float16* lds) {
  constexpr int CH = D / 8, RPI = 512 / D, N = kNarrowKeys / RPI, MAT = kNarrowKeys * D, DB = D / 16;
  const int lane = threadIdx.x & 63, quad = lane >> 4, row = lane & 15;
  const int i = row / x.share, j = row - i * x.share;
  const bool live = i < r.count;
  const int bound = r.keys;
  const int limit = r.prefix ? r.keys : r.behind + (live ? i : 0) + 1;
  const int full = r.prefix ? r.keys : r.behind + 1;
  const float c = a.scale * 1.44269504088896340736f;
  half8_t q[D / 32];
  {
    const _Float16* src = static_cast<const _Float16*>(a.q) +
        ((size_t)(r.first + (live ? i : 0)) * a.heads + seg.head * x.share + (live ? j : 0)) * D;
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) q[kk] = *reinterpret_cast<const half8_t*>(src + 32 * kk + 8 * quad);
  }
  Keys<D> keys(a, seg.head, pages, bound);
  auto stage = [&](int t, const _Float16* matrix, bool values, _Float16* dst) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int kr = n * RPI + lane / CH, key = t * kNarrowKeys + kr, p = keys.page(key);
      const int chunk = values ? value_chunk<D>(kr, lane % CH) : key_chunk<D>(kr, lane % CH);
      dma16(p < 0 ? (const void*)zeros : matrix + keys.at(p, key) + 8 * chunk, dst + n * RPI * D);
    }
  };
  float4_t o[DB] = {};
  float m = -kInfinity, l = 0.0f;
  bool odd = false;
  keys.begin(seg.t0 * kNarrowKeys);
  stage(seg.t0, keys.k, false, lds);
  stage(seg.t0, keys.v, true, lds + MAT);
  for (int t = seg.t0; t < seg.t1; ++t) {
    const bool more = t + 1 < seg.t1;
    const uint32_t seen = (uint32_t)__ballot(keys.page(t * kNarrowKeys + (lane & 31)) >= 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!r.prefix && (t + 1) * kNarrowKeys > full) {  // keys that some row does not see
#pragma unroll
      for (int n = 0; n < N; ++n) odd |= clear_odd(lds + MAT + n * RPI * D + 8 * lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    float s[8];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      float4_t acc = {};
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) {
        const int kr = 16 * kb + row;
        const half8_t k = *reinterpret_cast<const half8_t*>(lds + kr * D + 8 * key_chunk<D>(kr, 4 * kk + quad));
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[kk], acc, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * kb + e] = acc[e];
    }
    // lane: row lane % 16, keys 16 kb + 4 quad + e
    const int first = t * kNarrowKeys;
    if (first + kNarrowKeys > full || ~seen) {
      const int sees = limit - first - 4 * quad;
      const uint32_t left = seen >> (4 * quad);
      const uint32_t bits = sees <= 0 ? 0 : sees >= 32 ? left : left & ((1u << sees) - 1);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!(bits & (1u << (16 * (e / 4) + e % 4)))) s[e] = -kInfinity;
    }
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, s[e]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    float alpha;
    if (weights<8>(s, top, m, l, alpha, c)) {
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
    }
    const half8_t p = pack8(s);
    auto values = [&](int db) {
      const int r0 = 4 * quad + (row >> 2), chunk = value_chunk<D>(r0, 2 * db + ((lane & 3) >> 1));
      const _Float16* at = lds + MAT + r0 * D + 8 * chunk + 4 * (lane & 1);
      return join(read_transposed(at), read_transposed(at + 16 * D));
    };
#pragma unroll
    for (int db = 0; db < DB; ++db)
      o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(values(db), p, o[db], 0, 0, 0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile has been read
    if (more) {
      keys.reach((t + 1) * kNarrowKeys);
      stage(t + 1, keys.k, false, lds);
      stage(t + 1, keys.v, true, lds + MAT);
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (__any(odd)) {
    for (int key = max(seg.t0, full / kNarrowKeys) * kNarrowKeys; key < min(seg.t1 * kNarrowKeys, bound); ++key) {
      const int page = keys.entry(key >> x.page_shift);
      if (page < 0 || key >= limit) continue;
      const _Float16* v = keys.v + keys.at(page, key) + 4 * quad;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        float part[4] = {o[db][0], o[db][1], o[db][2], o[db][3]};
        add_odd(*reinterpret_cast<const half4_t*>(v + 16 * db), part);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[db][e] = part[e];
      }
    }
  }
  if (!live) return;
  const float norm = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    const int d = 16 * db + 4 * quad;
    const float4_t v = o[db] * norm;
    if (whole) {
      _Float16* out = static_cast<_Float16*>(a.out) + ((size_t)(r.first + i) * a.heads + seg.head * x.share + j) * D + d;
      *reinterpret_cast<uint2*>(out) = make_uint2(half2_from_fp32(v[0], v[1]), half2_from_fp32(v[2], v[3]));
    } else {
      *reinterpret_cast<float4_t*>(slot + 2 * kNarrowRows + row * D + d) = v;
    }
  }
  if (!whole && quad == 0) {
    slot[row] = m;
    slot[kNarrowRows + row] = l;
  }
}

// Every workgroup plans the whole call itself (a scan over the requests' key tiles), takes an equal
// share of the wide tiles and each of its waves an equal share of the narrow ones.
template <int D>
__global__ __launch_bounds__(kThreads, 2) void attend(const AttentionArgs a) {
  __shared__ __attribute__((aligned(16))) _Float16 tiles[kWaves * 8192];
  __shared__ int32_t starts[2][kAttentionMaxRequests + 2];
  __shared__ int32_t sums[2][kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const Extents x = extents_of(a);
  const int lists = a.requests + 1;
  int done[2] = {0, 0};  // tiles of the wide and the narrow list
  for (int base = 0; base < lists; base += kThreads) {
    const int b = base + tid;
    int mine[2] = {0, 0};
    if (b < lists) {
      const Request r = request_of(a, x, b);
      const int n = a.kv * (int)head_tiles(x, r);
      mine[0] = r.narrow ? 0 : n;
      mine[1] = r.narrow ? n : 0;
    }
    int scan[2] = {mine[0], mine[1]};
#pragma unroll
    for (int step = 1; step < 64; step <<= 1)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int below = __shfl_up(scan[k], step);
        if (lane >= step) scan[k] += below;
      }
    __syncthreads();
    if (lane == 63) {
      sums[0][wave] = scan[0];
      sums[1][wave] = scan[1];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int before = done[k];
      for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += sums[k][w];
        done[k] += sums[k][w];
      }
      if (b < lists) starts[k][b] = before + scan[k] - mine[k];
    }
  }
  if (tid < 2) starts[tid][lists] = tid ? done[1] : done[0];
  __syncthreads();
  const int quota[2] = {(done[0] + kGroups - 1) / kGroups, (done[1] + kStreams - 1) / kStreams};
  if (blockIdx.x == 0) {  // for the kernel that joins the segments
    int32_t* plan = static_cast<int32_t*>(a.workspace);
    if (tid < 2) plan[tid] = tid ? quota[1] : quota[0];
    for (int b = tid; b <= lists; b += kThreads) {
      plan[2 + b] = starts[0][b];
      plan[3 + lists + b] = starts[1][b];
    }
  }
  const bool alone = prefix_request(x, a.tokens, *a.prefix_length).keys == 0;
  float* const slots = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + plan_bytes(a.requests));

  const int wide_end = min((int)(blockIdx.x + 1) * quota[0], done[0]);
  for (int t = (int)blockIdx.x * quota[0]; t < wide_end;) {
    const int b = uniform(find(starts[0], lists, t));
    const Request r = request_of(a, x, b);
    Segment seg = segment_at(x, r, b, (starts[0][b + 1] - starts[0][b]) / a.kv, t - starts[0][b],
                             wide_end - t);
    seg.head = uniform(seg.head);
    seg.tile = uniform(seg.tile);
    seg.t0 = uniform(seg.t0);
    seg.t1 = uniform(seg.t1);
    wide_segment<D>(a, x, r, seg, r.prefix ? a.prefix_pages : a.table + (size_t)b * a.columns,
                    slots + slot_floats(kWideRows, D) * (size_t)(seg.item + blockIdx.x), alone && !r.prefix && seg.all,
                    tiles);
    t += seg.t1 - seg.t0;
  }
  __syncthreads();
  float* const narrow_base = slots + slot_floats(kWideRows, D) * (size_t)wide_slots(x);
  const int stream = wave * kGroups + blockIdx.x;  // neighbours in the list run on different CUs
  const int narrow_end = min((stream + 1) * quota[1], done[1]);
  for (int t = stream * quota[1]; t < narrow_end;) {
    const int b = uniform(find(starts[1], lists, t));
    const Request r = request_of(a, x, b);
    Segment seg = segment_at(x, r, b, (starts[1][b + 1] - starts[1][b]) / a.kv, t - starts[1][b],
                             narrow_end - t);
    seg.head = uniform(seg.head);
    seg.t0 = uniform(seg.t0);
    seg.t1 = uniform(seg.t1);
    narrow_segment<D>(a, x, r, seg, r.prefix ? a.prefix_pages : a.table + (size_t)b * a.columns,
                      narrow_base + slot_floats(kNarrowRows, D) * (size_t)(seg.item + stream),
                      alone && !r.prefix && seg.all, tiles + wave * 2 * kNarrowKeys * D);
    t += seg.t1 - seg.t0;
  }
}

// Joins the segments of a token's query heads: out = sum_p w_p O_p / sum_p w_p l_p, w_p = exp(m_p - max m).
// A workgroup takes one or all key heads of a token (HEADS; what the token's place in the plan costs is then
// shared), a thread four dimensions of a query head; threads beyond those of a key head share its segments.
template <int D, int THREADS>
__global__ __launch_bounds__(THREADS) void join_segments(const AttentionArgs a, int heads) {
  constexpr int VECS = D / 4, BATCH = 4;
  const int groups = a.kv / heads;
  const int token = blockIdx.x / groups, first_head = (blockIdx.x - token * groups) * heads;
  const int tid = threadIdx.x, lane = tid & 63;
  const Extents x = extents_of(a);
  const float c = a.scale * 1.44269504088896340736f;
  const Request all = request_of(a, x, a.requests);
  const int32_t* plan = static_cast<const int32_t*>(a.workspace);
  const float* const slots = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.workspace) + plan_bytes(a.requests));
  const float* const narrow_base = slots + slot_floats(kWideRows, D) * (size_t)wide_slots(x);

  struct Part {  // the token's rows in the slots of one list
    TokenSlots at;
    const float* base;
    int rows, quota;
  };
  auto part = [&](const Request& r, int b) {
    return Part{token_slots(x, r, b, plan[2 + (r.narrow ? a.requests + 2 : 0) + b], token), r.narrow ? narrow_base : slots,
                r.narrow ? kNarrowRows : kWideRows, plan[r.narrow ? 1 : 0]};
  };
  Part shared{}, mine{};
  if (token < all.count) {
    int b = 0;  // the token's request: offsets[b] <= token
    for (int i = 1; i < a.requests; i += 64)
      b += __popcll(__ballot(i + lane < a.requests && a.offsets[min(i + lane, a.requests)] <= token));
    const Request r = request_of(a, x, b);
    if (token >= r.first && token < r.first + r.count) {
      shared = part(all, a.requests);
      mine = part(r, b);
    }
  }
  const int vecs = x.share * VECS, sets = vecs < THREADS ? THREADS / vecs : 1, set = tid / vecs;
  __shared__ float4_t outs[THREADS];
  __shared__ float2 stats[THREADS];
  for (int head = first_head; head < first_head + heads; ++head) {
    const Slots one = shared.at.in(head, shared.quota), two = mine.at.in(head, mine.quota);
    if (two.count == 1 && all.keys == 0) continue;  // the segment wrote the output itself
    const int count = one.count + two.count;
    for (int v = tid - set * vecs; v < vecs; v += THREADS) {  // more than once where sets is 1
      const int j = v / VECS, vec = v - j * VECS;
      float m = -kInfinity, l = 0.0f;
      float4_t o = {};
      if (set < sets) {
        for (int p0 = set; p0 < count; p0 += BATCH * sets) {
          float mp[BATCH], lp[BATCH];
          float4_t op[BATCH];
#pragma unroll
          for (int n = 0; n < BATCH; ++n) {
            const int p = min(p0 + n * sets, count - 1);
            const bool first = p < one.count;
            const Part& from = first ? shared : mine;
            const int rows = first ? shared.rows : mine.rows, row = (first ? shared.at.row : mine.at.row) + j;
            const float* slot = from.base + slot_floats(rows, D) * (size_t)(first ? one.first + p : two.first + p - one.count);
            mp[n] = slot[row];
            lp[n] = slot[rows + row];
            op[n] = *reinterpret_cast<const float4_t*>(slot + 2 * rows + (size_t)row * D + 4 * vec);
          }
#pragma unroll
          for (int n = 0; n < BATCH; ++n) {
            if (p0 + n * sets >= count) break;
            const float next = fmaxf(m, mp[n]);
            const float f = m == -kInfinity ? 0.0f : exp2f((m - next) * c);
            const float g = mp[n] == -kInfinity ? 0.0f : exp2f((mp[n] - next) * c);
            l = l * f + lp[n] * g;
            o = o * f + op[n] * g;
            m = next;
          }
        }
      }
      if (sets == 1 && set) break;  // threads beyond the key head's
      if (sets > 1) {  // one round of this loop
        __syncthreads();
        outs[tid] = o;
        stats[tid] = make_float2(m, l);
        __syncthreads();
        if (set) continue;
        for (int s = 1; s < sets; ++s) {
          const float2 other = stats[tid + s * vecs];
          const float next = fmaxf(m, other.x);
          const float f = m == -kInfinity ? 0.0f : exp2f((m - next) * c);
          const float g = other.x == -kInfinity ? 0.0f : exp2f((other.x - next) * c);
          l = l * f + other.y * g;
          o = o * f + outs[tid + s * vecs] * g;
          m = next;
        }
      }
      const float4_t w = o * (l == 0.0f ? 0.0f : 1.0f / l);
      *reinterpret_cast<uint2*>(static_cast<_Float16*>(a.out) + ((size_t)token * a.heads + head * x.share) * D + 4 * v) =
          make_uint2(half2_from_fp32(w[0], w[1]), half2_from_fp32(w[2], w[3]));
    }
  }
}

template <int D>
hipError_t launch_dim(const AttentionArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((attend<D>), dim3(kGroups), dim3(kThreads), 0, stream, a);
  hipError_t status = hipGetLastError();
  if (status != hipSuccess) return status;
  const int64_t units = (int64_t)a.tokens * a.kv;
  if (units <= kGroups)
    hipLaunchKernelGGL((join_segments<D, 1024>), dim3((unsigned)units), dim3(1024), 0, stream, a, 1);
  else if (a.tokens < 4 * kGroups)
    hipLaunchKernelGGL((join_segments<D, 256>), dim3((unsigned)units), dim3(256), 0, stream, a, 1);
  else
    hipLaunchKernelGGL((join_segments<D, 256>), dim3((unsigned)a.tokens), dim3(256), 0, stream, a, a.kv);
  return hipGetLastError();
}

}  // namespace

size_t attention_workspace(const AttentionArgs& a) {
  const Extents x = extents_of(a);
  return plan_bytes(a.requests) + 4 * (slot_floats(kWideRows, a.dim) * (size_t)wide_slots(x) +
                                       slot_floats(kNarrowRows, a.dim) * (size_t)narrow_slots(x));
}

hipError_t launch_attention(const AttentionArgs& a, hipStream_t stream) {
  return a.dim == 64 ? launch_dim<64>(a, stream) : a.dim == 128 ? launch_dim<128>(a, stream) : hipErrorInvalidValue;
}

}  // namespace tensor_paged
