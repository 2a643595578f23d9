// Attention over a paged key/value cache, behind a prefix that all requests share (the mathematics and the
// arguments: tensor_paged_attention_v1 in tensor_hip.h; how the work is shared out: paged_plan.h).
//
// One pass over the keys with the running maximum m and sum l of each row's softmax: a tile of scores
// S^T = K Q^T (keys x rows) leaves the matrix cores with each lane holding scores of one row, so the softmax is
// in-lane but for one or two exchanges, and the weights are the B operand of O^T += V^T P^T as they
// are (the sum over keys takes them in any order, V^T's operand in the same).  Scores, m, l and O are fp32; the
// weights are rounded to fp16 for the product, 2^-11 of each, or 2^-32 of the largest where that is more (kLift); l is the
// sum of the rounded ones.  K and V tiles go to LDS by DMA, V^T comes out of it by transposing reads; chunks of 16
// bytes are swizzled by row so that both reads spread over the banks.
//
// Two kernels: `attend` leaves each segment's rows in a slot, `join_segments` adds up the slots of a row.
//
// Decode is bound by the cache's bytes: 256 requests of up to 4096 keys (2.1 GB, 8 key heads of 128) take 0.40 ms,
// 5.3 TB/s, where a copy of 2 GiB moves 5.0; one request behind a prefix of 131071 keys (0.54 GB) takes 107 us, 5.0
// TB/s.  Prompts are bound by the matrix cores and the power they draw (the clock falls to 1.6 GHz): 3 requests of 1024
// tokens behind 8192 + 1024 keys (325 GFLOP) take 0.39 ms, 0.83 PFLOP/s, 30 us of it joining, where an fp16 product of
// 8192^3 reaches 1.16.  The smallest calls are two launches and their chains of loads: one token of 1021 keys takes
// 12.4 us, 7 and 5.5 us of it the kernels.
#include <type_traits>

#include "gguf_common.h"
#include "paged_launch.h"
#include "paged_plan.h"

namespace tensor_paged {
namespace {

using tensor_gguf::dot2;
using tensor_gguf::float2_t;
using tensor_gguf::float4_t;
using tensor_gguf::half2_t;
using tensor_gguf::half2_from_fp32;
using tensor_gguf::half8_t;
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr int kThreads = 64 * kWaves;

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ size_t uniform(size_t v) {
  return (size_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v);
}

// threadIdx.x as a value of its own: what a segment derives from it is then not kept in registers outside
__device__ __forceinline__ int here() {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid;
}

__host__ __device__ inline Extents extents_of(const AttentionArgs& a) {
  return extents(a.tokens, a.requests, a.heads, a.kv, a.page_shift, a.columns, a.prefix_columns);
}
__device__ inline Request request_of(const AttentionArgs& a, const Extents& e, int b) {
  return b == a.requests ? prefix_request(e, a.offsets[b], *a.prefix_length)
                         : own_request(e, a.offsets[b], a.offsets[b + 1], a.lengths[b]);
}

template <typename T>
__device__ __forceinline__ T read_lds(uint32_t at) {
  return *(const T __attribute__((address_space(3)))*)(uintptr_t)at;
}
__device__ __forceinline__ half4_t read_transposed(uint32_t at) {
  typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((fp16x4 __attribute__((address_space(3)))*)(uintptr_t)at));
}

__device__ __forceinline__ half8_t join(half4_t a, half4_t b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The 16-byte chunk at which a row of a staged tile keeps chunk c, so that the lanes of half a wave read 64 different
// banks: keys' fragments are one chunk of eight consecutive rows, values' transposed ones four chunks of four rows
// (wide) or two of eight (narrow).
template <int D>
__device__ __forceinline__ int key_chunk(int row, int c) { return c ^ (row & (D / 8 - 1)); }
template <int D>
__device__ __forceinline__ int wide_value_chunk(int row, int c) { return c ^ (4 * (D == 128 ? row & 3 : (row >> 1) & 1)); }
template <int D>
__device__ __forceinline__ int narrow_value_chunk(int row, int c) { return c ^ (2 * (row & (D / 16 - 1))); }

// Loads of these values are waited for here, where no tile is on its way: the compiler, which does not know
// of those, waits for all loads before a value's first use.
template <int N>
__device__ __forceinline__ void settle(half8_t (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}

constexpr float kInfinity = __builtin_inff();

// Maximum over a lane and the one 32 away, and over those 16 apart: rows of lanes of two copies are exchanged.
// (Assembly, with the wait states a lane exchange needs after a vector write: the compiler takes the two
// results of its builtin for equal here.)
__device__ __forceinline__ float max32(float v) {
  float a = v, b = v;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return fmaxf(a, b);
}
__device__ __forceinline__ float max16(float v) {
  float a = v, b = v;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return fmaxf(a, b);
}
// The running maximum is raised (and the sums rescaled) only where a score passes it by this many
// powers of two: most tiles rescale nothing (3 x 1024 tokens behind 8192 keys: 386 us, 432 if every new maximum
// rescales).
constexpr float kLazy = 8.0f;
// Weights are kept times 2^kLift, as are l and O, in every segment alike: up to 2^15 then, where fp16 ends at 2^16.  Below
// 2^-14 fp16 keeps fewer bits and below 2^-25 none, so that keys which one key outweighs by 2^25 would be lost, however
// many (131072 of them are 0.4% of the values); lifted, that is 2^32.
constexpr float kLift = 7.0f;
// A weight's exponent is s c + (kLift - m c) in one operation, the sum in brackets rounded once for the row, or
// (s - m) c + kLift in two.  The rounding scales all weights of a segment alike, but from this m c on by more than
// their own in fp16, and from 2^24 on by more than fp16 holds: there wide segments take the second form, and narrow
// ones, whose time is the loads', everywhere (3 x 1024 tokens behind 8192 keys: 386 us, 408 with the second form for
// every row).
constexpr float kFar = 16384.0f;

__device__ const uint4 zeros[1] = {};

// 16 bytes a lane from global memory to LDS, lane l to dst + 16 l (dst, an LDS address, is the same in the whole wave).
// Written as assembly: the compiler makes every LDS read wait for all such loads in flight, of
// other buffers too; the waits here are written out where a stage is read.  (Nothing else here uses m0.)
__device__ __forceinline__ void dma16(const void* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(uniform((int)dst)), "v"(src) : "memory");
}
__device__ __forceinline__ void dma4(const void* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(uniform((int)dst)), "v"(src) : "memory");
}
// 16 rows of D values, one after another in memory from `base`, to LDS from dst on: D / 32 loads, which share the
// scalar part of their addresses (the offset of an instruction counts on both sides).
template <int D>
__device__ __forceinline__ void dma_rows(const void* base, const uint32_t (&offset)[D / 32], uint32_t dst) {
  if constexpr (D == 128)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\t"
                 "global_load_lds_dwordx4 %2, %5 offset:0x400\n\tglobal_load_lds_dwordx4 %3, %5 offset:0x800\n\t"
                 "global_load_lds_dwordx4 %4, %5 offset:0xc00"
                 :: "s"(uniform((int)dst)), "v"(offset[0]), "v"(offset[1]), "v"(offset[2]), "v"(offset[3]), "s"(base) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\t"
                 "global_load_lds_dwordx4 %2, %3 offset:0x400"
                 :: "s"(uniform((int)dst)), "v"(offset[0]), "v"(offset[1]), "s"(base) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const void __attribute__((address_space(3)))*)p;
}

// One key head of the cache behind a page list.  A wave holds a window of 64 entries of the list, one in
// each lane; the next window is on its way to LDS (`ring`, 128 entries of this wave) by then.
template <int D>
struct Keys {
  const _Float16 *k, *v;
  const int32_t* list;
  int32_t* ring;
  int pages, kv, head, shift, bound;  // keys from bound on are not there
  int lane;
  int first, window, flip;            // list entry of lane 0, this lane's page (-1: none), the window's half of the ring
  uint64_t there;                     // lanes that have a page
  __device__ Keys(const AttentionArgs& a, int head, const int32_t* list, int bound, int32_t* ring, int lane)
      : k(static_cast<const _Float16*>(a.k_cache)), v(static_cast<const _Float16*>(a.v_cache)), list(list), ring(ring),
        pages(a.pages), kv(a.kv), head(head), shift(a.page_shift), bound(bound), lane(lane) {}
  __device__ __forceinline__ int last() const { return max(bound - 1, 0) >> shift; }
  __device__ __forceinline__ int valid(int index, int page) const {
    return index <= last() && (unsigned)page < (unsigned)pages ? page : -1;  // no page of the cache: hides its keys
  }
  __device__ __forceinline__ int entry(int index) const { return valid(index, list[min(index, last())]); }
  __device__ __forceinline__ void fetch(int from, int half) const {
    dma4(list + min(from + lane, last()), lds_address(ring) + 256 * half);
  }
  __device__ __forceinline__ void open() {
    window = valid(first + lane, ring[64 * flip + lane]);
    there = __ballot(window >= 0);
  }
  // windows from the one of key `from` on, a tile's first: a tile's entries are in one window
  __device__ __forceinline__ void begin(int from) {
    first = from >> shift;
    flip = 0;
    fetch(first, 0);
    fetch(first + 64, 1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    open();
  }
  // (the window opened here was fetched before tiles that have been waited for since)
  __device__ __forceinline__ void reach(int from) {
    if (from >> shift < first + 64) return;
    first += 64;
    flip ^= 1;
    open();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    fetch(first + 64, flip ^ 1);
  }
  // whether the tile of COUNT keys at `from`, in the window, has a key, and all the pages that it has keys in
  template <int COUNT>
  __device__ __forceinline__ bool whole(int from) const {
    if (from >= bound) return false;  // (where a request's first tokens see nothing)
    const int at = (from >> shift) - first, entries = min((from + COUNT - 1) >> shift, last()) - first - at + 1;  // 1 to 64
    const uint64_t want = entries >= 64 ? ~0ull : (1ull << entries) - 1;
    return !(want & ~(there >> at));
  }
  // the page of a key of the window, -1 for none
  __device__ __forceinline__ int page(int key) const {
    const int p = __shfl(window, (key >> shift) - first);
    return key < bound ? p : -1;
  }
  // 64 bits: a cache passes 2^32 values
  __device__ __forceinline__ size_t at(int page, int key) const {
    return ((((size_t)(unsigned)page * kv + head) << shift) + (key & ((1 << shift) - 1))) * D;
  }
  // byte offset of a key that is there, the same in the whole wave
  __device__ __forceinline__ size_t row(int key) const {
    return 2 * at(__builtin_amdgcn_readlane(window, (key >> shift) - first), key);
  }
};

// A wave's rows of a tile, GROUPS times 16.  Where all its pages are there and hold 16 tokens or more, a group's
// rows lie one after another, and where is in scalar registers (those of a page that are past the last key are
// loaded too; a group past it is the last one again).  Otherwise each row is looked up, and a key that is not there
// read as zeros (pages of 8 tokens: 405 us for 256 requests of up to 4096 keys, 398 with pages of 16; 3 x 1024 tokens behind
// 8192 keys: 514 and 386).
template <int D, int COUNT, int GROUPS>
struct Rows {
  static constexpr int CH = D / 8, RPI = 512 / D, PER = D / 32;  // chunks of a row, rows of a load, loads of a group
  size_t at[GROUPS];
  bool fast;
  __device__ __forceinline__ void find(const Keys<D>& keys, int from, int r0) {
    fast = keys.shift >= 4 && keys.template whole<COUNT>(from);
    if (fast) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) at[g] = keys.row(min(from + r0 + 16 * g, (keys.bound - 1) & ~15));
    }
  }
  // lane_at: where a lane's 16 bytes are from the first of its load's rows
  __device__ __forceinline__ void load(const Keys<D>& keys, int from, int r0, const _Float16* matrix,
                                       const uint32_t (&lane_at)[PER], uint32_t dst) const {
    const int lane = keys.lane;
    dst += 2 * r0 * D;
    if (fast) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        dma_rows<D>(reinterpret_cast<const uint8_t*>(matrix) + uniform(at[g]), lane_at, dst + 32 * g * D);
    } else {
      int page[GROUPS * PER];
#pragma unroll
      for (int n = 0; n < GROUPS * PER; ++n) page[n] = keys.page(from + r0 + n * RPI + lane / CH);
#pragma unroll
      for (int n = 0; n < GROUPS * PER; ++n) {
        const int key = from + r0 + n * RPI + lane / CH;
        const uint32_t chunk = lane_at[n % PER] / 2 - (lane / CH) * D;
        dma16(page[n] < 0 ? (const void*)zeros : matrix + keys.at(page[n], key) + chunk, dst + 1024 * n);
      }
    }
  }
};

// Moves a row's running maximum m up to `top` where that passes it by 2^kLazy; true if the wave's sums have
// to be scaled by alpha.
__device__ __forceinline__ bool raise(float top, float& m, float& alpha, float c) {
  if (!__any((top - m) * c > kLazy || (m == -kInfinity && top > -kInfinity))) return false;
  const float next = fmaxf(m, top);
  alpha = m == -kInfinity ? 0.0f : exp2f((m - next) * c);
  m = next;
  return true;
}

// The weights of keys past the last one are 0, and so must be their values: this lane's rows of a staged tile,
// RPI rows apart from `key` on.
template <int D, int N>
__device__ __forceinline__ void clear_past(_Float16* at, int key, int bound) {
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (key + n * (512 / D) >= bound) *reinterpret_cast<uint4*>(at + 512 * n) = uint4{};
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

// One segment of a wide item: up to 128 rows, 32 a wave, against key tiles [t0, t1), of which the first x.lead of
// a request are the shared prefix's.
//
// A wave's 32 scores x 32 rows are one matrix product's result; while the weights of 32 keys are made (16 exponents a
// lane), the matrix cores have the scores of the next 32, and while O takes those weights, the next scores' maximum is
// found.  K is loaded two tiles ahead and V one, so that a wait is for loads issued a tile ago; two barriers a tile.  Two
// workgroups on a CU (256 registers a wave, 80 KB of LDS each) fill each other's waits: matrix cores 50% busy at
// 3 x 1024 tokens, no bank conflicts.  Eight waves a workgroup, tiles of 32 keys in three stages and other wave
// priorities were measured level or slower.
template <int D>
__device__ __forceinline__ void wide_segment(const AttentionArgs& a, const Extents& x, const Request& r, const Segment& seg,
                                             const int32_t* pages, int prefix_keys, float* slot, bool whole, _Float16* lds, int32_t* ring) {
  constexpr int CH = D / 8, RPI = 512 / D, N = D / 32;  // chunks of a row, rows of a load, loads of this wave's 16 rows
  constexpr int MAT = kWideKeys * D;  // values of one staged matrix
  constexpr int DB = D / 32, AHEAD = 4;
  const int tid = here(), lane = tid & 63, wr = uniform(tid >> 6);
  const int half = lane >> 5;
  const int row = wr * 32 + (lane & 31), ti = row / x.share, j = row - ti * x.share, i = seg.tile * x.per + ti;
  const bool live = ti < x.per && i < r.count;
  const int ti_first = uniform(wr * 32 / x.share), i_first = seg.tile * x.per + ti_first;
  const bool wave_live = ti_first < x.per && i_first < r.count;
  const int i_last = min(r.count, (seg.tile + 1) * x.per) - 1, lead = lead_of(x, r);
  const float c = a.scale * 1.44269504088896340736f;

  half8_t q[D / 16];
  {
    const _Float16* src = static_cast<const _Float16*>(a.q) +
        ((size_t)(r.first + (live ? i : seg.tile * x.per)) * a.heads + seg.head * x.share + (live ? j : 0)) * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) q[kk] = *reinterpret_cast<const half8_t*>(src + 16 * kk + 8 * half);
  }
  static_assert(kWideKeys == 16 * kWaves, "a wave loads 16 rows of a tile");
  using Tile = Rows<D, kWideKeys, 1>;
  const int r0 = 16 * wr;
  uint32_t k_lane[N], v_lane[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int kr = r0 + n * RPI + lane / CH;
    k_lane[n] = 2 * ((lane / CH) * D + 8 * key_chunk<D>(kr, lane % CH));
    v_lane[n] = 2 * ((lane / CH) * D + 8 * wide_value_chunk<D>(kr, lane % CH));
  }
  float16_t o[DB] = {};
  float m = -kInfinity, l = 0.0f, top;
  float off = kLift;  // kLift - m c; before the first key, kLift
  bool far = false;  // of some row of the wave: weights in two operations
  float s[16];  // scores, lane: row lane % 32, keys 8 (e / 4) + 4 half + e % 4

  // LDS addresses of this lane's fragments: a row of K in the tile at hand, its chunks; and four rows of V^T for
  // each 32 dimensions (a transposed read gives lane d of 16 four keys' values: rows of four, 16 dimensions of
  // each).  The two places of a tile differ in one bit.
  uint32_t k_at[D / 16], v_at[DB];
  const uint32_t lds_at = lds_address(lds);
  auto first_place = [&]() {
#pragma unroll
    for (int n = 0; n < D / 16; ++n) k_at[n] = lds_at + 2 * ((lane & 31) * D + 8 * key_chunk<D>(lane & 31, 2 * n + half));
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int vr = 4 * half + ((lane & 15) >> 2);
      v_at[db] = lds_at + 4 * MAT +
                 2 * (vr * D + 8 * wide_value_chunk<D>(vr, 4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 4 * (lane & 1));
    }
  };
  // S^T = K Q^T of 32 keys, `between(n)` after each of its D / 16 products; fragment reads stay AHEAD of them
  auto scores = [&](auto half_tile, auto between) {
    constexpr int AT = decltype(half_tile)::value * 64 * D;  // bytes
    auto fragment = [&](int n) { return read_lds<half8_t>(k_at[n] + AT); };
    half8_t k[AHEAD];
    float16_t acc = {};
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) k[n] = fragment(n);
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      __builtin_amdgcn_sched_barrier(0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[n % AHEAD], q[n], acc, 0, 0, 0);
      if (n + AHEAD < D / 16) k[n % AHEAD] = fragment(n + AHEAD);
      between(n);
    }
    __builtin_amdgcn_sched_barrier(0);
    return acc;
  };
  // the scores of keys [first, first + 32); edge: some may not be seen by some row
  int limit;  // this row's keys of the list at hand
  auto take = [&](const float16_t& acc, int first, bool edge, uint32_t seen) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = acc[e];
    if (edge) {
      // this lane's keys counted from 4 half: what it sees of them as bits
      const int sees = limit - first - 4 * half;
      const uint32_t left = seen >> (4 * half);
      const uint32_t bits = sees <= 0 ? 0 : sees >= 32 ? left : left & ((1u << sees) - 1);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!(bits & (1u << (8 * (e / 4) + e % 4)))) s[e] = -kInfinity;
    }
  };
  auto rescale = [&]() {
    float alpha;
    if (raise(max32(top), m, alpha, c)) {
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
      off = m == -kInfinity ? kLift : kLift - m * c;
      far = __any(!(fabsf(off) < kFar));
    }
  };
  // weights of the scores in s, made from half HALF of a tile, with the scores of the next 32 keys (half 1 - HALF of
  // the tile that k_at is at) on the matrix cores meanwhile if NEXT; then O^T += V^T P^T, and the new scores'
  // maximum meanwhile
  auto advance = [&](auto next, auto half_tile, int first, bool edge, uint32_t seen) {
    constexpr bool NEXT = decltype(next)::value;
    constexpr int HALF = decltype(half_tile)::value;
    float add = off;
    if (far) {
      const float base = m == -kInfinity ? 0.0f : m;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] -= base;
      add = kLift;
    }
    uint32_t p[8];
    auto weigh = [&](int i) {  // two scores to weights; the sum is of the weights as the product takes them
      const float2_t w = {__builtin_amdgcn_exp2f(s[2 * i] * c + add), __builtin_amdgcn_exp2f(s[2 * i + 1] * c + add)};
      p[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(w, half2_t));
      l = dot2(p[i], 0x3C003C00u, l);
      asm volatile("" : "+v"(p[i]), "+v"(l));  // made here, not where they are used
    };
    if constexpr (NEXT) {
      const float16_t acc = scores(std::integral_constant<int, 1 - HALF>{}, [&](int n) {
#pragma unroll
        for (int i = 0; i < 128 / D; ++i) weigh(128 / D * n + i);
      });
      take(acc, first, edge, seen);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) weigh(i);
    }
    auto values = [&](int n) {
      const uint32_t at = v_at[n % DB] + 2 * D * (32 * HALF + 16 * (n / DB));
      return join(read_transposed(at), read_transposed(at + 16 * D));
    };
    half8_t v[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) v[n] = values(n);
    top = -kInfinity;
#pragma unroll
    for (int n = 0; n < 2 * DB; ++n) {
      __builtin_amdgcn_sched_barrier(0);
      const int w = 4 * (n / DB);
      const half8_t weight = __builtin_bit_cast(half8_t, make_uint4(p[w], p[w + 1], p[w + 2], p[w + 3]));
      o[n % DB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[n % AHEAD], weight, o[n % DB], 0, 0, 0);
      if (n + AHEAD < 2 * DB) v[n % AHEAD] = values(n + AHEAD);
      if constexpr (NEXT) {
#pragma unroll
        for (int e = 8 / DB * n; e < 8 / DB * (n + 1); ++e) top = fmaxf(top, s[e]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };

#pragma unroll 1
  for (int from = seg.t0; from < seg.t1;) {  // the prefix's keys, the request's own
    const bool shared = r.prefix || from < lead;
    const int own = r.prefix || shared ? 0 : lead, t0 = from - own, t1 = (from < lead ? min(seg.t1, lead) : seg.t1) - own;
    from = t1 + own;
    const int bound = shared ? prefix_keys : min(r.keys, r.behind + i_last + 1);
    limit = shared ? prefix_keys : r.behind + (live ? i : i_first) + 1;
    Keys<D> keys(a, seg.head, shared ? a.prefix_pages : pages, bound, ring, lane);
    // Tiles up to `safe` are seen whole by every row of the workgroup.
    const int safe = shared ? bound : r.behind + seg.tile * x.per + 1;
    bool odd = false;
    // K of two tiles, V of two
    auto place_at = [&](int t) { return lds_at + ((t - t0) & 1) * 2 * MAT; };
    // A tile's way: its rows are found and its K loaded two tiles ahead, its V one.  `edge`: not all of it is seen by
    // all rows; `seen`: its keys that are there.
    Tile rows, rows1;
    bool edge, edge1 = false;
    uint64_t seen, seen1 = 0;
    auto find = [&](int t, Tile& to, bool& to_edge, uint64_t& to_seen) {
      const int from = t * kWideKeys;
      to.find(keys, from, r0);
      to_edge = from + kWideKeys > safe || !to.fast;
      to_seen = to.fast ? ~0ull : (uint64_t)__ballot(keys.page(from + lane) >= 0);
      to.load(keys, from, r0, keys.k, k_lane, place_at(t));
    };
    auto load_v = [&](int t, const Tile& of) { of.load(keys, t * kWideKeys, r0, keys.v, v_lane, place_at(t) + 4 * MAT); };
    auto step = [&](int t, auto more1, auto more2) {  // of tiles t + 1 and t + 2
      constexpr bool MORE1 = decltype(more1)::value, MORE2 = decltype(more2)::value;
      // V(t) has landed (K(t + 1) may be on its way), this wave's rows and after the barrier everyone's;
      // nobody reads V(t - 1) any more
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MORE1 ? N : 0) : "memory");
      _Float16* const mine = lds + ((t - t0) & 1) * MAT + 2 * MAT + r0 * D + 8 * lane;
      if ((t + 1) * kWideKeys > bound) clear_past<D, N>(mine, t * kWideKeys + r0 + lane / CH, bound);
      if (safe < bound && (t + 1) * kWideKeys > safe) {
#pragma unroll
        for (int n = 0; n < N; ++n) odd |= clear_odd(mine + n * 512);
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if constexpr (MORE1) load_v(t + 1, rows1);
      if (wave_live) {
        advance(std::true_type{}, std::integral_constant<int, 0>{}, t * kWideKeys + 32, edge, (uint32_t)(seen >> 32));
        rescale();
      }
      if constexpr (MORE1) {
        // the same of K(t + 1), V(t + 1) and K(t)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
      }
      edge = edge1;
      seen = seen1;
      if constexpr (MORE2) {
        keys.reach((t + 2) * kWideKeys);
        find(t + 2, rows1, edge1, seen1);
      }
      if (wave_live) {
#pragma unroll
        for (int n = 0; n < D / 16; ++n) k_at[n] ^= 2 * MAT;
        advance(more1, std::integral_constant<int, 1>{}, (t + 1) * kWideKeys, edge, (uint32_t)seen);
#pragma unroll
        for (int db = 0; db < DB; ++db) v_at[db] ^= 2 * MAT;
        if constexpr (MORE1) rescale();
      }
    };

    keys.begin(t0 * kWideKeys);
    settle(q);
    first_place();
    __syncthreads();  // the tiles' places are free
    find(t0, rows, edge, seen);
    load_v(t0, rows);
    if (t0 + 1 < t1) {
      keys.reach((t0 + 1) * kWideKeys);
      find(t0 + 1, rows1, edge1, seen1);
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * N) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
    }
    if (wave_live) {
      take(scores(std::integral_constant<int, 0>{}, [](int) {}), t0 * kWideKeys, edge, (uint32_t)seen);
      top = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
      rescale();
    }
    int t = t0;
    for (; t + 2 < t1; ++t) step(t, std::true_type{}, std::true_type{});
    if (t + 1 < t1) {
      step(t, std::true_type{}, std::false_type{});
      ++t;
    }
    step(t, std::false_type{}, std::false_type{});
    if (__syncthreads_or(odd)) {
      for (int key = max(t0, max(safe, 0) / kWideKeys) * kWideKeys; key < min(t1 * kWideKeys, bound); ++key) {
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
  }
  l += __shfl_xor(l, 32);
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
//
// Bound by the loads: each wave streams its keys alone, without barriers, K of the next tile on its way while V of
// this one is waited for; 8 waves a CU keep 128 KB in flight.
template <int D>
__device__ __forceinline__ void narrow_segment(const AttentionArgs& a, const Extents& x, const Request& r, const Segment& seg,
                                               const int32_t* pages, float* slot, bool whole, _Float16* lds, int32_t* ring) {
  constexpr int CH = D / 8, RPI = 512 / D, PER = D / 32, N = 2 * PER, MAT = kNarrowKeys * D, DB = D / 16;
  const int lane = here() & 63, quad = lane >> 4, row = lane & 15;
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
  Keys<D> keys(a, seg.head, pages, bound, ring, lane);
  using Tile = Rows<D, kNarrowKeys, 2>;
  uint32_t k_lane[PER], v_lane[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int kr = n * RPI + lane / CH;
    k_lane[n] = 2 * ((lane / CH) * D + 8 * key_chunk<D>(kr, lane % CH));
    v_lane[n] = 2 * ((lane / CH) * D + 8 * narrow_value_chunk<D>(kr, lane % CH));
  }
  float4_t o[DB] = {};
  float m = -kInfinity, l = 0.0f;
  bool odd = false;
  Tile rows;
  uint32_t seen, seen1 = 0;
  const uint32_t lds_at = lds_address(lds);
  auto find = [&](int t, uint32_t& to_seen) {
    rows.find(keys, t * kNarrowKeys, 0);
    to_seen = rows.fast ? ~0u : (uint32_t)__ballot(keys.page(t * kNarrowKeys + (lane & 31)) >= 0);
    rows.load(keys, t * kNarrowKeys, 0, keys.k, k_lane, lds_at);
  };
  keys.begin(seg.t0 * kNarrowKeys);
  settle(q);
  find(seg.t0, seen);
  rows.load(keys, seg.t0 * kNarrowKeys, 0, keys.v, v_lane, lds_at + 2 * MAT);
  for (int t = seg.t0; t < seg.t1; ++t) {
    const bool more = t + 1 < seg.t1;
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");  // K(t) has landed, V(t) is on its way
    float s[8];
    {
      half8_t k[2][D / 32];
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const int kr = 16 * kb + row;
          k[kb][kk] = *reinterpret_cast<const half8_t*>(lds + kr * D + 8 * key_chunk<D>(kr, 4 * kk + quad));
        }
      float4_t acc[2] = {};
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) acc[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[kb][kk], q[kk], acc[kb], 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = acc[e / 4][e % 4];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K(t) has been read
    if (more) {
      keys.reach((t + 1) * kNarrowKeys);
      find(t + 1, seen1);
    }
    // lane: row lane % 16, keys 16 (e / 4) + 4 quad + e % 4
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
    top = max32(max16(top));
    float alpha;
    if (raise(top, m, alpha, c)) {
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
    }
    const float base = m == -kInfinity ? 0.0f : m;
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2_t w = {__builtin_amdgcn_exp2f((s[2 * i] - base) * c + kLift),
                          __builtin_amdgcn_exp2f((s[2 * i + 1] - base) * c + kLift)};
      p[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(w, half2_t));
      l = dot2(p[i], 0x3C003C00u, l);
    }
    const half8_t weight = __builtin_bit_cast(half8_t, make_uint4(p[0], p[1], p[2], p[3]));
    // V(t) has landed, K(t + 1) is on its way
    if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (first + kNarrowKeys > full) {  // keys that some row does not see, or past the last
      if (first + kNarrowKeys > bound) clear_past<D, N>(lds + MAT + 8 * lane, first + lane / CH, bound);
      if (full < bound) {
#pragma unroll
        for (int n = 0; n < N; ++n) odd |= clear_odd(lds + MAT + n * 512 + 8 * lane);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    half8_t v[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int vr = 4 * quad + (row >> 2), chunk = narrow_value_chunk<D>(vr, 2 * db + ((lane & 3) >> 1));
      const uint32_t at = lds_at + 2 * (MAT + vr * D + 8 * chunk + 4 * (lane & 1));
      v[db] = join(read_transposed(at), read_transposed(at + 32 * D));
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[db], weight, o[db], 0, 0, 0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V(t) has been read
    if (more) rows.load(keys, (t + 1) * kNarrowKeys, 0, keys.v, v_lane, lds_at + 2 * MAT);
    seen = seen1;
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

// Sum over the lanes up to this one: shifts within rows of 16, then the rows' totals.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast 31 into rows 2 and 3
  return v;
}

// A token's rows in the slots of one list, as the joining kernel reads them: half a record.
struct TokenPart {
  TokenSlots at;
  Quota quota;
  __device__ bool narrow() const { return quota.few >= 0; }
};
static_assert(sizeof(TokenPart) == 2 * kRecord, "a record is two parts");

// Every workgroup plans the whole call itself (a scan over the requests' key tiles, 2 us, in place of a launch before
// this one), takes its share of the wide tiles and each of its waves its share of the narrow ones.
template <int D>
__global__ __launch_bounds__(kThreads, 2) void attend(const AttentionArgs a) {
  __shared__ __attribute__((aligned(32768))) _Float16 tiles[kWaves * 8192];  // (the places of a tile differ in one bit)
  __shared__ __attribute__((aligned(16))) int32_t rings[kWaves][128];
  __shared__ int32_t starts[3][kAttentionMaxRequests + 2];
  __shared__ int32_t sums[4][kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  Extents x = extents_of(a);
  const int lists = a.requests + 1;
  // tiles of the wide and the narrow list and items of the wide one, up to each request; the prefix comes last
  int done[3] = {0, 0, 0};
  Request all = request_of(a, x, a.requests);
  const int tokens = all.count;
  bool apart = false, broken = false;  // narrow requests, or ones without keys; offsets that do not ascend
  for (int base = 0; base < a.requests; base += kThreads) {
    const int b = base + tid;
    const bool real = b < a.requests;
    const Request r = request_of(a, x, min(b, a.requests - 1));
    const int span = real ? head_span(x, r) : 0;
    const int mine[3] = {r.narrow ? 0 : span, r.narrow ? span : 0, real ? head_items(x, r) : 0};
    const bool odd[2] = {(bool)__any(real && r.count && (r.narrow || !r.keys)), (bool)__any(real && a.offsets[b] > a.offsets[b + 1])};
    int scan[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) scan[k] = wave_scan(mine[k]);
    __syncthreads();
    if (lane == 63) {
#pragma unroll
      for (int k = 0; k < 3; ++k) sums[k][wave] = scan[k];
      sums[3][wave] = odd[0] | odd[1] << 1;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int before = done[k];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += sums[k][w];
        done[k] += sums[k][w];
      }
      if (real) starts[k][b] = before + scan[k] - mine[k];
    }
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      apart |= sums[3][w] & 1;
      broken |= sums[3][w] >> 1;
    }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) done[k] = uniform(done[k]);
  const int prefix_keys = uniform(all.keys);
  x.lead = uniform(apart ? 0 : lead_tiles(x, all, done[2]));
  if (x.lead) all.count = all.keys = 0;  // each request's items take it
  done[0] += x.lead * done[2];
  const int last[2] = {done[0], done[1]}, last_items = done[2];  // where the prefix begins
  {
    const int span = head_span(x, all);
    done[0] += all.narrow ? 0 : span;
    done[1] += all.narrow ? span : 0;
    done[2] += head_items(x, all);
  }
  x.cost = item_cost(a.kv * done[2]);
  if (x.cost + x.lead)  // each thread its own entries
    for (int b = tid; b < a.requests; b += kThreads) starts[0][b] += (x.cost + x.lead) * starts[2][b];
  done[0] += x.cost * done[2];
  if (uniform(broken)) done[0] = done[1] = 0;  // their sums may not hold: no row sees anything
  if (tid < 2) {
    starts[tid][a.requests] = tid ? last[1] : last[0] + x.cost * last_items;
    starts[tid][lists] = tid ? done[1] : done[0];
  }
  __syncthreads();
  const int positions[2] = {a.kv * done[0], a.kv * done[1]};
  const Quota wide = wide_quota(positions[0], positions[1]), narrow = narrow_quota(positions[1], wide.many);
  const bool alone = all.keys == 0;
  float* const slots = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + record_bytes(a.tokens));

  const auto requests = [&](int b) { return request_of(a, x, b); };
  auto list_of = [&](const Request& r, int b) { return r.prefix ? a.prefix_pages : a.table + (size_t)b * a.columns; };
  // what is the same in the whole wave, in scalar registers
  auto settle = [&](Walk<decltype(requests)>& walk) {
    walk.left = uniform(walk.left);
    walk.b = uniform(walk.b);
    walk.head = uniform(walk.head);
    walk.tile = uniform(walk.tile);
    walk.at = uniform(walk.at);
    walk.r.first = uniform(walk.r.first);
    walk.r.count = uniform(walk.r.count);
    walk.r.keys = uniform(walk.r.keys);
    walk.r.behind = uniform(walk.r.behind);
    walk.r.prefix = uniform(walk.r.prefix);
    walk.r.narrow = uniform(walk.r.narrow);
  };
  auto wide_list = [&]() {
    // Workgroups go round the eight XCDs in turn: neighbouring ranges, which read the same keys, are given to
    // one XCD, whose L2 then serves most of them.
    const int ranges = wide.many ? (positions[0] + wide.many - 1) / wide.many : 0, share = (ranges + 7) / 8;
    const int range = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= share || range >= ranges) return;
    Walk<decltype(requests)> walk(x, starts[0], requests, wide_items(x), range * wide.many, min((range + 1) * wide.many, positions[0]));
    Segment seg;
    for (settle(walk); walk.next(seg); walk.advance(), settle(walk)) {
      wide_segment<D>(a, x, walk.r, seg, list_of(walk.r, walk.b), prefix_keys,
                      slots + slot_floats(kWideRows, D) * (size_t)(seg.item + range), alone && !walk.r.prefix && seg.all,
                      tiles, rings[wave]);
    }
  };
  auto narrow_list = [&]() {
    float* const base = slots + slot_floats(kWideRows, D) * (size_t)wide_slots(x);
    // first the workgroups without wide work; neighbours in the list run on different CUs
    constexpr int half = kGroups / 2;
    const int stream = ((blockIdx.x < half) == (wide.many > 0) ? kStreams / 2 : 0) + wave * half + blockIdx.x % half;
    const int from = narrow.begin(stream), to = min(narrow.begin(stream + 1), positions[1]);
    if (from >= to) return;
    Walk<decltype(requests)> walk(x, starts[1], requests, narrow_items(x), from, to);
    Segment seg;
    for (settle(walk); walk.next(seg); walk.advance(), settle(walk)) {
      narrow_segment<D>(a, x, walk.r, seg, list_of(walk.r, walk.b),
                        base + slot_floats(kNarrowRows, D) * (size_t)(seg.item + stream), alone && !walk.r.prefix && seg.all,
                        tiles + wave * 2 * kNarrowKeys * D, rings[wave]);
    }
  };
  wide_list();
  __syncthreads();
  narrow_list();
  // Where the joining kernel finds each token's slots, worked out by the last workgroups, which have the least
  // other work in small calls.
  for (int t = (kGroups - 1 - (int)blockIdx.x) * kThreads + tid; t < a.tokens; t += kGroups * kThreads) {
    TokenPart* record = static_cast<TokenPart*>(a.workspace) + 2 * (size_t)t;
    const int own = find(a.offsets, a.requests, t);
    Request r = request_of(a, x, own);
    const bool real = t < tokens && t >= r.first && t < r.first + r.count;
#pragma unroll 1
    for (int part = 1; part >= 0; --part) {  // its own list, the prefix's
      TokenPart to{};
      const int b = part ? own : a.requests;
      if (real)
        to = TokenPart{token_slots(x, r, b, starts[r.narrow], r.narrow ? narrow_items(x) : wide_items(x), t), r.narrow ? narrow : wide};
      record[part] = to;
      r = all;
    }
  }
}

// Joins the segments of a row (a token's query head): out = sum_p w_p O_p / sum_p w_p l_p, w_p = exp(m_p - max m).
// D / 4 lanes, each with four dimensions, take a row, or (split > 1) as many sets of lanes share its segments and
// are added up through LDS.  A segment's maximum and sum are in one lane each, so that a lane computes one
// weight for all dimensions and the outputs' loads wait for nothing but the record.
//
// Bound by the slots' bytes in large calls (3 x 1024 tokens: 68 MB in and 17 out of 98304 rows, 28-34 us, much of it
// the workgroups' own start and index arithmetic) and by its chain of loads in small ones (5.5-6 us).  Four outputs in
// flight a lane: eight take more registers (392 us for that call, 386 with four; a prompt of 4096 tokens: 213 and 206).
template <int D, int THREADS>
__global__ __launch_bounds__(THREADS) void join_segments(const AttentionArgs a, int split) {
  constexpr int LANES = D / 4, SETS = THREADS / LANES, BATCH = 4;
  const int tid = threadIdx.x, lane = tid % LANES, set = tid / LANES, part = set % split;
  const int per = SETS / split, rows_all = a.tokens * a.heads, row = blockIdx.x * per + set / split;
  const Extents x = extents_of(a);
  const float c = a.scale * 1.44269504088896340736f;
  const int here = min(row, rows_all - 1), token = here / a.heads, head = here - token * a.heads;
  const int kv_head = head / x.share, j = head - kv_head * x.share;
  TokenPart parts[2];  // in the prefix's list and in its request's own
  __builtin_memcpy(parts, static_cast<const TokenPart*>(a.workspace) + 2 * (size_t)token, sizeof(parts));
  const float* const slots = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.workspace) + record_bytes(a.tokens));
  const float* from[2];  // the row's maximum in its first slot
  size_t stride[2];
  int count[2], sum_at[2], out_at[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const Slots s = parts[k].at.in(kv_head, parts[k].quota);
    const int rows = parts[k].narrow() ? kNarrowRows : kWideRows, at = parts[k].at.row + j;
    count[k] = s.count;
    stride[k] = slot_floats(rows, D);
    from[k] = slots + (parts[k].narrow() ? slot_floats(kWideRows, D) * (size_t)wide_slots(x) : 0) + stride[k] * (size_t)s.first + at;
    sum_at[k] = rows;
    out_at[k] = 2 * rows + at * (D - 1) + 4 * lane;
  }
  // rows whose only segment wrote the output itself
  const bool done = row >= rows_all || (count[1] == 1 && parts[0].at.tiles == 0);
  const int all = done ? 0 : count[0] + count[1];
  auto slot = [&](int p, bool k) { return from[k] + stride[k] * (size_t)(k ? p - count[0] : p); };
  // over the lanes of a set
  auto highest = [&](float v) {
#pragma unroll
    for (int step = LANES / 2; step > 0; step >>= 1) v = fmaxf(v, __shfl_xor(v, step));
    return v;
  };
  auto weight = [&](float v, float top) { return v == -kInfinity ? 0.0f : __builtin_amdgcn_exp2f((v - top) * c); };
  // this set's segments: part, part + split, ..
  float m = -kInfinity, l = 0.0f;
  float4_t o = {};
  for (int p0 = part; p0 < all; p0 += split * LANES) {
    const int n = min(LANES, (all - p0 + split - 1) / split);
    float4_t op[BATCH];
    auto load = [&](int i0) {
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int p = p0 + min(i0 + i, n - 1) * split;
        op[i] = *reinterpret_cast<const float4_t*>(slot(p, p >= count[0]) + out_at[p >= count[0]]);
      }
    };
    const int mine = p0 + min(lane, n - 1) * split;
    const float* at = slot(mine, mine >= count[0]);
    float mp = at[0], lp = at[sum_at[mine >= count[0]]];
    load(0);
    if (lane >= n) mp = -kInfinity;
    const float top = highest(fmaxf(m, mp)), w = weight(mp, top), f = weight(m, top);
    m = top;
    l = l * f + (lane < n ? w * lp : 0.0f);
    o *= f;
    for (int i0 = 0; i0 < n; i0 += BATCH) {
      if (i0) load(i0);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const float wi = __shfl(w, min(i0 + i, LANES - 1), LANES);
        if (i0 + i < n) o += op[i] * wi;
      }
    }
  }
#pragma unroll
  for (int step = LANES / 2; step > 0; step >>= 1) l += __shfl_xor(l, step);
  if (split > 1) {  // split <= LANES
    __shared__ float4_t outs[THREADS];
    __shared__ float2 stats[SETS];
    outs[tid] = o;
    if (lane == 0) stats[set] = make_float2(m, l);
    __syncthreads();
    if (part) return;
    const float2 other = stats[set + min(lane, split - 1)];
    const float ms = lane < split ? other.x : -kInfinity;
    const float w = weight(ms, highest(ms));
    l = lane < split ? w * other.y : 0.0f;
#pragma unroll
    for (int step = LANES / 2; step > 0; step >>= 1) l += __shfl_xor(l, step);
    o = float4_t{};
    for (int s = 0; s < split; ++s) o += outs[tid + s * LANES] * __shfl(w, s, LANES);
  }
  if (done) return;
  const float4_t v = o * (l == 0.0f ? 0.0f : 1.0f / l);
  *reinterpret_cast<uint2*>(static_cast<_Float16*>(a.out) + (size_t)row * D + 4 * lane) =
      make_uint2(half2_from_fp32(v[0], v[1]), half2_from_fp32(v[2], v[3]));
}

template <int D>
hipError_t launch_dim(const AttentionArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((attend<D>), dim3(kGroups), dim3(kThreads), 0, stream, a);
  hipError_t status = hipGetLastError();
  if (status != hipSuccess) return status;
  // Few rows: more sets of lanes for each, to 8192 or more in all (64 requests behind 16384 keys, 2048 rows of 34
  // segments: 56 us for the call, at 2048 sets as well, at 32768 65; with heads of 64: 34.6, 35.7, 38.5; 32 requests of up to
  // 2000 keys: 37.9, 37.1, 41.2).
  constexpr int lanes = D / 4;
  const int rows = a.tokens * a.heads;
  int split = 1;
  while (split < 16 && (int64_t)rows * split < 8192) split *= 2;
  const int threads = split * lanes > 256 ? 512 : 256, per = threads / lanes / split;
  const dim3 grid((unsigned)(((int64_t)rows + per - 1) / per));
  if (threads == 512) hipLaunchKernelGGL((join_segments<D, 512>), grid, dim3(512), 0, stream, a, split);
  else hipLaunchKernelGGL((join_segments<D, 256>), grid, dim3(256), 0, stream, a, split);
  return hipGetLastError();
}

}  // namespace

size_t attention_workspace(const AttentionArgs& a) {
  const Extents x = extents_of(a);
  return record_bytes(a.tokens) + 4 * (slot_floats(kWideRows, a.dim) * (size_t)wide_slots(x) +
                                       slot_floats(kNarrowRows, a.dim) * (size_t)narrow_slots(x));
}

hipError_t launch_attention(const AttentionArgs& a, hipStream_t stream) {
  return a.dim == 64 ? launch_dim<64>(a, stream) : a.dim == 128 ? launch_dim<128>(a, stream) : hipErrorInvalidValue;
}

}  // namespace tensor_paged
