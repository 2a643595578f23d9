// Host-side launch descriptors of the paged-cache operators.  Shapes have been validated by the
// C-ABI entry points before these run.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace tensor_paged {

struct SlotsArgs {
  const int32_t *lengths, *counts, *start, *free, *free_count, *table;
  int32_t *offsets, *lengths_out, *positions, *slots, *table_out, *free_left;
  int requests, columns, tokens, free_extent, page_shift;
};
// A launch has at most 2^32 - 1 threads along x.
constexpr int64_t kMostThreads = ((int64_t)1 << 32) - 1;
constexpr int kSlotsThreads = 256;  // of a request
hipError_t launch_slots(const SlotsArgs& args, hipStream_t stream);

struct RotaryArgs {
  const void *q, *k, *v;  // [tokens, heads, dim], [tokens, kv, dim] twice (v: nullptr without the store)
  const int32_t *positions, *slots;
  const float* angles;    // [reach, rotated]: cosines, then sines
  void *q_out, *k_out, *v_out;  // k_out, v_out: the caches with the store
  int tokens, heads, kv, dim, rotated, reach, pages, page_shift;
  bool interleaved, inverse, in_f32, out_f32;
};
int rotary_threads(const RotaryArgs& args);  // of a token's workgroup
hipError_t launch_rotary(const RotaryArgs& args, hipStream_t stream);

struct AttentionArgs {
  const void *q, *k_cache, *v_cache;  // fp16 [tokens, heads, dim], [pages, kv, page size, dim] twice
  void* out;                          // fp16 [tokens, heads, dim]
  const int32_t *offsets, *lengths;   // [requests + 1], [requests]
  const int32_t *table, *prefix_pages, *prefix_length;  // [requests, columns], [prefix_columns], [1]
  void* workspace;
  int tokens, heads, kv, dim, pages, page_shift, requests, columns, prefix_columns;
  float scale;
};
constexpr int kAttentionMaxRequests = 1024;
constexpr int kAttentionMaxShare = 128;  // query heads of one key head
// Bytes of workspace a call needs (tokens, requests, heads, kv, dim; the other fields are not read).
size_t attention_workspace(const AttentionArgs& args);
hipError_t launch_attention(const AttentionArgs& args, hipStream_t stream);

}  // namespace tensor_paged
