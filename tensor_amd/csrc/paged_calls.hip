// C-ABI entry points of the paged-cache operators: descriptor checks, then the launch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>

#include "buffer_check.h"
#include "paged_launch.h"
#include "paged_plan.h"

namespace {

using namespace tensor_abi;

int32_t check_ints(const TensorArgumentV1& arg, const char* name, int ordinal, int64_t* shape, uint32_t rank,
                   TensorErrorV1* error) {
  CHECK(check_buffer(arg, name, ordinal, TENSOR_INT32, shape, rank, 4, error));
  for (uint32_t axis = 0; axis < rank; ++axis)
    if (shape[axis] >= (int64_t)1 << 31) return fail(error, TENSOR_ERROR_ARGUMENT, "%s: too large", name);
  return TENSOR_OK;
}

// log2 of a page size: a power of two from 1 to 1024 tokens; -1 otherwise
int page_shift(int64_t size) {
  for (int shift = 0; shift <= 10; ++shift)
    if (size == (int64_t)1 << shift) return shift;
  return -1;
}

int32_t slots_call(const TensorCallV1* call, TensorErrorV1* error) {
  ok(error);
  CHECK(check_call(call, 14, error));
  const int ordinal = call->stream.device_ordinal;
  const TensorArgumentV1* a = call->arguments;
  uint64_t size = 0;
  CHECK(check_u32(a[13], "page_size", &size, error));
  const int shift = page_shift((int64_t)size);
  if (shift < 0) return fail(error, TENSOR_ERROR_ARGUMENT, "page_size: must be a power of two from 1 to 1024");
  if (a[6].kind != TENSOR_ARG_SCALAR || a[6].dtype != TENSOR_INT32)
    return fail(error, TENSOR_ERROR_ARGUMENT, "T: wrong argument kind or dtype");
  if (a[6].scalar >> 31 || !a[6].scalar) return fail(error, TENSOR_ERROR_ARGUMENT, "T: must be a positive int32");
  int64_t tokens[1] = {(int64_t)a[6].scalar}, one[1] = {1}, requests[1] = {-1}, free[1] = {-1}, table[2] = {-1, -1};
  CHECK(check_ints(a[0], "lengths", ordinal, requests, 1, error));
  if (requests[0] * tensor_paged::kSlotsThreads > tensor_paged::kMostThreads)
    return fail(error, TENSOR_ERROR_ARGUMENT, "lengths: less than 2^24 requests");
  table[0] = requests[0];
  int64_t ends[1] = {requests[0] + 1};
  CHECK(check_ints(a[1], "counts", ordinal, requests, 1, error));
  CHECK(check_ints(a[2], "start", ordinal, one, 1, error));
  CHECK(check_ints(a[3], "free", ordinal, free, 1, error));
  CHECK(check_ints(a[4], "free_count", ordinal, one, 1, error));
  CHECK(check_ints(a[5], "table", ordinal, table, 2, error));
  CHECK(check_ints(a[7], "offsets", ordinal, ends, 1, error));
  CHECK(check_ints(a[8], "lengths_out", ordinal, requests, 1, error));
  CHECK(check_ints(a[9], "positions", ordinal, tokens, 1, error));
  CHECK(check_ints(a[10], "slots", ordinal, tokens, 1, error));
  CHECK(check_ints(a[11], "table_out", ordinal, table, 2, error));
  CHECK(check_ints(a[12], "free_left", ordinal, one, 1, error));
  // Every workgroup sums the earlier requests' lengths and counts; only the table's entries are each one's own.
  CHECK(check_apart(call, {{7, "offsets", -1}, {8, "lengths_out", -1}, {9, "positions", -1}, {10, "slots", -1},
                           {11, "table_out", 5}, {12, "free_left", -1}}, error));
  CHECK(check_device(call, error));
  tensor_paged::SlotsArgs args{};
  args.lengths = pointer<const int32_t>(a[0]);
  args.counts = pointer<const int32_t>(a[1]);
  args.start = pointer<const int32_t>(a[2]);
  args.free = pointer<const int32_t>(a[3]);
  args.free_count = pointer<const int32_t>(a[4]);
  args.table = pointer<const int32_t>(a[5]);
  args.offsets = pointer<int32_t>(a[7]);
  args.lengths_out = pointer<int32_t>(a[8]);
  args.positions = pointer<int32_t>(a[9]);
  args.slots = pointer<int32_t>(a[10]);
  args.table_out = pointer<int32_t>(a[11]);
  args.free_left = pointer<int32_t>(a[12]);
  args.requests = (int)requests[0];
  args.columns = (int)table[1];
  args.tokens = (int)tokens[0];
  args.free_extent = (int)free[0];
  args.page_shift = shift;
  const hipError_t status = tensor_paged::launch_slots(args, stream_of(call));
  return status == hipSuccess ? TENSOR_OK : hip_fail(error, status, "slot map launch");
}

// The two rotary calls: [q, k, positions, angles, q_out, k_out, layout, inverse], and with the store
// [q, k, v, positions, slots, angles, q_out, k_cache, v_cache, layout].
int32_t rotary_call(const TensorCallV1* call, TensorErrorV1* error, bool store) {
  ok(error);
  CHECK(check_call(call, store ? 10 : 8, error));
  const int ordinal = call->stream.device_ordinal;
  const TensorArgumentV1* a = call->arguments;
  uint64_t layout = 0, inverse = 0;
  CHECK(check_u32(a[store ? 9 : 6], "layout", &layout, error));
  if (layout > 1) return fail(error, TENSOR_ERROR_ARGUMENT, "layout: 0 (halves) or 1 (interleaved)");
  if (!store) {
    CHECK(check_u32(a[7], "inverse", &inverse, error));
    if (inverse > 1) return fail(error, TENSOR_ERROR_ARGUMENT, "inverse: 0 or 1");
  }
  const uint32_t dtype = a[0].dtype;
  if (dtype != TENSOR_FLOAT16 && dtype != TENSOR_FLOAT32)
    return fail(error, TENSOR_ERROR_ARGUMENT, "q: wrong argument kind or dtype");
  const uint32_t out_dtype = store ? TENSOR_FLOAT16 : dtype;
  const TensorArgumentV1 &positions = a[store ? 3 : 2], &angles = a[store ? 5 : 3], &q_out = a[store ? 6 : 4];
  int64_t q[3] = {-1, -1, -1};
  CHECK(check_buffer(a[0], "q", ordinal, dtype, q, 3, 16, error));
  int64_t k[3] = {q[0], -1, q[2]}, tokens[1] = {q[0]}, table[2] = {-1, -1};
  CHECK(check_buffer(a[1], "k", ordinal, dtype, k, 3, 16, error));
  CHECK(check_ints(positions, "positions", ordinal, tokens, 1, error));
  CHECK(check_buffer(angles, "angles", ordinal, TENSOR_FLOAT32, table, 2, 16, error));
  if (table[1] % 2 || table[1] > q[2] || table[0] >= (int64_t)1 << 31)
    return fail(error, TENSOR_ERROR_ARGUMENT, "angles: an even number of columns, at most the head's dimensions");
  if (q[0] >= (int64_t)1 << 31 || q[1] >= 1 << 16 || k[1] >= 1 << 16 || q[2] > 4096 || (q[1] + 2 * k[1]) * q[2] > 255 * 65535)
    return fail(error, TENSOR_ERROR_ARGUMENT, "q, k: too many heads, or heads of more than 4096 dimensions");
  CHECK(check_buffer(q_out, "q_out", ordinal, out_dtype, q, 3, 16, error));
  tensor_paged::RotaryArgs args{};
  if (store) {
    CHECK(check_buffer(a[2], "v", ordinal, dtype, k, 3, 16, error));
    CHECK(check_ints(a[4], "slots", ordinal, tokens, 1, error));
    int64_t cache[4] = {-1, k[1], -1, k[2]};
    CHECK(check_buffer(a[7], "k_cache", ordinal, TENSOR_FLOAT16, cache, 4, 16, error));
    CHECK(check_buffer(a[8], "v_cache", ordinal, TENSOR_FLOAT16, cache, 4, 16, error));
    args.page_shift = page_shift(cache[2]);
    if (args.page_shift < 0 || cache[0] >= (int64_t)1 << 31)
      return fail(error, TENSOR_ERROR_ARGUMENT, "k_cache: pages of a power of two from 1 to 1024 tokens");
    CHECK(check_apart(call, {{6, "q_out", 0}, {7, "k_cache", -1}, {8, "v_cache", -1}}, error));
    args.pages = (int)cache[0];
    args.v = pointer<const void>(a[2]);
    args.slots = pointer<const int32_t>(a[4]);
    args.k_out = pointer<void>(a[7]);
    args.v_out = pointer<void>(a[8]);
  } else {
    CHECK(check_buffer(a[5], "k_out", ordinal, out_dtype, k, 3, 16, error));
    CHECK(check_apart(call, {{4, "q_out", 0}, {5, "k_out", 1}}, error));
    args.k_out = pointer<void>(a[5]);
  }
  args.heads = (int)q[1];
  args.kv = (int)k[1];
  args.dim = (int)q[2];
  args.rotated = (int)table[1];
  if (q[0] * tensor_paged::rotary_threads(args) > tensor_paged::kMostThreads)
    return fail(error, TENSOR_ERROR_ARGUMENT, "q: too many tokens for one call");
  CHECK(check_device(call, error));
  args.q = pointer<const void>(a[0]);
  args.k = pointer<const void>(a[1]);
  args.positions = pointer<const int32_t>(positions);
  args.angles = pointer<const float>(angles);
  args.q_out = pointer<void>(q_out);
  args.tokens = (int)q[0];
  args.reach = (int)table[0];
  args.interleaved = layout == 1;
  args.inverse = inverse == 1;
  args.in_f32 = dtype == TENSOR_FLOAT32;
  args.out_f32 = out_dtype == TENSOR_FLOAT32;
  const hipError_t status = tensor_paged::launch_rotary(args, stream_of(call));
  return status == hipSuccess ? TENSOR_OK : hip_fail(error, status, "rotary launch");
}

// Sizes an attention call takes, in the same words for the call and the workspace query.
int32_t check_attention(int64_t tokens, int64_t requests, int64_t heads, int64_t kv, int64_t dim, TensorErrorV1* error) {
  if (dim != 64 && dim != 128) return fail(error, TENSOR_ERROR_ARGUMENT, "heads of 64 or 128 dimensions");
  if (kv < 1 || heads < 1 || heads % kv || heads / kv > tensor_paged::kAttentionMaxShare || heads >= 1 << 16)
    return fail(error, TENSOR_ERROR_ARGUMENT, "heads: a multiple of the key heads, at most %d times as many",
                tensor_paged::kAttentionMaxShare);
  if (requests < 1 || requests > tensor_paged::kAttentionMaxRequests)
    return fail(error, TENSOR_ERROR_ARGUMENT, "1 to %d requests", tensor_paged::kAttentionMaxRequests);
  // (the joining kernel has a thread for four values, in workgroups of up to 512)
  if (tokens < 1 || tokens > 1 << 20 || tokens * heads * (dim / 4) > tensor_paged::kMostThreads - 512)
    return fail(error, TENSOR_ERROR_ARGUMENT, "q: 1 to 2^20 tokens, less than 2^34 - 2048 values");
  return TENSOR_OK;
}

int32_t attention_call(const TensorCallV1* call, TensorErrorV1* error) {
  ok(error);
  CHECK(check_call(call, 11, error));
  const int ordinal = call->stream.device_ordinal;
  const TensorArgumentV1* a = call->arguments;
  if (a[10].kind != TENSOR_ARG_SCALAR || a[10].dtype != TENSOR_FLOAT32)
    return fail(error, TENSOR_ERROR_ARGUMENT, "scale: wrong argument kind or dtype");
  if (a[10].scalar >> 32) return fail(error, TENSOR_ERROR_ARGUMENT, "scale: noncanonical scalar payload");
  float scale;
  const uint32_t bits = (uint32_t)a[10].scalar;
  std::memcpy(&scale, &bits, 4);
  if (!std::isfinite(scale) || scale < 0.0f)
    return fail(error, TENSOR_ERROR_ARGUMENT, "scale: must be positive and finite, or 0 for 1 / sqrt(dimensions)");
  int64_t q[3] = {-1, -1, -1}, cache[4] = {-1, -1, -1, -1}, ends[1] = {-1}, table[2] = {-1, -1}, prefix[1] = {-1}, one[1] = {1};
  CHECK(check_buffer(a[0], "q", ordinal, TENSOR_FLOAT16, q, 3, 16, error));
  cache[3] = q[2];
  CHECK(check_buffer(a[1], "k_cache", ordinal, TENSOR_FLOAT16, cache, 4, 16, error));
  CHECK(check_buffer(a[2], "v_cache", ordinal, TENSOR_FLOAT16, cache, 4, 16, error));
  CHECK(check_ints(a[3], "offsets", ordinal, ends, 1, error));
  int64_t requests[1] = {ends[0] - 1};
  CHECK(check_attention(q[0], requests[0], q[1], cache[1], q[2], error));
  CHECK(check_ints(a[4], "lengths", ordinal, requests, 1, error));
  table[0] = requests[0];
  CHECK(check_ints(a[5], "table", ordinal, table, 2, error));
  CHECK(check_ints(a[6], "prefix_pages", ordinal, prefix, 1, error));
  CHECK(check_ints(a[7], "prefix_length", ordinal, one, 1, error));
  CHECK(check_buffer(a[9], "out", ordinal, TENSOR_FLOAT16, q, 3, 16, error));
  tensor_paged::AttentionArgs args{};
  args.page_shift = page_shift(cache[2]);
  if (args.page_shift < 0 || cache[0] >= (int64_t)1 << 31)
    return fail(error, TENSOR_ERROR_ARGUMENT, "k_cache: pages of a power of two from 1 to 1024 tokens");
  args.tokens = (int)q[0];
  args.heads = (int)q[1];
  args.dim = (int)q[2];
  args.kv = (int)cache[1];
  args.pages = (int)cache[0];
  args.requests = (int)requests[0];
  // tables hold at most 2^24 tokens: key indices and a request's count of key tiles stay in 32 bits
  const int64_t reach = (int64_t)1 << 24;
  if (table[1] << args.page_shift > reach || prefix[0] << args.page_shift > reach)
    return fail(error, TENSOR_ERROR_ARGUMENT, "table, prefix_pages: more than 2^24 tokens of a request");
  args.columns = (int)table[1];
  args.prefix_columns = (int)prefix[0];
  if (tensor_paged::most_tiles(tensor_paged::extents(args.tokens, args.requests, args.heads, args.kv, args.page_shift,
                                                     args.columns, args.prefix_columns)) >= (int64_t)1 << 31)
    return fail(error, TENSOR_ERROR_ARGUMENT, "too many tokens, heads, requests and table columns for one call");
  int64_t workspace[1] = {-1};
  CHECK(check_buffer(a[8], "workspace", ordinal, TENSOR_UINT8, workspace, 1, 256, error));
  const size_t need = tensor_paged::attention_workspace(args);
  if ((uint64_t)workspace[0] < need)
    return fail(error, TENSOR_ERROR_ARGUMENT, "workspace: the call needs %zu bytes, %lld available", need,
                (long long)workspace[0]);
  CHECK(check_apart(call, {{8, "workspace", -1}, {9, "out", 0}}, error));  // (a row's segment reads its queries first)
  CHECK(check_device(call, error));
  args.q = pointer<const void>(a[0]);
  args.k_cache = pointer<const void>(a[1]);
  args.v_cache = pointer<const void>(a[2]);
  args.offsets = pointer<const int32_t>(a[3]);
  args.lengths = pointer<const int32_t>(a[4]);
  args.table = pointer<const int32_t>(a[5]);
  args.prefix_pages = pointer<const int32_t>(a[6]);
  args.prefix_length = pointer<const int32_t>(a[7]);
  args.workspace = pointer<void>(a[8]);
  args.out = pointer<void>(a[9]);
  args.scale = scale > 0.0f ? scale : 1.0f / std::sqrt((float)args.dim);
  const hipError_t status = tensor_paged::launch_attention(args, stream_of(call));
  return status == hipSuccess ? TENSOR_OK : hip_fail(error, status, "paged attention launch");
}

}  // namespace

extern "C" {

int32_t tensor_paged_slots_v1(const TensorCallV1* call, TensorErrorV1* error) { return slots_call(call, error); }

int32_t tensor_rotary_v1(const TensorCallV1* call, TensorErrorV1* error) { return rotary_call(call, error, false); }

int32_t tensor_rotary_store_v1(const TensorCallV1* call, TensorErrorV1* error) {
  return rotary_call(call, error, true);
}

int32_t tensor_paged_attention_v1(const TensorCallV1* call, TensorErrorV1* error) { return attention_call(call, error); }

int32_t tensor_paged_attention_workspace_v1(int64_t tokens, int64_t requests, int64_t heads, int64_t kv_heads,
                                            int64_t dim, uint64_t* bytes, TensorErrorV1* error) {
  if (!bytes) return fail(error, TENSOR_ERROR_ARGUMENT, "invalid workspace query");
  CHECK(check_attention(tokens, requests, heads, kv_heads, dim, error));
  tensor_paged::AttentionArgs args{};
  args.tokens = (int)tokens;
  args.requests = (int)requests;
  args.heads = (int)heads;
  args.kv = (int)kv_heads;
  args.dim = (int)dim;
  *bytes = tensor_paged::attention_workspace(args);
  return ok(error);
}

}  // extern "C"
