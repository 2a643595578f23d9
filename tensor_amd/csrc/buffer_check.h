// Checks of the buffers of an operator's call: contiguous ones of a given type and shape, written ones apart from
// the others.
#pragma once

#include <hip/hip_runtime.h>

#include "abi_check.h"

#define CHECK(expr) \
  if (int32_t s_ = (expr)) return s_

namespace tensor_abi {

// A contiguous device buffer of one dtype and the given shape; an extent of -1 is any, and is
// stored there.  Buffers of four-byte integers need 4-byte alignment, the others `align`.
inline int32_t check_buffer(const TensorArgumentV1& arg, const char* name, int ordinal, uint32_t dtype, int64_t* shape,
                            uint32_t rank, uint64_t align, TensorErrorV1* error) {
  const TensorBufferV1& b = arg.buffer;
  if (arg.kind != TENSOR_ARG_BUFFER || arg.dtype != dtype || b.dtype != dtype)
    return fail(error, TENSOR_ERROR_ARGUMENT, "%s: wrong argument kind or dtype", name);
  if (b.device_type != TENSOR_DEVICE_ROCM || b.device_ordinal != ordinal || !b.address || b.address % align ||
      b.rank != rank || !b.shape || !b.strides)
    return fail(error, TENSOR_ERROR_ARGUMENT, "%s: invalid buffer descriptor", name);
  uint64_t bytes = dtype == TENSOR_UINT8 ? 1 : dtype == TENSOR_FLOAT16 ? 2 : 4;
  for (int axis = (int)rank - 1; axis >= 0; --axis) {
    if (b.shape[axis] <= 0 || b.strides[axis] != (int64_t)bytes || (shape[axis] >= 0 && shape[axis] != b.shape[axis]))
      return fail(error, TENSOR_ERROR_ARGUMENT, "%s: shape, stride or size mismatch", name);
    if ((uint64_t)b.shape[axis] > ((uint64_t)1 << 46) / bytes)
      return fail(error, TENSOR_ERROR_ARGUMENT, "%s: too large", name);
    shape[axis] = b.shape[axis];
    bytes *= (uint64_t)b.shape[axis];
  }
  if (b.byte_size < bytes) return fail(error, TENSOR_ERROR_ARGUMENT, "%s: insufficient buffer storage", name);
  return TENSOR_OK;
}

// A buffer that a call writes: its argument, and the one (-1: none) that it may be itself, whose every value is read by
// the thread that writes it.
struct Written {
  int at;
  const char* name;
  int twin;
};

// Written buffers share no memory with the call's others, which other workgroups may not have read yet.
template <size_t N>
int32_t check_apart(const TensorCallV1* call, const Written (&written)[N], TensorErrorV1* error) {
  auto bytes = [&](uint32_t i) {
    const TensorBufferV1& b = call->arguments[i].buffer;
    return (uint64_t)b.shape[0] * (uint64_t)b.strides[0];  // contiguous (check_buffer)
  };
  for (const Written& w : written) {
    const uint64_t from = call->arguments[w.at].buffer.address, to = from + bytes(w.at);
    for (uint32_t i = 0; i < call->argument_count; ++i) {
      if ((int)i == w.at || call->arguments[i].kind != TENSOR_ARG_BUFFER) continue;
      const uint64_t other = call->arguments[i].buffer.address, end = other + bytes(i);
      if (end <= from || to <= other || ((int)i == w.twin && other == from && end == to)) continue;
      return fail(error, TENSOR_ERROR_ARGUMENT, "%s: written, and shares memory with argument %u", w.name, i);
    }
  }
  return TENSOR_OK;
}

template <typename T>
T* pointer(const TensorArgumentV1& arg) {
  return reinterpret_cast<T*>(arg.buffer.address);
}

inline hipStream_t stream_of(const TensorCallV1* call) { return reinterpret_cast<hipStream_t>(call->stream.handle); }

}  // namespace tensor_abi
