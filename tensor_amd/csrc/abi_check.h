// Status reporting and descriptor checks shared by the C-ABI entry points.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "tensor_hip.h"

namespace tensor_abi {

inline int32_t fail(TensorErrorV1* error, int32_t code, const char* format, ...) {
  if (error) {
    error->code = code;
    va_list args;
    va_start(args, format);
    std::vsnprintf(error->message, sizeof(error->message), format, args);
    va_end(args);
  }
  return code;
}

inline int32_t ok(TensorErrorV1* error) {
  if (error) {
    error->code = TENSOR_OK;
    error->message[0] = 0;
  }
  return TENSOR_OK;
}

inline int32_t hip_fail(TensorErrorV1* error, hipError_t status, const char* what) {
  return fail(error, TENSOR_ERROR_PROVIDER, "%s: %s (%s, %d)", what, hipGetErrorString(status),
              hipGetErrorName(status), (int)status);
}

// Common header checks of every kernel call (src/tensor/compiler/cpu.py:59-66).
// Pure descriptor checks only: nothing here touches the HIP runtime, so every
// argument error is reported before any device state is consulted.
inline int32_t check_call(const TensorCallV1* call, uint32_t arguments, TensorErrorV1* error) {
  if (!call || call->abi_version != TENSOR_ABI_VERSION || call->struct_size < sizeof(TensorCallV1))
    return fail(error, TENSOR_ERROR_ABI, "unsupported call ABI");
  if (call->flags || call->argument_count != arguments || !call->arguments)
    return fail(error, TENSOR_ERROR_ARGUMENT, "invalid argument count or flags");
  if (call->stream.device_type != TENSOR_DEVICE_ROCM || call->stream.device_ordinal < 0)
    return fail(error, TENSOR_ERROR_PROVIDER, "ROCm calls need a ROCm stream");
  return TENSOR_OK;
}

// The stream's ordinal must be the calling thread's current HIP device.
inline int32_t check_device(const TensorCallV1* call, TensorErrorV1* error) {
  int device = -1;
  hipError_t status = hipGetDevice(&device);
  if (status != hipSuccess) return hip_fail(error, status, "hipGetDevice");
  if (call->stream.device_ordinal != device)
    return fail(error, TENSOR_ERROR_PROVIDER, "stream ordinal %d is not the current device %d",
                (int)call->stream.device_ordinal, device);
  return TENSOR_OK;
}

inline int32_t check_u32(const TensorArgumentV1& arg, const char* name, uint64_t* value, TensorErrorV1* error) {
  if (arg.kind != TENSOR_ARG_SCALAR || arg.dtype != TENSOR_UINT32)
    return fail(error, TENSOR_ERROR_ARGUMENT, "%s: wrong argument kind or dtype", name);
  if (arg.scalar >> 32) return fail(error, TENSOR_ERROR_ARGUMENT, "%s: noncanonical scalar payload", name);
  *value = arg.scalar;
  return TENSOR_OK;
}

}  // namespace tensor_abi
