// C-ABI entry points of the norm and the 8-bit operators: descriptor checks, then the launch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>

#include "buffer_check.h"
#include "fp8_launch.h"

namespace {

using namespace tensor_abi;
using tensor_fp8::blocks_of;

constexpr int64_t kMostRows = ((int64_t)1 << 31) - 1;

int32_t check_values(const TensorArgumentV1& arg, const char* name, int ordinal, int64_t* shape, uint32_t rank,
                     TensorErrorV1* error) {
  if (arg.dtype != TENSOR_FLOAT16 && arg.dtype != TENSOR_FLOAT32)
    return fail(error, TENSOR_ERROR_ARGUMENT, "%s: wrong argument kind or dtype", name);
  return check_buffer(arg, name, ordinal, arg.dtype, shape, rank, 16, error);
}

// [x, (residual,) weight, out, (scales,) (residual_out,) eps]
int32_t norm_call(const TensorCallV1* call, TensorErrorV1* error, bool codes) {
  ok(error);
  const int plain = codes ? 5 : 4;
  const bool residual = call && call->argument_count == (uint32_t)plain + 2;
  CHECK(check_call(call, plain + (residual ? 2 : 0), error));
  const int ordinal = call->stream.device_ordinal;
  const TensorArgumentV1* a = call->arguments;
  const int weight = residual ? 2 : 1, out = weight + 1, scales = out + 1, residual_out = out + 1 + codes;
  const TensorArgumentV1& last = a[plain + (residual ? 2 : 0) - 1];
  if (last.kind != TENSOR_ARG_SCALAR || last.dtype != TENSOR_FLOAT32)
    return fail(error, TENSOR_ERROR_ARGUMENT, "eps: wrong argument kind or dtype");
  if (last.scalar >> 32) return fail(error, TENSOR_ERROR_ARGUMENT, "eps: noncanonical scalar payload");
  tensor_fp8::NormArgs args{};
  const uint32_t bits = (uint32_t)last.scalar;
  std::memcpy(&args.eps, &bits, 4);
  if (!std::isfinite(args.eps) || args.eps < tensor_fp8::kNormLeastEps)
    return fail(error, TENSOR_ERROR_ARGUMENT, "eps: must be finite and 2^-100 at least");
  int64_t x[2] = {-1, -1};
  CHECK(check_values(a[0], "x", ordinal, x, 2, error));
  int64_t width[1] = {x[1]};
  if (x[0] > kMostRows) return fail(error, TENSOR_ERROR_ARGUMENT, "x: too many rows");
  if (x[1] > tensor_fp8::kNormMaxWidth)
    return fail(error, TENSOR_ERROR_ARGUMENT, "x: rows of at most %d values", tensor_fp8::kNormMaxWidth);
  if (residual) {
    CHECK(check_values(a[1], "residual", ordinal, x, 2, error));
    CHECK(check_buffer(a[residual_out], "residual_out", ordinal, a[1].dtype, x, 2, 16, error));
  }
  CHECK(check_buffer(a[weight], "weight", ordinal, TENSOR_FLOAT32, width, 1, 16, error));
  if (codes) {
    int64_t blocks[2] = {blocks_of(x[1]), x[0]};
    CHECK(check_buffer(a[out], "codes", ordinal, TENSOR_UINT8, x, 2, 16, error));
    CHECK(check_buffer(a[scales], "scales", ordinal, TENSOR_FLOAT32, blocks, 2, 16, error));
    args.scales = pointer<float>(a[scales]);
  } else {
    CHECK(check_values(a[out], "out", ordinal, x, 2, error));
  }
  // a row is read before it is written, by the threads that write it
  const int twin = !codes && a[out].dtype == a[0].dtype ? 0 : -1;
  if (residual && codes) {
    CHECK(check_apart(call, {{out, "codes", -1}, {scales, "scales", -1}, {residual_out, "residual_out", 1}}, error));
  } else if (residual) {
    CHECK(check_apart(call, {{out, "out", twin}, {residual_out, "residual_out", 1}}, error));
  } else if (codes) {
    CHECK(check_apart(call, {{out, "codes", -1}, {scales, "scales", -1}}, error));
  } else {
    CHECK(check_apart(call, {{out, "out", twin}}, error));
  }
  args.x = pointer<const void>(a[0]);
  args.residual = residual ? pointer<const void>(a[1]) : nullptr;
  args.residual_out = residual ? pointer<void>(a[residual_out]) : nullptr;
  args.weight = pointer<const float>(a[weight]);
  args.out = pointer<void>(a[out]);
  args.rows = (int)x[0];
  args.width = (int)x[1];
  args.x_f32 = a[0].dtype == TENSOR_FLOAT32;
  args.residual_f32 = residual && a[1].dtype == TENSOR_FLOAT32;
  args.out_f32 = a[out].dtype == TENSOR_FLOAT32;
  if (tensor_fp8::norm_threads(args) > tensor_fp8::kMostThreads)
    return fail(error, TENSOR_ERROR_ARGUMENT, "x: too many rows for one call");
  CHECK(check_device(call, error));
  const hipError_t status = tensor_fp8::launch_norm(args, stream_of(call));
  return status == hipSuccess ? TENSOR_OK : hip_fail(error, status, "norm launch");
}

// [x, codes, scales, gated]
int32_t quantize_call(const TensorCallV1* call, TensorErrorV1* error) {
  ok(error);
  CHECK(check_call(call, 4, error));
  const int ordinal = call->stream.device_ordinal;
  const TensorArgumentV1* a = call->arguments;
  uint64_t gated = 0;
  CHECK(check_u32(a[3], "gated", &gated, error));
  if (gated > 1) return fail(error, TENSOR_ERROR_ARGUMENT, "gated: 0 or 1");
  int64_t x[2] = {-1, -1}, codes[2] = {-1, -1};
  CHECK(check_values(a[0], "x", ordinal, x, 2, error));
  if (gated && x[1] % 2) return fail(error, TENSOR_ERROR_ARGUMENT, "x: gated rows hold as many gates as values");
  codes[0] = x[0];
  codes[1] = gated ? x[1] / 2 : x[1];
  if (x[0] > kMostRows || codes[1] > (int64_t)1 << 30) return fail(error, TENSOR_ERROR_ARGUMENT, "x: too large");
  int64_t scales[2] = {blocks_of(codes[1]), x[0]};
  CHECK(check_buffer(a[1], "codes", ordinal, TENSOR_UINT8, codes, 2, 16, error));
  CHECK(check_buffer(a[2], "scales", ordinal, TENSOR_FLOAT32, scales, 2, 16, error));
  CHECK(check_apart(call, {{1, "codes", -1}, {2, "scales", -1}}, error));
  tensor_fp8::QuantizeArgs args{};
  args.x = pointer<const void>(a[0]);
  args.codes = pointer<uint8_t>(a[1]);
  args.scales = pointer<float>(a[2]);
  args.rows = (int)x[0];
  args.width = (int)codes[1];
  args.gated = gated == 1;
  args.x_f32 = a[0].dtype == TENSOR_FLOAT32;
  if (tensor_fp8::quantize_threads(args) > tensor_fp8::kMostThreads)
    return fail(error, TENSOR_ERROR_ARGUMENT, "x: too large for one call");
  CHECK(check_device(call, error));
  const hipError_t status = tensor_fp8::launch_quantize(args, stream_of(call));
  return status == hipSuccess ? TENSOR_OK : hip_fail(error, status, "quantize launch");
}

// [x, x_scales, w, w_scales, out]
int32_t linear_call(const TensorCallV1* call, TensorErrorV1* error) {
  ok(error);
  CHECK(check_call(call, 5, error));
  const int ordinal = call->stream.device_ordinal;
  const TensorArgumentV1* a = call->arguments;
  int64_t x[2] = {-1, -1};
  CHECK(check_buffer(a[0], "x", ordinal, TENSOR_UINT8, x, 2, 16, error));
  if (x[1] % 16) return fail(error, TENSOR_ERROR_ARGUMENT, "x: rows of a multiple of 16 values");
  int64_t w[2] = {-1, x[1]};
  CHECK(check_buffer(a[2], "w", ordinal, TENSOR_UINT8, w, 2, 16, error));
  int64_t x_scales[2] = {blocks_of(x[1]), x[0]}, w_scales[2] = {blocks_of(w[0]), blocks_of(x[1])}, out[2] = {x[0], w[0]};
  CHECK(check_buffer(a[1], "x_scales", ordinal, TENSOR_FLOAT32, x_scales, 2, 16, error));
  CHECK(check_buffer(a[3], "w_scales", ordinal, TENSOR_FLOAT32, w_scales, 2, 16, error));
  CHECK(check_values(a[4], "out", ordinal, out, 2, error));
  if (x[0] > 1 << 20 || w[0] > 1 << 22 || x[1] > 1 << 20)
    return fail(error, TENSOR_ERROR_ARGUMENT, "x, w: at most 2^20 rows of x, 2^22 of w, and 2^20 columns");
  if (x[0] * w[0] > (int64_t)1 << 35) return fail(error, TENSOR_ERROR_ARGUMENT, "out: at most 2^35 values");
  CHECK(check_apart(call, {{4, "out", -1}}, error));
  CHECK(check_device(call, error));
  tensor_fp8::LinearArgs args{};
  args.x = pointer<const uint8_t>(a[0]);
  args.x_scales = pointer<const float>(a[1]);
  args.w = pointer<const uint8_t>(a[2]);
  args.w_scales = pointer<const float>(a[3]);
  args.out = pointer<void>(a[4]);
  args.m = (int)x[0];
  args.n = (int)w[0];
  args.k = (int)x[1];
  args.out_f32 = a[4].dtype == TENSOR_FLOAT32;
  const hipError_t status = tensor_fp8::launch_linear(args, stream_of(call));
  return status == hipSuccess ? TENSOR_OK : hip_fail(error, status, "8-bit linear launch");
}

}  // namespace

extern "C" {

int32_t tensor_rms_norm_v1(const TensorCallV1* call, TensorErrorV1* error) { return norm_call(call, error, false); }

int32_t tensor_rms_norm_fp8_v1(const TensorCallV1* call, TensorErrorV1* error) { return norm_call(call, error, true); }

int32_t tensor_quantize_fp8_v1(const TensorCallV1* call, TensorErrorV1* error) { return quantize_call(call, error); }

int32_t tensor_fp8_linear_v1(const TensorCallV1* call, TensorErrorV1* error) { return linear_call(call, error); }

}  // extern "C"
