// Linear layer on 8-bit operands with a scale for each block of 128 (fp8_common.h):
//   out[m, n] = sum_b (sx[b, m] sw[n / 128, b]) sum_{k in block b} x[m, k] w[n, k]
// The inner sum is the matrix cores', on operands widened to fp16, the outer one fp32 vector arithmetic on its results.
#include "fp8_common.h"

namespace tensor_fp8 {
namespace {

typedef int int8v_t __attribute__((ext_vector_type(8)));

// 8 codes as the fp16 values that they stand for (exactly; NaN stays NaN)
__device__ __forceinline__ half8_t widened(int lo, int hi) {
  half8_t v;
  const int words[2] = {lo, hi};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(words[i], 1.0f, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(words[i], 1.0f, true);
    v[4 * i] = a[0]; v[4 * i + 1] = a[1]; v[4 * i + 2] = b[0]; v[4 * i + 3] = b[1];
  }
  return v;
}

// 16 weight rows x 16 activation rows: lane l has column l % 16 and rows 4 (l / 16) ..
__device__ __forceinline__ float4_t products(int8v_t w, int8v_t x) {
  float4_t sum = {};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(widened(w[2 * i], w[2 * i + 1]), widened(x[2 * i], x[2 * i + 1]), sum, 0, 0, 0);
  return sum;
}

// This lane's 32 bytes of a row's 128 columns from k on: chunks of 16 at l / 16 and 4 + l / 16 (any order does that
// both operands share), zeros past the row's end.
__device__ __forceinline__ int8v_t fragment(const uint8_t* row, int k, int columns, int lane) {
  uint4 v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = k + 16 * (4 * i + (lane >> 4));
    v[i] = at < columns ? *reinterpret_cast<const uint4*>(row + at) : uint4{};
  }
  return int8v_t{(int)v[0].x, (int)v[0].y, (int)v[0].z, (int)v[0].w, (int)v[1].x, (int)v[1].y, (int)v[1].z, (int)v[1].w};
}

template <typename Out>
__global__ __launch_bounds__(256) void linear_kernel(const LinearArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = (blockIdx.x * 4 + wave) * 16, m0 = blockIdx.y * 16;
  if (n0 >= a.n) return;
  const int m = min(m0 + (lane & 15), a.m - 1), n = min(n0 + (lane & 15), a.n - 1), blocks = (a.k + kBlock - 1) / kBlock;
  const uint8_t *x = a.x + (size_t)m * a.k, *w = a.w + (size_t)n * a.k;
  float4_t sum = {};
  for (int b = 0; b < blocks; ++b) {
    const float scale = a.x_scales[(size_t)b * a.m + m] * a.w_scales[(size_t)(n0 / kBlock) * blocks + b];
    sum += products(fragment(w, b * kBlock, a.k, lane), fragment(x, b * kBlock, a.k, lane)) * scale;
  }
  if (m0 + (lane & 15) >= a.m) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int at = n0 + 4 * (lane >> 4) + e;
    if (at < a.n) static_cast<Out*>(a.out)[(size_t)m * a.n + at] = (Out)sum[e];
  }
}

}  // namespace

hipError_t launch_linear(const LinearArgs& a, hipStream_t stream) {
  const dim3 grid((a.n + 63) / 64, (a.m + 15) / 16);
  if (a.out_f32) hipLaunchKernelGGL((linear_kernel<float>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((linear_kernel<_Float16>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace tensor_fp8
