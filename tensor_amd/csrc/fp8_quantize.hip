// Rows as 8-bit codes with a scale for each 128 columns (fp8_common.h): of x, or of silu(g) u for rows [g | u],
// silu(g) = g / (1 + exp(-g)), in fp32.
#include "fp8_common.h"

namespace tensor_fp8 {
namespace {

constexpr int kThreads = 256, kLanes = kBlock / 8;  // lanes of a block

template <typename X, bool GATED>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const QuantizeArgs a, int blocks) {
  const int64_t index = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  const bool live = index < (int64_t)a.rows * blocks;
  const int64_t here = live ? index : 0;
  const int row = (int)(here / blocks), block = (int)(here - (int64_t)row * blocks);
  const Chunk chunk(block * kBlock + 8 * (threadIdx.x % kLanes), a.width);
  const X* x = static_cast<const X*>(a.x) + (size_t)row * a.width * (GATED ? 2 : 1) + chunk.at;
  float8_t y = load8(x, chunk.count);
  if constexpr (GATED) {
    const float8_t up = load8(x + a.width, chunk.count);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = y[e] / (1.0f + exp2f(-1.44269504088896340736f * y[e])) * up[e];
  }
  const float scale = block_scale(y, chunk);
  if (!live) return;
  store_codes(a.codes + (size_t)row * a.width + chunk.at, y, scale, chunk);
  if (threadIdx.x % kLanes == 0) a.scales[(size_t)block * a.rows + row] = scale;
}

}  // namespace

int64_t quantize_threads(const QuantizeArgs& a) {
  const int64_t blocks = (int64_t)a.rows * blocks_of(a.width), per = kThreads / kLanes;
  return (blocks + per - 1) / per * kThreads;
}

hipError_t launch_quantize(const QuantizeArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)(quantize_threads(a) / kThreads)), block(kThreads);
  const int blocks = (int)blocks_of(a.width);
#define LAUNCH(X, G) hipLaunchKernelGGL((quantize_kernel<X, G>), grid, block, 0, stream, a, blocks)
  if (a.x_f32) {
    if (a.gated) LAUNCH(float, true); else LAUNCH(float, false);
  } else {
    if (a.gated) LAUNCH(_Float16, true); else LAUNCH(_Float16, false);
  }
#undef LAUNCH
  return hipGetLastError();
}

}  // namespace tensor_fp8
