// Root-mean-square norm of rows, with the residual's addition or without, its result as values or in 8 bits:
//   h = x + r, r' = h, y = h / sqrt(mean(h^2) + eps) * weight; codes and scales of y (fp8_common.h)
// in fp32: h enters the norm as it is summed, not as r' rounds it; one rounding of y and of r'.
//
// Bound by the bytes: one pass, the row in registers between its sum and its results.  A row is the work of 16 threads up to 128
// columns (four rows a wave: heads of 128, 81880 rows in 8.4 us, 5.0 TB/s), of a wave up to 512, of 256 threads up to 8192
// (8192 x 4096 with fp16 residual to 8 bits: 47.3 us, 5.0 TB/s; 512 or 1024 threads where there are few rows), of 1024 beyond; 8
// columns a thread and load.
// One row (4096 columns) takes 2.3 us on the GPU, and 3.7 of the host to submit.
#include "fp8_common.h"

namespace tensor_fp8 {
namespace {

constexpr int kFewRows = 512;  // two a CU

struct None {};
struct Codes {};

template <typename T>
struct IsNone { static constexpr bool value = false; };
template <>
struct IsNone<None> { static constexpr bool value = true; };
template <typename T>
struct IsCodes { static constexpr bool value = false; };
template <>
struct IsCodes<Codes> { static constexpr bool value = true; };

// sum over the T threads of a row
template <int T>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
  for (int step = (T < 64 ? T : 64) / 2; step > 0; step >>= 1) v += __shfl_xor(v, step);
  if constexpr (T > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[wave] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) v += part[w];
  }
  return v;
}

// T threads of a row, C chunks of 8 columns each
template <typename X, typename R, typename Out, int T, int C>
__global__ __launch_bounds__(T < 256 ? 256 : T) void norm_kernel(const NormArgs a) {
  constexpr int ROWS = T < 256 ? 256 / T : 1;
  __shared__ float part[T > 64 ? T / 64 : 1];
  const int t = threadIdx.x % T;
  const int64_t at_row = (int64_t)blockIdx.x * ROWS + threadIdx.x / T;
  const bool live = at_row < a.rows;
  const size_t row = (size_t)(live ? at_row : a.rows - 1), begin = row * a.width;

  float8_t h[C], weight[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const Chunk chunk(8 * (t + T * c), a.width);
    h[c] = load8(static_cast<const X*>(a.x) + begin + chunk.at, chunk.count);
    if constexpr (!IsNone<R>::value) h[c] += load8(static_cast<const R*>(a.residual) + begin + chunk.at, chunk.count);
    weight[c] = load8(a.weight + chunk.at, chunk.count);
  }
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const Chunk chunk(8 * (t + T * c), a.width);
    if constexpr (!IsNone<R>::value)
      if (live) store8(static_cast<R*>(a.residual_out) + begin + chunk.at, h[c], chunk);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (chunk.has(e)) sum += h[c][e] * h[c][e];
  }
  sum = row_sum<T>(sum, part);
  float mean = sum / (float)a.width + a.eps;
  if (!(mean < kInfinity)) {  // squares past fp32: the same of h 2^-80
    sum = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const Chunk chunk(8 * (t + T * c), a.width);
      h[c] *= 0x1p-80f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (chunk.has(e)) sum += h[c][e] * h[c][e];
    }
    sum = row_sum<T>(sum, part);
    mean = sum / (float)a.width + a.eps * 0x1p-80f * 0x1p-80f;
  }
  const float inverse = rsqrtf(mean);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int column = 8 * (t + T * c);
    const Chunk chunk(column, a.width);
    const float8_t y = h[c] * inverse * weight[c];
    if constexpr (IsCodes<Out>::value) {
      const float scale = block_scale(y, chunk);
      if (live) {
        store_codes(static_cast<uint8_t*>(a.out) + begin + chunk.at, y, scale, chunk);
        if (t % 16 == 0 && column < a.width) a.scales[(size_t)(column / kBlock) * a.rows + row] = scale;
      }
    } else if (live) {
      store8(static_cast<Out*>(a.out) + begin + chunk.at, y, chunk);
    }
  }
}

// Few rows leave CUs idle, so a row is the work of twice the threads or four times, 8 columns each.  By 256 threads and by more, in
// us: to 8 bits with an fp32 residual 1 x 5120 4.8 and 4.3, 64 x 8192 6.0 and 4.9, 512 x 6144 10.1 and 9.2; to fp16 with an fp16
// one 1 x 4096 3.1 and 2.9, 512 x 8192 8.4 and 7.8, 512 x 6144 6.9 and 7.1.  The line is where fp16 results lose: 1024 x 6144
// 9.7 and 11.0.  Results in 8 bits gain past it as well, which it leaves: 600 x 8192 13.7 and 11.8, 8192 x 6144 107.5 and 99.7.
int threads_of(const NormArgs& a) {
  const int width = a.width;
  if (a.rows <= kFewRows && width > 2048 && width <= 8192) return width <= 4096 ? 512 : 1024;
  return width <= 128 ? 16 : width <= 512 ? 64 : width <= 8192 ? 256 : 1024;
}

template <typename X, typename R, typename Out>
hipError_t launch_typed(const NormArgs& a, hipStream_t stream) {
  const int threads = threads_of(a), rows = threads < 256 ? 256 / threads : 1;
  const dim3 grid((unsigned)(((int64_t)a.rows + rows - 1) / rows)), block(threads < 256 ? 256 : threads);
#define LAUNCH(T, C) hipLaunchKernelGGL((norm_kernel<X, R, Out, T, C>), grid, block, 0, stream, a)
  if (a.width <= 128) LAUNCH(16, 1);
  else if (a.width <= 512) LAUNCH(64, 1);
  else if (a.width <= 2048) LAUNCH(256, 1);
  else if (threads == 512) LAUNCH(512, 1);
  else if (threads == 1024 && a.width <= 8192) LAUNCH(1024, 1);
  else if (a.width <= 4096) LAUNCH(256, 2);
  else if (a.width <= 6144) LAUNCH(256, 3);
  else if (a.width <= 8192) LAUNCH(256, 4);
  else if (a.width <= 16384) LAUNCH(1024, 2);
  else LAUNCH(1024, 4);
#undef LAUNCH
  return hipGetLastError();
}

template <typename X, typename R>
hipError_t launch_out(const NormArgs& a, hipStream_t stream) {
  if (a.scales) return launch_typed<X, R, Codes>(a, stream);
  return a.out_f32 ? launch_typed<X, R, float>(a, stream) : launch_typed<X, R, _Float16>(a, stream);
}

template <typename X>
hipError_t launch_residual(const NormArgs& a, hipStream_t stream) {
  if (!a.residual) return launch_out<X, None>(a, stream);
  return a.residual_f32 ? launch_out<X, float>(a, stream) : launch_out<X, _Float16>(a, stream);
}

}  // namespace

int64_t norm_threads(const NormArgs& a) {
  const int threads = threads_of(a), rows = threads < 256 ? 256 / threads : 1;
  return ((int64_t)a.rows + rows - 1) / rows * (threads < 256 ? 256 : threads);
}

hipError_t launch_norm(const NormArgs& a, hipStream_t stream) {
  return a.x_f32 ? launch_residual<float>(a, stream) : launch_residual<_Float16>(a, stream);
}

}  // namespace tensor_fp8
