// Rows as 8-bit codes with a scale for each 128 columns (fp8_common.h): of x, or of silu(g) u for rows [g | u],
// silu(g) = g / (1 + exp(-g)), in fp32.
//
// Bound by the bytes: 16 lanes of 8 columns are a block, which meet in its largest magnitude.  4093 x 12288 gated in 47 us
// (5.4 TB/s; 61 with rows of blocks one at a time, whose scales lay a row of the scales apart), 8 x 4096 in 2.6 us on the GPU.
#include "fp8_common.h"

namespace tensor_fp8 {
namespace {

constexpr int kThreads = 256, kLanes = kBlock / 8;  // lanes of a block

// silu(g) v.  The product that exp takes is rounded once, so a result is off by up to |g| 2^-24 of it where the gate is closed:
// fp32 inputs by 1 unit of 2^-24 rms from -2 on, by 7 from -20 to -8, by 14 (33 at the most) from -40 to -20, where the gate lets
// 2^-24 of a value through and less.  A product in two parts would be three instructions a value more.  Of 402 million codes of
// gated rows 349 differ from those of 64 bits, 371 by a library's exp and quotient in fp32.
// Below -80 exp(-g) passes fp32, or what it leaves of the quotient does, while g exp(g) v may not: there exp(g) = m 2^n enters by
// its exponent, half before and half after v.
__device__ __forceinline__ float8_t gated(float8_t g, float8_t v) {
  constexpr float kLog2 = 1.44269504088896340736f;
  float8_t y;
  float least = g[0];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y[e] = g[e] * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2 * g[e])) * v[e];
    least = fminf(least, g[e]);
  }
  if (least < -80.0f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (!(g[e] < -80.0f)) continue;
      const float power = fmaxf(kLog2 * g[e], -1024.0f), whole = floorf(power);  // (g exp(g) v is 0 from -1024 on)
      const int n = (int)whole, half = n / 2;
      y[e] = ldexpf(ldexpf(g[e] * exp2f(power - whole), half) * v[e], n - half);
    }
  }
  return y;
}

// A workgroup has 16 / ROWS blocks of ROWS rows at a time, UNITS times: of eight rows, so that the scales of a block lie next
// to each other, twice, with the loads of both in flight.
template <typename X, bool GATED, int ROWS, int UNITS>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const QuantizeArgs a, int groups) {
  const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int rows_at = blockIdx.x / groups;
  const int row0 = rows_at * ROWS * UNITS + group % ROWS;
  const int block = (blockIdx.x - rows_at * groups) * (16 / ROWS) + group / ROWS;
  const Chunk chunk(block * kBlock + 8 * lane, a.width);
  float8_t y[UNITS], up[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const X* x = static_cast<const X*>(a.x) + (size_t)min(row0 + u * ROWS, a.rows - 1) * a.width * (GATED ? 2 : 1) + chunk.at;
    y[u] = load8(x, chunk.count);
    if constexpr (GATED) up[u] = load8(x + a.width, chunk.count);
  }
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int row = row0 + u * ROWS;
    if constexpr (GATED) y[u] = gated(y[u], up[u]);
    const float scale = block_scale(y[u], chunk);
    if (row >= a.rows || block * kBlock >= a.width) continue;
    store_codes(a.codes + (size_t)row * a.width + chunk.at, y[u], scale, chunk);
    if (lane == 0) a.scales[(size_t)block * a.rows + row] = scale;
  }
}

constexpr int kRows = 8, kUnits = 2;
// Few rows take a row of 16 blocks, so that no lane is without one (8 rows of 4096: 3.8 us either way).
bool few(const QuantizeArgs& a) { return a.rows < 4 * kRows * kUnits; }

// workgroups along the columns, and of all
int groups_of(const QuantizeArgs& a) { return (int)((blocks_of(a.width) + (few(a) ? 15 : 16 / kRows - 1)) / (few(a) ? 16 : 16 / kRows)); }
int64_t workgroups_of(const QuantizeArgs& a) {
  const int rows = few(a) ? 1 : kRows * kUnits;
  return (int64_t)groups_of(a) * (((int64_t)a.rows + rows - 1) / rows);
}

}  // namespace

int64_t quantize_threads(const QuantizeArgs& a) { return workgroups_of(a) * kThreads; }

hipError_t launch_quantize(const QuantizeArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)workgroups_of(a)), block(kThreads);
  const int groups = groups_of(a);
#define LAUNCH(X, G) \
  if (few(a)) hipLaunchKernelGGL((quantize_kernel<X, G, 1, 1>), grid, block, 0, stream, a, groups); \
  else hipLaunchKernelGGL((quantize_kernel<X, G, kRows, kUnits>), grid, block, 0, stream, a, groups)
  if (a.x_f32) {
    if (a.gated) { LAUNCH(float, true); } else { LAUNCH(float, false); }
  } else {
    if (a.gated) { LAUNCH(_Float16, true); } else { LAUNCH(_Float16, false); }
  }
#undef LAUNCH
  return hipGetLastError();
}

}  // namespace tensor_fp8
