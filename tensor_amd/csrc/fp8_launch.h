// Host-side launch descriptors of the norm and the 8-bit operators.  Shapes have been validated by the C-ABI entry
// points before these run.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tensor_fp8 {

constexpr int kBlock = 128;           // values of a row that share a scale; rows of weights that do
constexpr int kNormMaxWidth = 32768;  // a row is held in registers
constexpr float kNormLeastEps = 0x1p-100f;  // squares that are lost below fp32 are lost beside it too
// A launch has at most 2^32 - 1 threads along x.
constexpr int64_t kMostThreads = ((int64_t)1 << 32) - 1;
constexpr int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

struct NormArgs {
  const void *x, *residual;  // [rows, width]; residual nullptr: none
  const float* weight;       // [width]
  void *out, *residual_out;  // out: [rows, width], or codes
  float* scales;             // nullptr, or of codes: [blocks, rows]
  int rows, width;
  float eps;
  bool x_f32, residual_f32, out_f32;
};
int64_t norm_threads(const NormArgs& args);
hipError_t launch_norm(const NormArgs& args, hipStream_t stream);

struct QuantizeArgs {
  const void* x;   // [rows, width], or gated [rows, 2 width]
  uint8_t* codes;  // [rows, width]
  float* scales;   // [blocks, rows]
  int rows, width;
  bool gated, x_f32;
};
int64_t quantize_threads(const QuantizeArgs& args);
hipError_t launch_quantize(const QuantizeArgs& args, hipStream_t stream);

struct LinearArgs {
  const uint8_t *x, *w;             // [m, k], [n, k]
  const float *x_scales, *w_scales; // [blocks of k, m], [blocks of n, blocks of k]
  void* out;                        // [m, n]
  int m, n, k;
  bool out_f32;
};
hipError_t launch_linear(const LinearArgs& args, hipStream_t stream);

}  // namespace tensor_fp8
