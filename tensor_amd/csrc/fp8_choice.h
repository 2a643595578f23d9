// Which kernel an 8-bit linear takes (fp8_linear.hip): plain host code without HIP, so that a CPU test can compile it by
// itself.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace tensor_fp8 {

// What a call would take in one of the kernels, in microseconds: workgroups go round the CUs, `beside` at a time on one of
// them; a round costs `start`, and a step of K `alone` with one workgroup on a CU, `full` with `beside`.  Fitted to calls
// of 20 to 96 steps and 1 to 4096 rows with weights out of the caches.  There the kernel chosen takes longer than the fastest of
// them by 0.1% in the mean of 85 calls with fp16 results (3% at the worst) and 0.4% in that of 48 with fp32 ones (20%: 512 x 2500 x
// 2544 in 21.1 us, 17.6 by 128 x 64 tiles with loaders).  Beyond it, with 4 to 20 steps or weights of 470 MB, it is 2.0% of 40 and
// 1.4% of 20 calls, 20% at the worst (32 x 57344 x 8192 in 108 us, 90 by 128 x 64 tiles: where the weights' bytes outweigh the
// estimates, the first of the equal ones is taken).
struct LinearCost {
  int bn, bm, beside;
  float start, alone, full;
  float of(int m, int n, int k) const {
    const int64_t groups = (int64_t)((n + bn - 1) / bn) * ((m + bm - 1) / bm), most = (groups + 255) / 256;  // most on a CU
    if (groups > (int64_t)1 << 22) return 1e30f;  // (launches of up to 2^32 - 1 threads)
    const int64_t rounds = most / beside, rest = most % beside;
    const float steps = (float)((k + 127) / 128), more = beside > 1 ? (full - alone) / (beside - 1) : 0.0f;
    const float weights = (float)n * (float)k / 4.7e6f;  // what their bytes take, whichever kernel it is
    const float time = most == 1 ? start + steps * alone
                                 : rounds * (start + steps * full) + (rest ? start + steps * (alone + more * (rest - 1)) : 0.0f);
    return time > weights ? time : weights;
  }
};

// linear_rows, then linear_tiles
constexpr LinearCost kLinearFp16[] = {
    {16, 8, 2, 1.0f, 0.124f, 0.175f}, {32, 16, 1, 1.8f, 0.142f, 0.117f}, {16, 32, 1, 1.8f, 0.131f, 0.101f},
    {32, 32, 1, 2.4f, 0.163f, 0.155f}, {32, 64, 1, 4.5f, 0.20f, 0.173f},
    {64, 64, 2, 3.6f, 0.27f, 0.53f}, {128, 64, 2, 4.1f, 0.49f, 0.74f}, {128, 128, 1, 7.1f, 0.53f, 0.47f},
    {256, 128, 1, 11.1f, 0.76f, 0.72f}, {256, 256, 1, 12.0f, 1.44f, 1.38f}};
constexpr LinearCost kLinearFp32[] = {
    {16, 8, 2, 1.5f, 0.12f, 0.165f}, {32, 16, 1, 1.9f, 0.14f, 0.13f}, {16, 32, 1, 1.9f, 0.13f, 0.10f},
    {32, 32, 1, 2.7f, 0.17f, 0.15f}, {32, 64, 1, 4.9f, 0.22f, 0.20f},
    {64, 64, 2, 4.8f, 0.34f, 0.80f}, {64, 64, 2, 5.2f, 0.35f, 0.67f}, {128, 64, 2, 6.6f, 0.62f, 1.28f},
    {128, 64, 2, 5.7f, 0.69f, 1.09f}, {128, 128, 1, 5.5f, 1.04f, 1.03f}, {128, 128, 2, 10.0f, 1.02f, 1.71f}};

template <size_t N>
int cheapest(const LinearCost (&costs)[N], int m, int n, int k) {
  int best = 0;
  for (int i = 1; i < (int)N; ++i)
    if (costs[i].of(m, n, k) < costs[best].of(m, n, k)) best = i;
  return best;
}

inline int linear_kernel(int m, int n, int k, bool out_f32) {
  return out_f32 ? cheapest(kLinearFp32, m, n, k) : cheapest(kLinearFp16, m, n, k);
}

}  // namespace tensor_fp8
