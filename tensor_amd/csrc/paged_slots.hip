// One step's bookkeeping of a paged key/value cache from the requests' lengths: for request b with
// l_b tokens held and n_b new ones, pages of S tokens,
//   held_b = ceil(l_b / S), wanted_b = ceil((l_b + n_b) / S), both at most the table's columns;
//   its new pages are numbers base_b .. of the step, base_b the sum of wanted - held over earlier
//   requests, and page number r is free[free_count - 1 - r] (the list is a stack), -1 past its end;
//   token i of it has place l_b + i, position start + place and slot table[b][place / S] * S + place % S
//   (-1 without a page), and stands at row offset_b + i, offset_b the sum of earlier n.
//
// Integers only: bound by the launch and by the table, read and written once.  A workgroup per
// request sums the earlier requests' counts and pages itself (the lengths stay in L2: 256 requests
// are 2 KB), so that one launch does without a scan, a flag or a wait between workgroups; grid.y
// shares the tokens of long prompts and the columns of wide tables.  4.5 us for 8 requests and for 256 with tables of
// 2048 columns (4.2 MB): the launch.
#include "paged_launch.h"

namespace tensor_paged {
namespace {

constexpr int kThreads = kSlotsThreads;

// Sums past int32 stop at its ends: a wrapped length would be none, a wrapped position padding.
__device__ __forceinline__ int saturated(int64_t v) { return (int)max(min(v, (int64_t)INT32_MAX), (int64_t)INT32_MIN); }

__global__ __launch_bounds__(kThreads) void paged_slots(const SlotsArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int S = 1 << a.page_shift;
  auto columns = [&](int64_t tokens) {
    const int64_t pages = (tokens + S - 1) >> a.page_shift;
    return (int)(pages < a.columns ? pages : a.columns);
  };
  // sums over the earlier requests: tokens and pages (64 bits: lengths are the caller's)
  int64_t tokens = 0, pages = 0;
  for (int i = tid; i < b; i += kThreads) {
    const int64_t l = max(a.lengths[i], 0), n = max(a.counts[i], 0);
    tokens += n;
    pages += columns(l + n) - columns(l);
  }
#pragma unroll
  for (int step = 32; step > 0; step >>= 1) {
    tokens += __shfl_xor(tokens, step);
    pages += __shfl_xor(pages, step);
  }
  __shared__ int64_t part[2][kThreads / 64];
  if (lane == 0) {
    part[0][wave] = tokens;
    part[1][wave] = pages;
  }
  __syncthreads();
  tokens = part[0][0] + part[0][1] + part[0][2] + part[0][3];
  pages = part[1][0] + part[1][1] + part[1][2] + part[1][3];

  const int64_t l = max(a.lengths[b], 0), n = max(a.counts[b], 0);
  const int held = columns(l), wanted = columns(l + n);
  const int start = *a.start;
  const int available = min(max(*a.free_count, 0), a.free_extent);
  const int32_t* row = a.table + (size_t)b * a.columns;
  int32_t* row_out = a.table_out + (size_t)b * a.columns;
  auto page = [&](int column) {
    if (column < held) return row[column];
    const int64_t rank = pages + column - held;
    return column < wanted && rank < available ? a.free[available - 1 - rank] : -1;
  };
  const int first = blockIdx.y * kThreads + tid, stride = gridDim.y * kThreads;
  for (int column = first; column < a.columns; column += stride) row_out[column] = page(column);
  const int64_t room = min((int64_t)a.tokens - tokens, n);  // rows of this request's tokens in the outputs
  for (int64_t i = first; i < room; i += stride) {
    const int64_t place = l + i, column = place >> a.page_shift;
    const int32_t p = column < a.columns ? page((int)column) : -1;
    // (a page whose slots pass 31 bits has none: a wrapped one would be another page's)
    a.slots[tokens + i] = p < 0 || p >> (31 - a.page_shift) ? -1 : (p << a.page_shift) + (int)(place & (S - 1));
    a.positions[tokens + i] = saturated(start + place);
  }
  if (blockIdx.y == 0 && tid == 0) {
    a.offsets[b] = (int)min(tokens, (int64_t)a.tokens);
    a.lengths_out[b] = saturated(l + n);
  }
  if (b == a.requests - 1) {
    const int64_t all = tokens + n;
    for (int64_t i = all + first; i < a.tokens; i += stride) {
      a.slots[i] = -1;
      a.positions[i] = -1;
    }
    if (blockIdx.y == 0 && tid == 0) {
      a.offsets[a.requests] = (int)min(all, (int64_t)a.tokens);
      *a.free_left = saturated(available - (pages + wanted - held));
    }
  }
}

}  // namespace

hipError_t launch_slots(const SlotsArgs& a, hipStream_t stream) {
  // shares of 4096 table columns, or of 4096 tokens a request on average (a prompt of 120000 tokens among four requests:
  // 17 us, 102 in one share; 256 requests with 2048 columns take one either way)
  const int by_table = (a.columns + 4095) / 4096, by_tokens = a.tokens / a.requests / 4096 + 1;
  const int shares = by_table > by_tokens ? by_table : by_tokens;
  hipLaunchKernelGGL(paged_slots, dim3(a.requests, shares < 64 ? shares : 64), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace tensor_paged
