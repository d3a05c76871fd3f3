// The part of the counting sort that does not depend on what is sorted.
#include "sort_ids.h"

namespace spmm {
namespace {

// One thread a digit: counts of the tiles before, and the sum of all.
__global__ __launch_bounds__(64) void add_digits(int bins, int64_t tiles, uint32_t* counts, uint32_t* totals) {
  const int b = blockIdx.x * 64 + threadIdx.x;
  if (b >= bins) return;
  uint32_t sum = 0;
  for (int64_t t = 0; t < tiles; t += 8) {
    uint32_t c[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) c[u] = t + u < tiles ? counts[(t + u) * bins + b] : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (t + u < tiles) {
        counts[(t + u) * bins + b] = sum;
        sum += c[u];
      }
  }
  totals[b] = sum;
}

}  // namespace

spmm_status launch_add_digits(int bins, int64_t tiles, uint32_t* counts, uint32_t* totals, hipStream_t s) {
  hipLaunchKernelGGL(add_digits, dim3(static_cast<unsigned>(ceil_div(bins, 64))), dim3(64), 0, s, bins, tiles, counts,
                     totals);
  return check_launch("add_digits");
}

}  // namespace spmm
