// The part of the sort that does not depend on what is sorted.
#include "sort_ids.h"

namespace spmm {
namespace {

// Counts of the tiles before, and the sum of all, for kBins digits (a cache line)
// a work-group: kShares threads a digit take kTiles tiles each at a time.
constexpr int kBins = 32, kShares = 32, kTiles = 8;
__global__ __launch_bounds__(kBins * kShares) void add_digits(int bins, int64_t tiles, uint32_t* counts,
                                                              uint32_t* totals) {
  __shared__ uint32_t sums[kShares][kBins];
  const int bin = threadIdx.x % kBins, share = threadIdx.x / kBins, b = blockIdx.x * kBins + bin;
  uint32_t carry = 0;
  for (int64_t t0 = 0; t0 < tiles; t0 += kShares * kTiles) {
    const int64_t t = t0 + share * kTiles;
    uint32_t c[kTiles], own = 0;
#pragma unroll
    for (int u = 0; u < kTiles; ++u) c[u] = b < bins && t + u < tiles ? counts[(t + u) * bins + b] : 0;
#pragma unroll
    for (int u = 0; u < kTiles; ++u) own += c[u];
    __syncthreads();  // readers of the last sums are done
    sums[share][bin] = own;
    __syncthreads();
    uint32_t at = carry;
#pragma unroll
    for (int s = 0; s < kShares; ++s) {
      const uint32_t v = sums[s][bin];
      at += s < share ? v : 0;
      carry += v;
    }
#pragma unroll
    for (int u = 0; u < kTiles; ++u)
      if (b < bins && t + u < tiles) {
        counts[(t + u) * bins + b] = at;
        at += c[u];
      }
  }
  if (share == 0 && b < bins) totals[b] = carry;
}

}  // namespace

spmm_status launch_add_digits(int bins, int64_t tiles, uint32_t* counts, uint32_t* totals, hipStream_t s) {
  hipLaunchKernelGGL(add_digits, dim3(static_cast<unsigned>(ceil_div(bins, kBins))), dim3(kBins * kShares), 0, s, bins,
                     tiles, counts, totals);
  return check_launch("add_digits");
}

}  // namespace spmm
