// A 64 x 64 tile of a matrix product in fp32, for operands of any stride.
#pragma once

#include "numeric.h"

namespace spmm {

constexpr int kThreads = 256;
constexpr int kTile = 64;   // output tile of a work-group, both ways
constexpr int kDepth = 16;  // of the sum, per step through LDS

// An operand of a product: element (i, k) at p[i * step + k * depth_step].
template <typename T>
struct Operand {
  const T* p;
  int64_t step, depth_step;
};

// acc += A B over `depth`, for a 64 x 64 tile with `rows` x `cols` of it
// inside the matrix: a thread holds rows 4 (t / 16) + i and columns 4 (t % 16) + j.
template <typename T>
__device__ inline void multiply_tile(Operand<T> a, Operand<T> b, int64_t rows, int64_t cols, int64_t depth,
                                     float (&acc)[4][4]) {
  __shared__ float as[kDepth][kTile + 1], bs[kDepth][kTile + 1];
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
  for (int64_t k0 = 0; k0 < depth; k0 += kDepth) {
    __syncthreads();
    for (int e = threadIdx.x; e < kTile * kDepth; e += kThreads) {
      // neighbouring threads along whichever way is contiguous
      const int ai = a.step == 1 ? e % kTile : e / kDepth, ak = a.step == 1 ? e / kTile : e % kDepth;
      const int bi = b.step == 1 ? e % kTile : e / kDepth, bk = b.step == 1 ? e / kTile : e % kDepth;
      as[ak][ai] = ai < rows && k0 + ak < depth ? static_cast<float>(a.p[ai * a.step + (k0 + ak) * a.depth_step]) : 0.0f;
      bs[bk][bi] = bi < cols && k0 + bk < depth ? static_cast<float>(b.p[bi * b.step + (k0 + bk) * b.depth_step]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += as[k][4 * ti + i] * bs[k][4 * tj + j];
  }
}

template <typename T>
__device__ inline void store_tile(T* out, int64_t stride, int64_t rows, int64_t cols, const float (&acc)[4][4]) {
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * ti + i < rows && 4 * tj + j < cols) out[(4 * ti + i) * stride + 4 * tj + j] = static_cast<T>(acc[i][j]);
}

}  // namespace spmm
