// Newton-Schulz orthogonalisation of matrix updates.
//
// X0 = U / (|U|_F + eps), then each step X <- a X + (b A + c A A) X with
// A = X X^T, which maps X's singular values by a s + b s^3 + c s^5 and leaves
// its singular vectors.  Matrices with more rows than columns are turned, so
// that A is the smaller of the two Gram matrices.
#include <climits>
#include <cmath>
#include <type_traits>

#include "fma_tile.h"

namespace spmm {
namespace {

constexpr int kNormParts = 64;  // work-groups that add up one matrix's squares

// Partial sums of squares in fp64: no overflow, and no loss against the total.
template <typename T>
__global__ __launch_bounds__(kThreads) void square_sums(const T* __restrict__ u, int64_t elements,
                                                        double* __restrict__ parts) {
  const T* m = u + blockIdx.y * elements;
  double s = 0.0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < elements;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const double v = static_cast<double>(static_cast<float>(m[i]));
    s += v * v;
  }
  __shared__ double lds[kThreads];
  lds[threadIdx.x] = s;
  __syncthreads();
  for (int d = kThreads / 2; d > 0; d >>= 1) {
    if (static_cast<int>(threadIdx.x) < d) lds[threadIdx.x] += lds[threadIdx.x + d];
    __syncthreads();
  }
  if (threadIdx.x == 0) parts[blockIdx.y * kNormParts + blockIdx.x] = lds[0];
}

// X0 in fp32, turned where `tall`.
template <typename T>
__global__ __launch_bounds__(kThreads) void scale_update(const T* __restrict__ u, int64_t rows, int64_t cols, bool tall,
                                                         double eps, const double* __restrict__ parts,
                                                         float* __restrict__ x) {
  double s = 0.0;
  for (int i = 0; i < kNormParts; ++i) s += parts[blockIdx.y * kNormParts + i];
  const double norm = sqrt(s) + eps;
  const int64_t elements = rows * cols;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < elements;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t to = tall ? i % cols * rows + i / cols : i;
    x[blockIdx.y * elements + to] =
        static_cast<float>(static_cast<double>(static_cast<float>(u[blockIdx.y * elements + i])) / norm);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void store_result(const float* __restrict__ x, int64_t rows, int64_t cols,
                                                         bool tall, T* __restrict__ out) {
  const int64_t elements = rows * cols;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < elements;
       i += static_cast<int64_t>(gridDim.x) * kThreads)
    out[blockIdx.y * elements + i] = static_cast<T>(x[blockIdx.y * elements + (tall ? i % cols * rows + i / cols : i)]);
}

// out = alpha * left right + beta * add, [m, n] each of a batch; `turned`:
// right is stored [n, depth].
__global__ __launch_bounds__(kThreads) void product(const float* __restrict__ left, const float* __restrict__ right,
                                                    bool turned, const float* add, int64_t m, int64_t n, int64_t depth,
                                                    float alpha, float beta, float* out) {
  const int64_t across = (n + kTile - 1) / kTile, down = (m + kTile - 1) / kTile;
  const int64_t batch = blockIdx.x / (across * down);
  const int64_t r0 = blockIdx.x / across % down * kTile, c0 = blockIdx.x % across * kTile;
  const int64_t rows = m - r0 < kTile ? m - r0 : kTile, cols = n - c0 < kTile ? n - c0 : kTile;
  float acc[4][4] = {};
  const float* r = right + batch * n * depth;
  multiply_tile<float>({left + (batch * m + r0) * depth, depth, 1},
                       turned ? Operand<float>{r + c0 * depth, depth, 1} : Operand<float>{r + c0, 1, n}, rows, cols,
                       depth, acc);
  const int64_t at = (batch * m + r0) * n + c0;
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t e = at + (4 * ti + i) * n + 4 * tj + j;
      if (4 * ti + i < rows && 4 * tj + j < cols)
        out[e] = alpha * acc[i][j] + (add != nullptr ? beta * add[e] : 0.0f);
    }
}

spmm_status check_desc(const spmm_orthogonalize_desc* d) {
  if (d == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null descriptor");
  if (!dense_type(d->value_type))
    return fail(SPMM_ERR_CONTRACT, "orthogonalize supports only FP16, BF16 and FP32 tensors");
  if (d->batch < 0 || d->rows < 0 || d->width < 0) return fail(SPMM_ERR_CONTRACT, "orthogonalize: negative extent");
  if (d->batch > 65535 || d->rows > INT32_MAX || d->width > INT32_MAX)
    return fail(SPMM_ERR_CONTRACT, "orthogonalize takes at most 65535 matrices with extents below 2^31");
  if (d->steps < 0) return fail(SPMM_ERR_INVALID_ARGUMENT, "orthogonalize: steps must not be negative");
  if (d->steps > 0 && d->coefficients == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "orthogonalize: null coefficients");
  for (int64_t i = 0; i < 3 * d->steps; ++i)
    if (!std::isfinite(d->coefficients[i]))
      return fail(SPMM_ERR_INVALID_ARGUMENT, "orthogonalize: coefficients must be finite");
  if (!(d->eps >= 0.0) || std::isinf(d->eps))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "orthogonalize: eps must be finite and not negative");
  return SPMM_OK;
}

// X twice (a step reads one and writes the other), A, its polynomial, and the
// sums of squares; m <= n the matrix's extents.
struct Layout {
  int64_t m, n;
  size_t x, gram, parts;
  explicit Layout(const spmm_orthogonalize_desc* d) {
    m = d->rows < d->width ? d->rows : d->width;
    n = d->rows < d->width ? d->width : d->rows;
    x = align_up(static_cast<size_t>(d->batch * m * n) * sizeof(float), 256);
    gram = align_up(static_cast<size_t>(d->batch * m * m) * sizeof(float), 256);
    parts = align_up(static_cast<size_t>(d->batch * kNormParts) * sizeof(double), 256);
  }
  size_t total() const { return 2 * x + 2 * gram + parts; }
};

template <typename T>
spmm_status run(const spmm_orthogonalize_desc* d, const Layout& l, const void* update, void* out, char* ws,
                hipStream_t s) {
  const bool tall = d->rows > d->width;
  float* x = reinterpret_cast<float*>(ws);
  float* y = reinterpret_cast<float*>(ws + l.x);
  float* gram = reinterpret_cast<float*>(ws + 2 * l.x);
  float* poly = reinterpret_cast<float*>(ws + 2 * l.x + l.gram);
  double* parts = reinterpret_cast<double*>(ws + 2 * l.x + 2 * l.gram);
  const T* u = static_cast<const T*>(update);
  const int64_t elements = l.m * l.n;
  const unsigned blocks = static_cast<unsigned>(ceil_div(elements, kThreads) < 1024 ? ceil_div(elements, kThreads) : 1024);
  const unsigned batch = static_cast<unsigned>(d->batch);
  hipLaunchKernelGGL(square_sums<T>, dim3(kNormParts, batch), dim3(kThreads), 0, s, u, elements, parts);
  hipLaunchKernelGGL(scale_update<T>, dim3(blocks, batch), dim3(kThreads), 0, s, u, d->rows, d->width, tall, d->eps,
                     parts, x);
  auto multiply = [&](const float* a, const float* b, bool turned, const float* add, int64_t n, int64_t depth,
                      double alpha, double beta, float* to) {
    const int64_t tiles = ceil_div(l.m, kTile) * ceil_div(n, kTile) * d->batch;
    hipLaunchKernelGGL(product, dim3(static_cast<unsigned>(tiles)), dim3(kThreads), 0, s, a, b, turned, add, l.m, n,
                       depth, static_cast<float>(alpha), static_cast<float>(beta), to);
  };
  for (int64_t i = 0; i < d->steps; ++i) {
    const double* c = d->coefficients + 3 * i;
    multiply(x, x, true, nullptr, l.m, l.n, 1.0, 0.0, gram);
    multiply(gram, gram, true, gram, l.m, l.m, c[2], c[1], poly);
    multiply(poly, x, false, x, l.n, l.m, 1.0, c[0], y);
    std::swap(x, y);
  }
  hipLaunchKernelGGL(store_result<T>, dim3(blocks, batch), dim3(kThreads), 0, s, x, d->rows, d->width, tall,
                     static_cast<T*>(out));
  return check_launch("orthogonalize");
}

}  // namespace
}  // namespace spmm

using namespace spmm;

extern "C" {

spmm_status spmm_orthogonalize_workspace(const spmm_orthogonalize_desc* d, size_t* bytes) {
  clear_error();
  if (bytes == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null argument");
  if (spmm_status st = check_desc(d)) return st;
  *bytes = Layout(d).total();
  return SPMM_OK;
}

spmm_status spmm_orthogonalize_run(const spmm_orthogonalize_desc* d, const void* update, void* out, void* workspace,
                                   size_t workspace_bytes, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_desc(d)) return st;
  if (d->batch == 0 || d->rows == 0 || d->width == 0) return SPMM_OK;
  if (update == nullptr || out == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "orthogonalize: null device pointer");
  const Layout l(d);
  if (workspace == nullptr || workspace_bytes < l.total())
    return fail(SPMM_ERR_CONTRACT, "orthogonalize: workspace too small: need " + std::to_string(l.total()) + " bytes");
  if (ceil_div(l.m, kTile) * ceil_div(l.n, kTile) * d->batch > INT32_MAX)
    return fail(SPMM_ERR_OVERFLOW, "orthogonalize: too many tiles for one launch");
  char* ws = static_cast<char*>(workspace);
  hipStream_t s = as_stream(stream);
  switch (d->value_type) {
    case SPMM_VALUE_F16: return run<_Float16>(d, l, update, out, ws, s);
    case SPMM_VALUE_BF16: return run<__bf16>(d, l, update, out, ws, s);
    default: return run<float>(d, l, update, out, ws, s);
  }
}

}  // extern "C"
