// Layer norm over the last dimension, forward and backward.
//
// With z = (x - mean) * rstd, y = z w + b and g = dy w, a row's gradient is
// dx = rstd * (g - mean(g) - z mean(g z)); dw and db are the column sums of
// dy z and dy over all rows.  Statistics and sums are fp32; the variance is
// the mean of squared distances from the mean (a second pass over the row),
// which keeps its digits where the mean is large against the spread.
#include <climits>
#include <cmath>

#include "numeric.h"

namespace spmm {
namespace {

constexpr int kThreads = 256;

struct NormArgs {
  int64_t rows, width, x_stride, grad_stride;
  float eps;
  bool param_f32;
};

// A piece of weight or bias: `param_type` is the value type or fp32; `other`
// where the vector is absent.
template <typename T>
__device__ inline void load_param(const void* p, bool f32, int64_t c, int64_t width, float other,
                                  float (&v)[kPiece<T>]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) v[i] = other;
  } else if (f32) {
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) v[i] = c + i < width ? static_cast<const float*>(p)[c + i] : 0.0f;
  } else {
    load_piece(static_cast<const T*>(p) + c, width - c, v);
  }
}

__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// Sums of K values over the work-group, the same on every thread.
template <int K>
__device__ inline void block_sum(float (&v)[K]) {
  __shared__ float part[K][16];
  const int wave = threadIdx.x >> 6, waves = (blockDim.x + 63) >> 6;
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
  __syncthreads();  // readers of the previous sum are done
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) part[k][wave] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = 0.0f;
    for (int w = 0; w < waves; ++w) v[k] += part[k][w];
  }
}

// One work-group per row, the row read once per statistic.
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_forward_wide(NormArgs a, const T* __restrict__ x,
                                                              const void* __restrict__ w, const void* __restrict__ b,
                                                              T* __restrict__ y, float* mean, float* rstd) {
  constexpr int V = kPiece<T>;
  const float inv = 1.0f / static_cast<float>(a.width);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* xr = x + r * a.x_stride;
    float s[1] = {0.0f};
    for (int64_t c = threadIdx.x * V; c < a.width; c += kThreads * V) {
      float v[V];
      load_piece(xr + c, a.width - c, v);
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += v[i];
    }
    block_sum(s);
    const float m = s[0] * inv;
    s[0] = 0.0f;
    for (int64_t c = threadIdx.x * V; c < a.width; c += kThreads * V) {
      float v[V];
      load_piece(xr + c, a.width - c, v);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i < a.width) s[0] += (v[i] - m) * (v[i] - m);
    }
    block_sum(s);
    const float rs = 1.0f / sqrtf(s[0] * inv + a.eps);
    if (threadIdx.x == 0 && mean != nullptr) mean[r] = m;
    if (threadIdx.x == 0 && rstd != nullptr) rstd[r] = rs;
    for (int64_t c = threadIdx.x * V; c < a.width; c += kThreads * V) {
      float v[V], wv[V], bv[V];
      load_piece(xr + c, a.width - c, v);
      load_param<T>(w, a.param_f32, c, a.width, 1.0f, wv);
      load_param<T>(b, a.param_f32, c, a.width, 0.0f, bv);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (v[i] - m) * rs * wv[i] + bv[i];
      store_piece(y + r * a.width + c, a.width - c, v);
    }
  }
}

// dx of one row per work-group.
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_backward_wide(NormArgs a, const T* __restrict__ x,
                                                               const void* __restrict__ w,
                                                               const float* __restrict__ mean,
                                                               const float* __restrict__ rstd,
                                                               const T* __restrict__ grad, T* __restrict__ dx) {
  constexpr int V = kPiece<T>;
  const float inv = 1.0f / static_cast<float>(a.width);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* xr = x + r * a.x_stride;
    const T* gr = grad + r * a.grad_stride;
    const float m = mean[r], rs = rstd[r];
    float s[2] = {0.0f, 0.0f};
    for (int64_t c = threadIdx.x * V; c < a.width; c += kThreads * V) {
      float v[V], d[V], wv[V];
      load_piece(xr + c, a.width - c, v);
      load_piece(gr + c, a.width - c, d);
      load_param<T>(w, a.param_f32, c, a.width, 1.0f, wv);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i < a.width) {
          s[0] += d[i] * wv[i];
          s[1] += d[i] * wv[i] * ((v[i] - m) * rs);
        }
    }
    block_sum(s);
    const float g0 = s[0] * inv, g1 = s[1] * inv;
    for (int64_t c = threadIdx.x * V; c < a.width; c += kThreads * V) {
      float v[V], d[V], wv[V];
      load_piece(xr + c, a.width - c, v);
      load_piece(gr + c, a.width - c, d);
      load_param<T>(w, a.param_f32, c, a.width, 1.0f, wv);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = rs * (d[i] * wv[i] - g0 - (v[i] - m) * rs * g1);
      store_piece(dx + r * a.width + c, a.width - c, v);
    }
  }
}

// Column sums of dy z and dy over a chunk of rows: work-group (i, p) adds the
// rows of chunk p for kThreads columns.  part: [chunks][2][width].
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_columns_wide(NormArgs a, const T* __restrict__ x,
                                                              const float* __restrict__ mean,
                                                              const float* __restrict__ rstd,
                                                              const T* __restrict__ grad, int64_t chunk,
                                                              float* __restrict__ part) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= a.width) return;
  const int64_t r0 = blockIdx.y * chunk, r1 = r0 + chunk < a.rows ? r0 + chunk : a.rows;
  float dw = 0.0f, db = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float d = static_cast<float>(grad[r * a.grad_stride + c]);
    dw += d * ((static_cast<float>(x[r * a.x_stride + c]) - mean[r]) * rstd[r]);
    db += d;
  }
  float* p = part + static_cast<int64_t>(blockIdx.y) * 2 * a.width;
  p[c] = dw;
  p[a.width + c] = db;
}

// Adds the chunks' partial sums in order and rounds once.  One wave of each
// work-group takes every 16th chunk for 64 columns of dw (blockIdx.y 0) or db.
constexpr int kReduceWaves = 16;
template <typename P>
__global__ __launch_bounds__(64 * kReduceWaves) void norm_reduce(const float* __restrict__ part, int64_t chunks,
                                                                 int64_t width, P* dweight, P* dbias) {
  __shared__ float sums[kReduceWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  P* out = blockIdx.y == 0 ? dweight : dbias;
  float s = 0.0f;
  if (c < width) {
    const float* p = part + static_cast<int64_t>(blockIdx.y) * width + c;
    for (int64_t k = wave; k < chunks; k += kReduceWaves) s += p[k * 2 * width];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < width && out != nullptr) {
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < kReduceWaves; ++k) s += sums[k][lane];
    out[c] = static_cast<P>(s);
  }
}

// Row chunks of the column sums: enough for the chip, and few enough that the
// partial sums stay small against the rows.
int64_t column_chunks(int64_t rows, int64_t width) {
  int64_t want = ceil_div(4096, ceil_div(width, kThreads));
  if (want > ceil_div(rows, 16)) want = ceil_div(rows, 16);
  return want < 1 ? 1 : want;
}

unsigned row_blocks(int64_t rows) { return static_cast<unsigned>(rows < 65536 ? rows : 65536); }

spmm_status check_norm_desc(const spmm_norm_desc* d, const char* op) {
  if (d == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null descriptor");
  if (!dense_type(d->value_type))
    return fail(SPMM_ERR_CONTRACT, std::string(op) + " supports only FP16, BF16 and FP32 tensors");
  if (d->param_type != d->value_type && d->param_type != SPMM_VALUE_F32)
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": weight and bias must have the type of x or FP32");
  if (d->rows < 0) return fail(SPMM_ERR_CONTRACT, std::string(op) + ": negative extent");
  if (d->width < 1 || d->width > INT32_MAX)
    return fail(SPMM_ERR_CONTRACT, std::string(op) + " requires 1 <= width < 2^31, but got " + std::to_string(d->width));
  if (d->rows > 1 && d->x_stride < d->width)
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": rows of x overlap");
  if (!(d->eps >= 0.0) || std::isinf(d->eps))
    return fail(SPMM_ERR_INVALID_ARGUMENT, std::string(op) + ": eps must be finite and not negative");
  return SPMM_OK;
}

NormArgs norm_args(const spmm_norm_desc* d) {
  return {d->rows, d->width, d->x_stride, d->grad_stride, static_cast<float>(d->eps), d->param_type == SPMM_VALUE_F32};
}

template <typename T>
spmm_status run_forward(const spmm_norm_desc* d, const void* x, const void* w, const void* b, void* y, float* mean,
                        float* rstd, hipStream_t s) {
  hipLaunchKernelGGL(norm_forward_wide<T>, dim3(row_blocks(d->rows)), dim3(kThreads), 0, s, norm_args(d),
                     static_cast<const T*>(x), w, b, static_cast<T*>(y), mean, rstd);
  return check_launch("layer_norm");
}

template <typename T>
spmm_status run_backward(const spmm_norm_desc* d, const void* x, const void* w, const float* mean, const float* rstd,
                         const void* grad, void* dx, void* dw, void* db, float* part, hipStream_t s) {
  const NormArgs a = norm_args(d);
  const T *tx = static_cast<const T*>(x), *tg = static_cast<const T*>(grad);
  int64_t chunks = 0;
  if (d->rows > 0 && dx != nullptr) {
    hipLaunchKernelGGL(norm_backward_wide<T>, dim3(row_blocks(d->rows)), dim3(kThreads), 0, s, a, tx, w, mean, rstd,
                       tg, static_cast<T*>(dx));
    if (spmm_status st = check_launch("layer_norm_grad")) return st;
  }
  if (dw == nullptr && db == nullptr) return SPMM_OK;
  if (d->rows > 0) {
    const int64_t chunk = ceil_div(d->rows, column_chunks(d->rows, d->width));
    chunks = ceil_div(d->rows, chunk);
    hipLaunchKernelGGL(norm_columns_wide<T>,
                       dim3(static_cast<unsigned>(ceil_div(d->width, kThreads)), static_cast<unsigned>(chunks)),
                       dim3(kThreads), 0, s, a, tx, mean, rstd, tg, chunk, part);
    if (spmm_status st = check_launch("layer_norm_grad columns")) return st;
  }
  const dim3 grid(static_cast<unsigned>(ceil_div(d->width, 64)), 2);
  if (d->param_type == SPMM_VALUE_F32)
    hipLaunchKernelGGL(norm_reduce<float>, grid, dim3(64 * kReduceWaves), 0, s, part, chunks, d->width,
                       static_cast<float*>(dw), static_cast<float*>(db));
  else
    hipLaunchKernelGGL(norm_reduce<T>, grid, dim3(64 * kReduceWaves), 0, s, part, chunks, d->width,
                       static_cast<T*>(dw), static_cast<T*>(db));
  return check_launch("layer_norm_grad reduce");
}

size_t grad_workspace_bytes(const spmm_norm_desc* d) {
  return static_cast<size_t>(column_chunks(d->rows, d->width)) * 2 * static_cast<size_t>(d->width) * sizeof(float);
}

}  // namespace
}  // namespace spmm

using namespace spmm;

extern "C" {

spmm_status spmm_layer_norm_run(const spmm_norm_desc* d, const void* x, const void* weight, const void* bias, void* y,
                                float* mean, float* rstd, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_norm_desc(d, "layer_norm")) return st;
  if (d->rows == 0) return SPMM_OK;
  if (x == nullptr || y == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "layer_norm: null device pointer");
  hipStream_t s = as_stream(stream);
  switch (d->value_type) {
    case SPMM_VALUE_F16: return run_forward<_Float16>(d, x, weight, bias, y, mean, rstd, s);
    case SPMM_VALUE_BF16: return run_forward<__bf16>(d, x, weight, bias, y, mean, rstd, s);
    default: return run_forward<float>(d, x, weight, bias, y, mean, rstd, s);
  }
}

spmm_status spmm_layer_norm_grad_workspace(const spmm_norm_desc* d, size_t* bytes) {
  clear_error();
  if (bytes == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null argument");
  if (spmm_status st = check_norm_desc(d, "layer_norm")) return st;
  *bytes = grad_workspace_bytes(d);
  return SPMM_OK;
}

spmm_status spmm_layer_norm_grad_run(const spmm_norm_desc* d, const void* x, const void* weight, const float* mean,
                                     const float* rstd, const void* grad, void* dx, void* dweight, void* dbias,
                                     void* workspace, size_t workspace_bytes, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_norm_desc(d, "layer_norm")) return st;
  if (d->rows > 1 && d->grad_stride < d->width) return fail(SPMM_ERR_CONTRACT, "layer_norm: rows of grad overlap");
  if (dx == nullptr && dweight == nullptr && dbias == nullptr) return SPMM_OK;
  if (d->rows > 0 && (x == nullptr || mean == nullptr || rstd == nullptr || grad == nullptr))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "layer_norm: null device pointer");
  if ((dweight != nullptr || dbias != nullptr) && (workspace == nullptr || workspace_bytes < grad_workspace_bytes(d)))
    return fail(SPMM_ERR_CONTRACT, "layer_norm: workspace too small: need " + std::to_string(grad_workspace_bytes(d)) +
                                       " bytes");
  float* part = static_cast<float*>(workspace);
  hipStream_t s = as_stream(stream);
  switch (d->value_type) {
    case SPMM_VALUE_F16:
      return run_backward<_Float16>(d, x, weight, mean, rstd, grad, dx, dweight, dbias, part, s);
    case SPMM_VALUE_BF16:
      return run_backward<__bf16>(d, x, weight, mean, rstd, grad, dx, dweight, dbias, part, s);
    default: return run_backward<float>(d, x, weight, mean, rstd, grad, dx, dweight, dbias, part, s);
  }
}

}  // extern "C"
