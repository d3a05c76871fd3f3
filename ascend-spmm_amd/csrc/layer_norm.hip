// Layer norm over the last dimension, forward and backward.
//
// With z = (x - mean) * rstd, y = z w + b and g = dy w, a row's gradient is
// dx = rstd * (g - mean(g) - z mean(g z)); dw and db are the column sums of
// dy z and dy over all rows.  Statistics and sums are fp32; the variance is
// the mean of squared distances from the mean (a second pass over the row),
// which keeps its digits where the mean is large against the spread.
#include <climits>
#include <cmath>
#include <type_traits>

#include "numeric.h"

namespace spmm {
namespace {

constexpr int kThreads = 256;

// Most work-groups.  Each of the backward kernel leaves one row of partial sums
// of the parameters' gradients, which cost more to write and add the more there
// are: 65536 x 1024 bf16 takes 75 + 4 us (with adding them) with 512, and 768
// gained nothing; the forward pass 50 us with 2048, 46 with 4096.  Both move
// 5.3 TB/s and more.
constexpr int64_t kBackwardGroups = 512, kForwardGroups = 4096;

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

// Sums of K values over the L lanes that share a row: a part of a wave, or
// the whole work-group.
template <int L, int K>
__device__ inline void row_sum(float (&v)[K]) {
  if constexpr (L > 64) {
    block_sum(v);
  } else {
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], d);
  }
}

// The register kernels.  L lanes share a row (a work-group of 256 has 256 / L
// rows at once, or one of more than a wave) and each holds I pieces of 16 bytes of it, so x (and
// grad) is read once.  A group walks rows a grid apart and loads the next
// row's pieces before it reduces the current one.
template <typename T, int L, int I>
struct RowTile {
  static constexpr int V = kPiece<T>;
  static constexpr int kBlock = L > 64 ? L : kThreads;
  static constexpr int kGroups = kBlock / L;

  __device__ static inline int64_t column(int i) { return static_cast<int64_t>((i * L + threadIdx.x % L)) * V; }

  __device__ static inline void load(const T* row, int64_t width, piece_t<T> (&v)[I]) {
#pragma unroll
    for (int i = 0; i < I; ++i) v[i] = load_raw(row + column(i), width - column(i));
  }
};

template <typename T, int L, int I>
__global__ __launch_bounds__((RowTile<T, L, I>::kBlock)) void norm_forward(NormArgs a, const T* __restrict__ x,
                                                                           const void* __restrict__ w,
                                                                           const void* __restrict__ b,
                                                                           T* __restrict__ y, float* mean, float* rstd) {
  using Tile = RowTile<T, L, I>;
  constexpr int V = Tile::V;
  const float count = static_cast<float>(a.width);
  const int64_t step = static_cast<int64_t>(gridDim.x) * Tile::kGroups;
  int64_t r = static_cast<int64_t>(blockIdx.x) * Tile::kGroups + threadIdx.x / L;
  float wv[I][V], bv[I][V];
  piece_t<T> next[I];
  if (r < a.rows) Tile::load(x + r * a.x_stride, a.width, next);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    load_param<T>(w, a.param_f32, Tile::column(i), a.width, 1.0f, wv[i]);
    load_param<T>(b, a.param_f32, Tile::column(i), a.width, 0.0f, bv[i]);
  }
  // Groups of a work-group stay together (block_sum's barriers).
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * Tile::kGroups; r0 < a.rows; r0 += step, r += step) {
    float v[I][V], s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = static_cast<float>(next[i][j]);
    if (r + step < a.rows) Tile::load(x + (r + step) * a.x_stride, a.width, next);
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += v[i][j];
    row_sum<L>(s);
    const float m = s[0] / count;
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = Tile::column(i) + j < a.width ? v[i][j] - m : 0.0f;
        s[0] += v[i][j] * v[i][j];
      }
    row_sum<L>(s);
    const float rs = 1.0f / sqrtf(s[0] / count + a.eps);
    if (r >= a.rows) continue;
    if (threadIdx.x % L == 0 && mean != nullptr) mean[r] = m;
    if (threadIdx.x % L == 0 && rstd != nullptr) rstd[r] = rs;
#pragma unroll
    for (int i = 0; i < I; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = v[i][j] * rs * wv[i][j] + bv[i][j];
      store_piece(y + r * a.width + Tile::column(i), a.width - Tile::column(i), v[i]);
    }
  }
}

// dx of each row, and the column sums of dy z and dy over the rows of the
// work-group: part[group][2][width].
template <typename T, int L, int I>
__global__ __launch_bounds__((RowTile<T, L, I>::kBlock)) void norm_backward(NormArgs a, const T* __restrict__ x,
                                                                            const void* __restrict__ w,
                                                                            const float* __restrict__ mean,
                                                                            const float* __restrict__ rstd,
                                                                            const T* __restrict__ grad,
                                                                            T* __restrict__ dx, float* part) {
  using Tile = RowTile<T, L, I>;
  constexpr int V = Tile::V;
  const float count = static_cast<float>(a.width);
  const int64_t step = static_cast<int64_t>(gridDim.x) * Tile::kGroups;
  int64_t r = static_cast<int64_t>(blockIdx.x) * Tile::kGroups + threadIdx.x / L;
  float wv[I][V], dw[I][V] = {}, db[I][V] = {}, nm = 0.0f, nrs = 0.0f;
  piece_t<T> nx[I] = {}, ng[I] = {};
  auto fetch = [&](int64_t row) {
    Tile::load(x + row * a.x_stride, a.width, nx);
    Tile::load(grad + row * a.grad_stride, a.width, ng);
    nm = mean[row];
    nrs = rstd[row];
  };
  if (r < a.rows) fetch(r);
#pragma unroll
  for (int i = 0; i < I; ++i) load_param<T>(w, a.param_f32, Tile::column(i), a.width, 1.0f, wv[i]);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * Tile::kGroups; r0 < a.rows; r0 += step, r += step) {
    float z[I][V], g[I][V], s[2] = {0.0f, 0.0f};
    const float m = nm, rs = nrs;
    const bool live = r < a.rows;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        z[i][j] = static_cast<float>(nx[i][j]);
        g[i][j] = static_cast<float>(ng[i][j]);
      }
    if (r + step < a.rows) fetch(r + step);
    if (live) {
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const bool in = Tile::column(i) + j < a.width;
          z[i][j] = in ? (z[i][j] - m) * rs : 0.0f;
          dw[i][j] += g[i][j] * z[i][j];
          db[i][j] += g[i][j];
          g[i][j] = in ? g[i][j] * wv[i][j] : 0.0f;
          s[0] += g[i][j];
          s[1] += g[i][j] * z[i][j];
        }
    }
    if (dx == nullptr) continue;
    row_sum<L>(s);
    if (!live) continue;
    const float g0 = s[0] / count, g1 = s[1] / count;
#pragma unroll
    for (int i = 0; i < I; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) g[i][j] = rs * (g[i][j] - g0 - z[i][j] * g1);
      store_piece(dx + r * a.width + Tile::column(i), a.width - Tile::column(i), g[i]);
    }
  }
  if (part == nullptr) return;
  // The work-group's groups in turn: within a wave by lane exchange, then the
  // waves through LDS.
  float* p = part + static_cast<int64_t>(blockIdx.x) * 2 * a.width;
  if constexpr (L <= 64) {
    constexpr int W = Tile::kBlock / 64;
    __shared__ float lds[W][2][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < I; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int d = L; d < 64; d <<= 1) {
          dw[i][j] += __shfl_xor(dw[i][j], d);
          db[i][j] += __shfl_xor(db[i][j], d);
        }
      }
      __syncthreads();
      if (lane < L)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          lds[wave][0][lane * V + j] = dw[i][j];
          lds[wave][1][lane * V + j] = db[i][j];
        }
      __syncthreads();
      for (int k = threadIdx.x; k < 2 * L * V; k += Tile::kBlock) {
        const int which = k / (L * V), c = k % (L * V);
        const int64_t col = static_cast<int64_t>(i) * L * V + c;
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < W; ++q) sum += lds[q][which][c];
        if (col < a.width) p[which * a.width + col] = sum;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int64_t col = Tile::column(i) + j;
        if (col < a.width) {
          p[col] = dw[i][j];
          p[a.width + col] = db[i][j];
        }
      }
  }
}

// Wider rows than the registers of a work-group hold: one work-group per row,
// the row read three times, for the mean, the variance and the result (4096 x
// 20000 bf16: 103 us, 67 at the rate of a copy).
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_forward_wide(NormArgs a, const T* __restrict__ x,
                                                              const void* __restrict__ w, const void* __restrict__ b,
                                                              T* __restrict__ y, float* mean, float* rstd) {
  constexpr int V = kPiece<T>;
  const float count = static_cast<float>(a.width);
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
    const float m = s[0] / count;
    s[0] = 0.0f;
    for (int64_t c = threadIdx.x * V; c < a.width; c += kThreads * V) {
      float v[V];
      load_piece(xr + c, a.width - c, v);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i < a.width) s[0] += (v[i] - m) * (v[i] - m);
    }
    block_sum(s);
    const float rs = 1.0f / sqrtf(s[0] / count + a.eps);
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
  const float count = static_cast<float>(a.width);
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
    const float g0 = s[0] / count, g1 = s[1] / count;
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
#pragma unroll 8
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

// Calls f(L, I) with the lanes per row and pieces per lane for rows of
// `width`: the fewest lanes that hold the row in one piece each, then up to
// four pieces each of one to eight waves (more would not leave registers for
// the sums).  False where the row is wider than that.
template <typename T, typename F>
bool with_tile(int64_t width, F f) {
  const int64_t pieces = ceil_div(width, kPiece<T>);
#define SPMM_TILE(L, I) \
  if (pieces <= (L) * (I)) return f(std::integral_constant<int, L>(), std::integral_constant<int, I>()), true
  SPMM_TILE(8, 1);
  SPMM_TILE(16, 1);
  SPMM_TILE(32, 1);
  SPMM_TILE(64, 1);
  SPMM_TILE(64, 2);
  SPMM_TILE(64, 4);
  SPMM_TILE(128, 3);
  SPMM_TILE(128, 4);
  SPMM_TILE(256, 3);
  SPMM_TILE(256, 4);
  SPMM_TILE(512, 3);
  SPMM_TILE(512, 4);
#undef SPMM_TILE
  return false;
}

int64_t tile_groups(int64_t width, int64_t piece) {
  const int64_t pieces = ceil_div(width, piece);
  for (int64_t lanes = 8; lanes <= 64; lanes *= 2)
    if (pieces <= lanes) return kThreads / lanes;
  return pieces <= 256 ? kThreads / 64 : 1;
}

// Work-groups of the backward kernel: each has four rows per group at least,
// so that its partial sums cost little against its rows.
int64_t backward_blocks(int64_t rows, int64_t groups) {
  const int64_t want = ceil_div(rows, 4 * groups);
  return want < kBackwardGroups ? want : kBackwardGroups;
}

template <typename T>
spmm_status run_forward(const spmm_norm_desc* d, const void* x, const void* w, const void* b, void* y, float* mean,
                        float* rstd, hipStream_t s) {
  const bool tiled = with_tile<T>(d->width, [&](auto L, auto I) {
    using Tile = RowTile<T, decltype(L)::value, decltype(I)::value>;
    const int64_t blocks = ceil_div(d->rows, Tile::kGroups), most = kForwardGroups;
    hipLaunchKernelGGL((norm_forward<T, decltype(L)::value, decltype(I)::value>),
                       dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(Tile::kBlock), 0, s,
                       norm_args(d), static_cast<const T*>(x), w, b, static_cast<T*>(y), mean, rstd);
  });
  if (tiled) return check_launch("layer_norm");
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
  const bool sums = dw != nullptr || db != nullptr;
  const bool tiled = d->rows > 0 && with_tile<T>(d->width, [&](auto L, auto I) {
    using Tile = RowTile<T, decltype(L)::value, decltype(I)::value>;
    chunks = backward_blocks(d->rows, Tile::kGroups);
    hipLaunchKernelGGL((norm_backward<T, decltype(L)::value, decltype(I)::value>),
                       dim3(static_cast<unsigned>(chunks)), dim3(Tile::kBlock), 0, s, a, tx, w, mean, rstd, tg,
                       static_cast<T*>(dx), sums ? part : nullptr);
  });
  if (tiled)
    if (spmm_status st = check_launch("layer_norm_grad")) return st;
  if (!tiled && d->rows > 0 && dx != nullptr) {
    hipLaunchKernelGGL(norm_backward_wide<T>, dim3(row_blocks(d->rows)), dim3(kThreads), 0, s, a, tx, w, mean, rstd,
                       tg, static_cast<T*>(dx));
    if (spmm_status st = check_launch("layer_norm_grad")) return st;
  }
  if (!sums) return SPMM_OK;
  if (!tiled && d->rows > 0) {
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
  const int64_t piece = 16 / dense_type_bytes(d->value_type);
  const bool tiled = ceil_div(d->width, piece) <= 2048;  // the widest tile
  const int64_t chunks = tiled ? backward_blocks(d->rows, tile_groups(d->width, piece))
                               : column_chunks(d->rows, d->width);
  return static_cast<size_t>(chunks) * 2 * static_cast<size_t>(d->width) * sizeof(float);
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
  const size_t need = dweight != nullptr || dbias != nullptr ? grad_workspace_bytes(d) : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(SPMM_ERR_CONTRACT, "layer_norm: workspace too small: need " + std::to_string(need) + " bytes");
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
