// Newton-Schulz orthogonalisation of matrix updates.
//
// X0 = U / (|U|_F + eps), then each step X <- a X + (b A + c A A) X with
// A = X X^T, which maps X's singular values by a s + b s^3 + c s^5 and leaves
// its singular vectors.  Matrices with more rows than columns are turned, so
// that A is the smaller of the two Gram matrices.  A step is three products:
// A = X X^T, P = b A + c A A and a X + P X.
//
// X, A and P are held as fp16 planes, scaled by powers of two so that their
// entries stay in fp16's range: a bound on X's largest singular value follows
// from the coefficients, and no entry exceeds it.  The sum of a high and a low
// plane has 22 bits or more, and three products of planes (high high, high
// low, low high) added in fp32 give what fp32 products give.
//
// A bf16 update is rounded to 8 bits at the end, so its factors need fewer:
// one product of high planes, of 11 bits.  X keeps its low plane for a X, so
// that weak directions, which the steps raise most, are not lost beside strong
// ones; and the diagonals of A and P, where most of these matrices lies, are
// carried in fp32: with D what the high plane leaves of the diagonal, A A is
// taken as Ah Ah + D Ah + Ah D, and P X as Ph X + D X.  Against 64 bits the
// result is 1.05 to 1.4 times as far off as its rounding alone.
//
// Planes are padded with zeros to multiples of 64, which all products keep.
#include <climits>
#include <cmath>
#include <type_traits>
#include <utility>

#include "mma_ring.h"

namespace spmm {
namespace {

typedef _Float16 half;

constexpr int kThreads = 256;
constexpr int kNormParts = 64;  // work-groups that add up one matrix's squares
constexpr int64_t kCus = 256;

// Partial sums of squares in fp64: no overflow, and no loss against the total.
template <typename T>
__global__ __launch_bounds__(kThreads) void square_sums(const T* __restrict__ u, int64_t elements,
                                                        double* __restrict__ parts) {
  const T* m = u + blockIdx.y * elements;
  double s = 0.0;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * kPiece<T>; i < elements;
       i += static_cast<int64_t>(gridDim.x) * kThreads * kPiece<T>) {
    float v[kPiece<T>];
    load_piece(m + i, elements - i, v);
#pragma unroll
    for (int e = 0; e < kPiece<T>; ++e) s += static_cast<double>(v[e]) * static_cast<double>(v[e]);
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
  __shared__ double waves[kThreads / 64];
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 64; ++w) s += waves[w];
    parts[blockIdx.y * kNormParts + blockIdx.x] = s;
  }
}

// |U|_F + eps, by the 64 lanes of a wave alike.
__device__ inline double norm_of(const double* parts, double eps) {
  double s = parts[threadIdx.x & 63];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
  return sqrt(s) + eps;
}

__device__ inline void to_planes(float v, half& hi, half& lo) {
  hi = static_cast<half>(v);
  lo = static_cast<half>(v - static_cast<float>(hi));
}

// The planes of X0 times `scale`, of padded extents mp x np, turned where
// `tall`.  A work-group takes a tile of 64 x 64 through LDS.
template <typename T>
__global__ __launch_bounds__(kThreads) void scale_update(const T* __restrict__ u, int64_t rows, int64_t cols, bool tall,
                                                         double eps, double scale, const double* __restrict__ parts,
                                                         int64_t mp, int64_t np, half* __restrict__ hi,
                                                         half* __restrict__ lo) {
  __shared__ float tile[64][65];
  const double factor = scale / norm_of(parts + blockIdx.z * kNormParts, eps);
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 64, c0 = static_cast<int64_t>(blockIdx.x) * 64;
  const int64_t u0 = tall ? c0 : r0, v0 = tall ? r0 : c0;
  const T* m = u + blockIdx.z * rows * cols;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = wave; i < 64; i += kThreads / 64) {
    const bool in = u0 + i < rows && v0 + lane < cols;
    const double v = in ? static_cast<double>(static_cast<float>(m[(u0 + i) * cols + v0 + lane])) * factor : 0.0;
    if (tall) tile[lane][i] = static_cast<float>(v);
    else tile[i][lane] = static_cast<float>(v);
  }
  __syncthreads();
  for (int i = wave; i < 64; i += kThreads / 64) {
    const int64_t at = (blockIdx.z * mp + r0 + i) * np + c0 + lane;
    to_planes(tile[i][lane], hi[at], lo[at]);
  }
}

// A matrix of a batch in planes [rows][ld]; lo may be null.
struct Planes {
  half* hi;
  half* lo;
  int64_t ld, size;  // of a row, of a matrix
};

// What is done with the sums of a product: v = alpha * sum + (beta + alpha *
// (left[i] + right[j])) * E(i, j), E the planes `add` (and left[i] on the
// diagonal, where right is used), then stored as planes, or as the result.
struct Finish {
  float alpha, beta;
  Planes add;          // hi null: none
  const float* left;   // [batch][rows], what the high planes leave of a diagonal, or null
  bool both;           // right is left, and E lacks it on the diagonal
  Planes to;
  float* diagonal;     // [batch][rows]: what to.hi leaves of the diagonal, or null
  int64_t diagonal_rows;
  void* out;           // the result, [rows][cols] of the update's type and shape, or null
  int64_t rows, cols;
  bool tall;
};

template <typename T>
__device__ inline void finish_four(const Finish& f, int64_t batch, int64_t row, int64_t col, f32x4 sum) {
  f32x4 v = sum * f.alpha;
  if (f.add.hi != nullptr) {
    const int64_t at = batch * f.add.size + row * f.add.ld + col;
    const f16x4 h = *reinterpret_cast<const f16x4*>(f.add.hi + at);
    f16x4 l = {};
    if (f.add.lo != nullptr) l = *reinterpret_cast<const f16x4*>(f.add.lo + at);
    const float* d = f.left == nullptr ? nullptr : f.left + batch * f.diagonal_rows;
    const float r = d == nullptr ? 0.0f : d[row];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = static_cast<float>(h[e]) + static_cast<float>(l[e]);
      float w = f.beta + f.alpha * r;
      if (f.both) {
        w += f.alpha * d[col + e];
        if (row == col + e) x += r;
      }
      v[e] += w * x;
    }
  }
  if (f.out != nullptr) {
    T* out = static_cast<T*>(f.out) + batch * f.rows * f.cols;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t i = f.tall ? col + e : row, j = f.tall ? row : col + e;
      if (i < f.rows && j < f.cols) out[i * f.cols + j] = static_cast<T>(v[e]);
    }
    return;
  }
  f16x4 h, l;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = static_cast<half>(v[e]);
    l[e] = static_cast<half>(v[e] - static_cast<float>(h[e]));
    if (f.diagonal != nullptr && row == col + e)
      f.diagonal[batch * f.diagonal_rows + row] = v[e] - static_cast<float>(h[e]);
  }
  const int64_t at = batch * f.to.size + row * f.to.ld + col;
  *reinterpret_cast<f16x4*>(f.to.hi + at) = h;
  if (f.to.lo != nullptr) *reinterpret_cast<f16x4*>(f.to.lo + at) = l;
}

// The product of `left` [m][depth] with `right`, [n][depth], or [depth][n]
// where kTurned; extents are padded ones.
struct Product {
  Planes left, right;
  int64_t m, n, depth;
  int64_t splits;  // parts of the depth, each a sum of its own
  float* sums;     // [splits][batch][m][n] where there are several
};

__device__ inline mma::Operand<half> operand(const Planes& p, int64_t batch, int64_t first, int64_t most, int64_t rows,
                                             int64_t depth, bool turned) {
  const int64_t at = batch * p.size + (turned ? first : first * p.ld);
  return {p.hi + at, p.lo == nullptr ? nullptr : p.lo + at, p.ld, rows - first < most ? rows - first : most, depth};
}

// Tiles of a work-group in order: splits fastest outside a matrix's tiles.
template <typename T, bool kTurned, int kPlanes>
__global__ __launch_bounds__(mma::kThreads, 2) void product_large(Product p, Finish f) {
  __shared__ __align__(1024) char lds[mma::kLdsBytes];
  const int64_t down = (p.m + mma::kTile - 1) / mma::kTile, across = (p.n + mma::kTile - 1) / mma::kTile;
  const int64_t block = mma::run_of_xcd(blockIdx.x, gridDim.x), batch = block / (down * across);
  int64_t i, j;
  mma::place_tile(block % (down * across), down, across, i, j);
  const int64_t r0 = i * mma::kTile, c0 = j * mma::kTile;
  mma::Sums s;
  mma::multiply_tile<half, false, kTurned, kPlanes>(operand(p.left, batch, r0, mma::kTile, p.m, p.depth, false),
                                                    operand(p.right, batch, c0, mma::kTile, p.n, p.depth, kTurned), lds, s);
  mma::for_sums(s, [&](int row, int col, f32x4 v) {
    if (r0 + row < p.m && c0 + col < p.n) finish_four<T>(f, batch, r0 + row, c0 + col, v);
  });
}

template <typename T, bool kTurned, bool kPair>
__global__ __launch_bounds__(mma::kThreads128, kPair ? 1 : 2) void product_small(Product p, Finish f) {
  typedef mma::Ring<half, false, kTurned, kPair> Tile;
  __shared__ __align__(1024) char lds[Tile::kLdsBytes];
  const int64_t down = (p.m + 127) / 128, across = (p.n + 127) / 128;
  const int64_t block = mma::run_of_xcd(blockIdx.x, gridDim.x);
  const int64_t split = block / (down * across) % p.splits, batch = block / (down * across * p.splits);
  int64_t i, j;
  mma::place_tile(block % (down * across), down, across, i, j);
  const int64_t r0 = i * 128, c0 = j * 128;
  const int64_t steps = (p.depth + Tile::kDepth - 1) / Tile::kDepth;
  mma::Sums128<128> s;
  s.clear();
  Tile::add(operand(p.left, batch, r0, 128, p.m, p.depth, false), operand(p.right, batch, c0, 128, p.n, p.depth, kTurned),
            lds, static_cast<int>(steps * split / p.splits), static_cast<int>(steps * (split + 1) / p.splits), s);
  const int64_t batches = gridDim.x / (down * across * p.splits);
  float* to = p.sums + (split * batches + batch) * p.m * p.n;
  s.each([&](int row, int col, f32x4 v) {
    if (r0 + row >= p.m || c0 + col >= p.n) return;
    if (p.splits > 1) *reinterpret_cast<f32x4*>(to + (r0 + row) * p.n + c0 + col) = v;
    else finish_four<T>(f, batch, r0 + row, c0 + col, v);
  });
}

// Adds the splits' sums in order and finishes them.
template <typename T>
__global__ __launch_bounds__(kThreads) void finish_sums(Product p, Finish f, int64_t batches) {
  const int64_t fours = p.m * p.n / 4, n = fours * batches;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t k = 0; k < p.splits; ++k) s += *reinterpret_cast<const f32x4*>(p.sums + (k * n + i) * 4);
    const int64_t e = i % fours * 4;
    finish_four<T>(f, i / fours, e / p.n, e % p.n, s);
  }
}

// X0 itself (no steps): the planes' sum, unscaled.
template <typename T>
__global__ __launch_bounds__(kThreads) void store_planes(Finish f, int64_t mp, int64_t batches) {
  const int64_t fours = mp * f.add.ld / 4;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < fours * batches;
       i += static_cast<int64_t>(gridDim.x) * kThreads)
    finish_four<T>(f, i / fours, i % fours * 4 / f.add.ld, i % fours * 4 % f.add.ld, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
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

// Largest |c1 s + c3 s^3 + c5 s^5| for 0 <= s <= most.
double largest(double c1, double c3, double c5, double most) {
  auto at = [&](double s) { return std::fabs(s * (c1 + s * s * (c3 + s * s * c5))); };
  double found = at(most);
  // where the slope c1 + 3 c3 t + 5 c5 t^2 is zero, t = s^2
  const double a = 5 * c5, b = 3 * c3, root = b * b - 4 * a * c1;
  double t[2] = {-1.0, -1.0};
  if (a == 0.0) {
    if (b != 0.0) t[0] = -c1 / b;
  } else if (root >= 0.0) {
    t[0] = (-b + std::sqrt(root)) / (2 * a);
    t[1] = (-b - std::sqrt(root)) / (2 * a);
  }
  for (double v : t)
    if (v > 0.0 && v < most * most) found = std::fmax(found, at(std::sqrt(v)));
  return found;
}

// Power of two that takes entries of at most `most` to 2^13 .. 2^14: a quarter
// of fp16's range is left for rounding, and low planes stay clear of its least.
double scale_for(double most) {
  if (!(most > 1e-30)) most = 1e-30;
  return std::exp2(std::floor(std::log2(16384.0 / most)));
}

// X twice (a step reads one and writes the other), A and P in planes, their
// diagonals' rests, the sums of squares, and the sums of split products.
// m <= n: the matrix's extents, mp and np padded.
struct Layout {
  int64_t m, n, mp, np;
  bool pair;  // three products of planes; else one
  size_t x, gram, diagonal, parts, sums;
  explicit Layout(const spmm_orthogonalize_desc* d) {
    m = d->rows < d->width ? d->rows : d->width;
    n = d->rows < d->width ? d->width : d->rows;
    mp = align_up(m, 64);
    np = align_up(n, 64);
    pair = d->value_type != SPMM_VALUE_BF16 || m < 128;
    x = align_up(static_cast<size_t>(d->batch * mp * np) * sizeof(half), 256);
    gram = align_up(static_cast<size_t>(d->batch * mp * mp) * sizeof(half), 256);
    diagonal = align_up(static_cast<size_t>(d->batch * mp) * sizeof(float), 256);
    parts = align_up(static_cast<size_t>(d->batch * kNormParts) * sizeof(double), 256);
    sums = 0;
    for (const bool wide : {false, true}) {
      const int64_t cols = wide ? np : mp, depth = wide ? mp : np, k = splits(d->batch, mp, cols, depth);
      const size_t bytes = k > 1 ? static_cast<size_t>(k * d->batch * mp * cols) * sizeof(float) : 0;
      sums = sums > bytes ? sums : bytes;
    }
  }
  size_t total() const { return 4 * x + 4 * gram + 2 * diagonal + parts + sums; }

  // The large tile where three quarters of the CUs get one, and fill it.
  static bool large(int64_t batch, int64_t rows, int64_t cols) {
    return rows > 128 && cols > 128 && batch * ceil_div(rows, mma::kTile) * ceil_div(cols, mma::kTile) >= kCus * 3 / 4;
  }
  // Parts of the depth, of four steps or more, where there are few tiles.
  static int64_t splits(int64_t batch, int64_t rows, int64_t cols, int64_t depth) {
    if (batch == 0 || rows == 0 || cols == 0 || large(batch, rows, cols)) return 1;
    const int64_t tiles = batch * ceil_div(rows, 128) * ceil_div(cols, 128);
    int64_t k = kCus / tiles, most = depth / (4 * mma::kDepth);
    k = k < most ? k : most;
    return k < 1 ? 1 : k;
  }
};

template <typename T, bool kTurned, bool kPair>
spmm_status multiply(Product p, const Finish& f, int64_t batch, hipStream_t s) {
  if (Layout::large(batch, p.m, p.n)) {
    const unsigned tiles = static_cast<unsigned>(ceil_div(p.m, mma::kTile) * ceil_div(p.n, mma::kTile) * batch);
    hipLaunchKernelGGL((product_large<T, kTurned, kPair ? 3 : 1>), dim3(tiles), dim3(mma::kThreads), 0, s, p, f);
    return check_launch("orthogonalize product");
  }
  p.splits = Layout::splits(batch, p.m, p.n, p.depth);
  const unsigned tiles = static_cast<unsigned>(ceil_div(p.m, 128) * ceil_div(p.n, 128) * batch * p.splits);
  hipLaunchKernelGGL((product_small<T, kTurned, kPair>), dim3(tiles), dim3(mma::kThreads128), 0, s, p, f);
  if (spmm_status st = check_launch("orthogonalize product")) return st;
  if (p.splits == 1) return SPMM_OK;
  const int64_t blocks = ceil_div(p.m * p.n / 4 * batch, kThreads);
  hipLaunchKernelGGL(finish_sums<T>, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(kThreads), 0, s, p,
                     f, batch);
  return check_launch("orthogonalize sums");
}

template <typename T, bool kTurned>
spmm_status multiply(const Product& p, const Finish& f, int64_t batch, bool pair, hipStream_t s) {
  if constexpr (std::is_same_v<T, __bf16>)
    if (!pair) return multiply<T, kTurned, false>(p, f, batch, s);
  return multiply<T, kTurned, true>(p, f, batch, s);
}

template <typename T>
spmm_status run(const spmm_orthogonalize_desc* d, const Layout& l, const void* update, void* out, char* ws,
                hipStream_t s) {
  const bool tall = d->rows > d->width;
  auto take = [&](size_t bytes) {
    char* p = ws;
    ws += bytes;
    return p;
  };
  auto planes = [&](size_t bytes, int64_t ld, bool low) {
    half* hi = reinterpret_cast<half*>(take(bytes));
    half* lo = reinterpret_cast<half*>(take(bytes));
    return Planes{hi, low ? lo : nullptr, ld, l.mp * ld};
  };
  Planes x = planes(l.x, l.np, true), y = planes(l.x, l.np, true);
  const Planes gram = planes(l.gram, l.mp, l.pair), poly = planes(l.gram, l.mp, l.pair);
  float* gram_rest = l.pair ? nullptr : reinterpret_cast<float*>(ws);
  take(l.diagonal);
  float* poly_rest = l.pair ? nullptr : reinterpret_cast<float*>(ws);
  take(l.diagonal);
  double* parts = reinterpret_cast<double*>(take(l.parts));
  float* sums = reinterpret_cast<float*>(ws);
  const T* u = static_cast<const T*>(update);
  const unsigned batch = static_cast<unsigned>(d->batch);
  double bound = 1.0, sx = scale_for(bound);
  hipLaunchKernelGGL(square_sums<T>, dim3(kNormParts, batch), dim3(kThreads), 0, s, u, l.m * l.n, parts);
  hipLaunchKernelGGL(scale_update<T>, dim3(static_cast<unsigned>(l.np / 64), static_cast<unsigned>(l.mp / 64), batch),
                     dim3(kThreads), 0, s, u, d->rows, d->width, tall, d->eps, sx, parts, l.mp, l.np, x.hi, x.lo);
  if (spmm_status st = check_launch("orthogonalize scale")) return st;
  Finish f{};
  f.diagonal_rows = l.mp;
  f.rows = d->rows;
  f.cols = d->width;
  f.tall = tall;
  if (d->steps == 0) {
    f.beta = static_cast<float>(1.0 / sx);
    f.add = x;
    f.out = out;
    const int64_t blocks = ceil_div(l.mp * l.np / 4 * d->batch, kThreads);
    hipLaunchKernelGGL(store_planes<T>, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(kThreads), 0, s,
                       f, l.mp, d->batch);
    return check_launch("orthogonalize result");
  }
  for (int64_t i = 0; i < d->steps; ++i) {
    const double *c = d->coefficients + 3 * i, t = bound * bound;
    // b t + c t^2 on [0, bound^2], as an odd polynomial's largest
    double high = std::fabs(c[1] * t + c[2] * t * t);
    if (c[2] != 0.0 && -c[1] / (2 * c[2]) > 0.0 && -c[1] / (2 * c[2]) < t)
      high = std::fmax(high, std::fabs(c[1] * c[1] / (4 * c[2])));
    const double sa = scale_for(t), sp = scale_for(high);
    bound = largest(c[0], c[1], c[2], bound);
    const double next = i + 1 < d->steps ? scale_for(bound) : 1.0;
    Finish g = f;
    g.alpha = static_cast<float>(sa / (sx * sx));
    g.to = gram;
    g.diagonal = gram_rest;
    if (spmm_status st = multiply<T, false>({x, x, l.mp, l.mp, l.np, 1, sums}, g, d->batch, l.pair, s)) return st;
    g.alpha = static_cast<float>(sp * c[2] / (sa * sa));
    g.beta = static_cast<float>(sp * c[1] / sa);
    g.add = gram;
    g.left = gram_rest;
    g.both = gram_rest != nullptr;
    g.to = poly;
    g.diagonal = poly_rest;
    if (spmm_status st = multiply<T, false>({gram, gram, l.mp, l.mp, l.mp, 1, sums}, g, d->batch, l.pair, s)) return st;
    g.alpha = static_cast<float>(next / (sp * sx));
    g.beta = static_cast<float>(next * c[0] / sx);
    g.add = x;
    g.left = poly_rest;
    g.both = false;
    g.to = y;
    g.diagonal = nullptr;
    g.out = i + 1 < d->steps ? nullptr : out;
    if (spmm_status st = multiply<T, true>({poly, x, l.mp, l.np, l.mp, 1, sums}, g, d->batch, l.pair, s)) return st;
    std::swap(x, y);
    sx = next;
  }
  return SPMM_OK;
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
  if (ceil_div(l.mp, 128) * ceil_div(l.np, 128) * d->batch > INT32_MAX / 64 || l.np / 64 > 65535 * 64 || l.mp / 64 > 65535)
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
