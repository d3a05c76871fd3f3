// Newton-Schulz orthogonalisation of matrix updates.
//
// X0 = U / (|U|_F + eps), then each step X <- a X + (b A + c A A) X with
// A = X X^T, which maps X's singular values by a s + b s^3 + c s^5 and leaves
// its singular vectors.  Matrices with more rows than columns are turned, so
// that A is the smaller of the two Gram matrices.  A step is three products:
// A = X X^T, P = b A + c A A and a X + P X.
//
// X is held in fp32.  The products' factors are fp16 planes, a high and a low
// one whose sum has 22 bits or more of what it stands for; three products of
// planes (low high, high low, high high) added in fp32 give what fp32 products
// give.  Planes are scaled by powers of two so that they stay in fp16's range
// whatever the matrix holds: X's rows for A = X X^T by their own size each, X's
// columns for P X by theirs, A's and P's rows by what X's rows bound them to.
// So a weak row or column keeps its digits beside strong ones, and a small
// matrix keeps them too.  A step takes row and column norms to at most
// |a + b s^2 + c s^4| times what they were, s up to X's largest singular value,
// which the coefficients bound as well: the exponents of every step follow from
// those of X0 without another look at X (Levels).
//
// The diagonals of A and P, where most of these matrices lies, are carried in
// fp32 and are zeros in the planes: with D the diagonal, A A is taken as A' A' +
// D A' + A' D + D D, and P X as P' X + D X.  Matrix instructions cut their sums
// to fp32 (they do not round), always to the same side; without the large
// terms, and with products of low planes summed apart or first, little is lost.
//
// A bf16 update is rounded to 8 bits at the end, so its factors need fewer: one
// product of high planes, of 11 bits, unless the caller asks for all (precise).
// Against 64 bits a 4096 x 4096 result is 1.74e-3 off so (the rounding to 8
// bits alone is 1.66e-3), in a third of the matrix instructions.
//
// Planes are padded with zeros to multiples of 64, which all products keep.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>
#include <utility>

#include "mma_ring.h"

namespace spmm {
namespace {

typedef _Float16 half;

constexpr int kThreads = 256;
constexpr int64_t kCus = 256;

// Exponents of magnitudes: v < 2^e, no smaller than kLeast, so that a plane's
// scale 2^(14 - e) and its inverse are fp32 numbers.
constexpr int kLeast = -112, kMost = 126;

__host__ __device__ inline int clamped(int e) { return e < kLeast ? kLeast : e > kMost ? kMost : e; }
__device__ inline float power(int e) { return __builtin_bit_cast(float, (e + 127) << 23); }
// Takes magnitudes below 2^e to below 2^14: a quarter of fp16's range is left
// for rounding.
__device__ inline float scale_of(int e) { return power(14 - e); }
__device__ inline float unscale_of(int e) { return power(e - 14); }

// Of a step: exponents of the growth of X's rows and columns so far, of X's
// largest singular value, and of the largest |b + c s^2|, which bounds P's
// entries against the rows that it is made of.
struct Levels {
  int growth, bound, high;
};
// X's row or column whose norm in X0 is below 2^e; of A's row; of P's row.
__device__ inline int level_x(const Levels& l, int e) {
  e += l.growth;
  return clamped(e < l.bound ? e : l.bound);
}
__device__ inline int level_a(const Levels& l, int e) { return clamped(level_x(l, e) + l.bound); }
__device__ inline int level_p(const Levels& l, int e) { return clamped(level_x(l, e) + l.bound + l.high); }

// Exponent for a row or column of `count` entries, the largest of them `most`:
// its norm is at most sqrt(count) times that.
__device__ inline int exponent_of(double most, int64_t count) {
  const double v = most * sqrt(static_cast<double>(count));
  if (!(v > 0.0)) return kLeast;
  return clamped(static_cast<int>((__builtin_bit_cast(unsigned long long, v) >> 52 & 2047)) - 1022);
}

// What a first pass over the update finds in tiles of kMeasureRows rows and a
// piece of 16 bytes for each lane across: each row's and each column's largest
// magnitude, and sums of squares in fp64 (no overflow, and no loss against the
// total).
constexpr int kMeasureRows = 32;
template <typename T>
constexpr int kMeasureCols = 64 * kPiece<T>;
struct Measures {
  float* rows;   // [batch][rows][tiles across]
  float* cols;   // [batch][tiles down][cols]
  double* sums;  // [batch][tiles]
};

template <typename T>
__global__ __launch_bounds__(kThreads) void measure_update(const T* __restrict__ u, int64_t rows, int64_t cols,
                                                           Measures w) {
  constexpr int V = kPiece<T>, kWaves = kThreads / 64, kEach = kMeasureRows / kWaves;
  const unsigned across = static_cast<unsigned>((cols + kMeasureCols<T> - 1) / kMeasureCols<T>);
  const unsigned tiles = gridDim.x, down = tiles / across, i = blockIdx.x / across, j = blockIdx.x - i * across;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r0 = static_cast<int64_t>(i) * kMeasureRows + wave * kEach;
  const int64_t c0 = static_cast<int64_t>(j) * kMeasureCols<T> + lane * V;
  const T* m = u + blockIdx.y * rows * cols;
  piece_t<T> x[kEach];
#pragma unroll
  for (int r = 0; r < kEach; ++r) x[r] = load_raw(m + (r0 + r) * cols + c0, r0 + r < rows ? cols - c0 : 0);
  double s = 0.0;
  float col[V] = {}, row[kEach] = {};
#pragma unroll
  for (int r = 0; r < kEach; ++r)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float v = static_cast<float>(x[r][e]);
      s += static_cast<double>(v) * static_cast<double>(v);
      col[e] = fmaxf(col[e], fabsf(v));
      row[r] = fmaxf(row[r], fabsf(v));
    }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    s += __shfl_xor(s, d);
#pragma unroll
    for (int r = 0; r < kEach; ++r) row[r] = fmaxf(row[r], __shfl_xor(row[r], d));
  }
  __shared__ float high[kWaves][kMeasureCols<T>];
  __shared__ double sums[kWaves];
#pragma unroll
  for (int e = 0; e < V; ++e) high[wave][lane * V + e] = col[e];
  if (lane == 0) {
    sums[wave] = s;
#pragma unroll
    for (int r = 0; r < kEach; ++r)
      if (r0 + r < rows) w.rows[(blockIdx.y * rows + r0 + r) * across + j] = row[r];
  }
  __syncthreads();
  for (int k = threadIdx.x; k < kMeasureCols<T>; k += kThreads) {
    const int64_t c = static_cast<int64_t>(j) * kMeasureCols<T> + k;
    float most = 0.0f;
#pragma unroll
    for (int n = 0; n < kWaves; ++n) most = fmaxf(most, high[n][k]);
    if (c < cols) w.cols[(static_cast<int64_t>(blockIdx.y) * down + i) * cols + c] = most;
  }
  if (threadIdx.x == 0) {
    for (int k = 1; k < kWaves; ++k) s += sums[k];
    w.sums[static_cast<int64_t>(blockIdx.y) * tiles + blockIdx.x] = s;
  }
}

// The factor that takes the update to X0, and the exponents of X0's rows and
// columns, padded ones among them (`tall`: of the update's columns and rows).
// The first work-groups take a row of the update a wave, the rest a column a
// lane; each adds up the sums of squares for itself, in the same order.
struct Exponents {
  int* rows;  // [batch][mp]
  int* cols;  // [batch][np]
  double* factor;
};

__global__ __launch_bounds__(kThreads) void update_exponents(Measures w, int64_t rows, int64_t cols, int64_t down,
                                                             int64_t across, bool tall, double eps, int64_t rows_padded,
                                                             int64_t cols_padded, Exponents x) {
  const int64_t tiles = across * down, batch = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double s = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < tiles; i += kThreads) s += w.sums[batch * tiles + i];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
  __shared__ double waves[kThreads / 64];
  if (lane == 0) waves[wave] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int k = 0; k < kThreads / 64; ++k) s += waves[k];
  const double factor = 1.0 / (sqrt(s) + eps);
  if (blockIdx.x == 0 && threadIdx.x == 0) x.factor[batch] = factor;

  constexpr int kRows = kThreads / 64;
  const int64_t row_blocks = (rows_padded + kRows - 1) / kRows;
  float most = 0.0f;
  if (blockIdx.x < row_blocks) {
    const int64_t r = blockIdx.x * kRows + wave;
    if (r < rows)
#pragma unroll 4
      for (int64_t k = lane; k < across; k += 64) most = fmaxf(most, w.rows[(batch * rows + r) * across + k]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    if (lane == 0 && r < rows_padded)
      (tall ? x.cols : x.rows)[batch * rows_padded + r] = exponent_of(most * factor, cols);
  } else {
    __shared__ float high[kThreads / 64][64];
    const int64_t c = (blockIdx.x - row_blocks) * 64 + lane;
    if (c < cols)
#pragma unroll 16
      for (int64_t k = wave; k < down; k += kThreads / 64) most = fmaxf(most, w.cols[(batch * down + k) * cols + c]);
    high[wave][lane] = most;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kThreads / 64; ++k) most = fmaxf(most, high[k][lane]);
    if (wave == 0 && c < cols_padded) (tall ? x.rows : x.cols)[batch * cols_padded + c] = exponent_of(most * factor, rows);
  }
}

// A matrix of a batch in planes [rows][ld]; lo may be null.
struct Planes {
  half* hi;
  half* lo;
  int64_t ld, size;  // of a row, of a matrix
};

// X0 in fp32, and in planes scaled by rows and by columns, of padded extents
// mp x np, turned where `tall`.  A work-group takes a tile of 64 x 64 through
// LDS.
template <typename T>
__global__ __launch_bounds__(kThreads) void scale_update(const T* __restrict__ u, int64_t rows, int64_t cols, bool tall,
                                                         Exponents e, Levels l, int64_t mp, int64_t np,
                                                         float* __restrict__ x, Planes by_row, Planes by_col) {
  __shared__ float tile[64][65];
  const double factor = e.factor[blockIdx.z];
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 64, c0 = static_cast<int64_t>(blockIdx.x) * 64;
  const int64_t u0 = tall ? c0 : r0, v0 = tall ? r0 : c0;
  const T* m = u + blockIdx.z * rows * cols;
  typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  const int c = threadIdx.x % 16 * 4;
  Four loaded[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t r = u0 + threadIdx.x / 16 + 16 * k, left = r < rows ? cols - v0 - c : 0;
    const T* at = m + r * cols + v0 + c;
    if (left >= 4) loaded[k] = *reinterpret_cast<const Four*>(at);
    else
#pragma unroll
      for (int n = 0; n < 4; ++n) loaded[k][n] = n < left ? at[n] : static_cast<T>(0.0f);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int i = threadIdx.x / 16 + 16 * k;
      const float v = static_cast<float>(static_cast<double>(static_cast<float>(loaded[k][n])) * factor);
      if (tall) tile[c + n][i] = v;
      else tile[i][c + n] = v;
    }
  __syncthreads();
  float across[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) across[k] = scale_of(level_x(l, e.cols[blockIdx.z * np + c0 + c + k]));
  for (int i = threadIdx.x / 16; i < 64; i += kThreads / 16) {
    const int64_t at = (blockIdx.z * mp + r0 + i) * np + c0 + c;
    const float down = scale_of(level_x(l, e.rows[blockIdx.z * mp + r0 + i]));
    f32x4 v;
    f16x4 rh, rl, ch, cl;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = tile[i][c + k];
      rh[k] = static_cast<half>(v[k] * down);
      rl[k] = static_cast<half>(v[k] * down - static_cast<float>(rh[k]));
      ch[k] = static_cast<half>(v[k] * across[k]);
      cl[k] = static_cast<half>(v[k] * across[k] - static_cast<float>(ch[k]));
    }
    *reinterpret_cast<f32x4*>(x + at) = v;
    *reinterpret_cast<f16x4*>(by_row.hi + at) = rh;
    *reinterpret_cast<f16x4*>(by_col.hi + at) = ch;
    if (by_row.lo == nullptr) continue;
    *reinterpret_cast<f16x4*>(by_row.lo + at) = rl;
    *reinterpret_cast<f16x4*>(by_col.lo + at) = cl;
  }
}

// X0 itself (no steps).
template <typename T>
__global__ __launch_bounds__(kThreads) void store_scaled(const T* u, int64_t elements, const double* __restrict__ factor,
                                                         T* out) {
  const double f = factor[blockIdx.y];
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < elements;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t at = blockIdx.y * elements + i;
    out[at] = static_cast<T>(static_cast<float>(static_cast<double>(static_cast<float>(u[at])) * f));
  }
}

// What is done with a product's sums, unscaled:
//   kGram:   A = sum.
//   kPoly:   P = alpha sum + (beta + alpha (d[i] + d[j])) A', d A's diagonal and
//            A' A without it; on the diagonal alpha sum + (beta + alpha d) d.
//   kUpdate: X = sum + (alpha + d[i]) X, d P's diagonal; stored in fp32 and in
//            planes by rows and by columns.
//   kLast:   the same, stored as the result.
enum Kind { kGram, kPoly, kUpdate, kLast };

struct Finish {
  float alpha, beta;
  const int *row_exponents, *col_exponents;  // of X0: [batch][diagonals], [batch][width]
  Levels now, next;                          // of the step, and after it (kUpdate)
  Planes add;                                // kPoly: A
  const float* left;                         // [batch][diagonals]: d; not for kGram
  Planes to;                                 // by rows; not for kLast
  Planes across;                             // kUpdate: by columns
  float* x;                                  // kUpdate, kLast: X, [batch][diagonals][width]
  float* diagonal;                           // kGram, kPoly: [batch][diagonals], of the result
  int64_t diagonals, width;                  // padded extents
  void* out;                                 // kLast: the result, [rows][cols] of the update's type and shape
  int64_t rows, cols;
  bool tall;
};

// What a row or column of the result takes part with: the power of two that its
// sums are to be multiplied by, the scale of its planes, and its d.
struct Line {
  float sums, planes, left;
};
template <Kind kKind>
__device__ inline Line line_of(const Finish& f, int e, float left) {
  if constexpr (kKind == kGram) return {unscale_of(level_x(f.now, e)), scale_of(level_a(f.now, e)), 0.0f};
  if constexpr (kKind == kPoly) return {unscale_of(level_a(f.now, e)), scale_of(level_p(f.now, e)), left};
  return {unscale_of(level_p(f.now, e)), kKind == kUpdate ? scale_of(level_x(f.next, e)) : 0.0f, left};
}
template <Kind kKind>
__device__ inline Line row_of(const Finish& f, int64_t batch, int row) {
  const int64_t at = batch * f.diagonals + row;
  return line_of<kKind>(f, f.row_exponents[at], kKind == kGram ? 0.0f : f.left[at]);
}
template <Kind kKind>
__device__ inline Line column_of(const Finish& f, int64_t batch, int col) {
  if constexpr (kKind == kUpdate || kKind == kLast) {
    const int e = f.col_exponents[batch * f.width + col];
    return {unscale_of(level_x(f.now, e)), kKind == kUpdate ? scale_of(level_x(f.next, e)) : 0.0f, 0.0f};
  } else {
    return row_of<kKind>(f, batch, col);
  }
}

// Neighbouring columns of a row of X or A, as they are loaded: fours or eights.
template <Kind kKind, int kCols>
struct Addend {
  typedef half Halves __attribute__((ext_vector_type(kCols)));
  typedef float Floats __attribute__((ext_vector_type(kCols)));
  std::conditional_t<kKind == kUpdate || kKind == kLast, Floats, Halves> hi;
  Halves lo;
};

template <Kind kKind, bool kPair, int kCols>
__device__ inline Addend<kKind, kCols> load_addend(const Finish& f, int64_t batch, int row, int col) {
  typedef Addend<kKind, kCols> Add;
  Add a = {};
  if constexpr (kKind == kPoly) {
    const int64_t at = batch * f.add.size + row * f.add.ld + col;
    a.hi = *reinterpret_cast<const typename Add::Halves*>(f.add.hi + at);
    if constexpr (kPair) a.lo = *reinterpret_cast<const typename Add::Halves*>(f.add.lo + at);
  } else if constexpr (kKind != kGram) {
    a.hi = *reinterpret_cast<const typename Add::Floats*>(f.x + (batch * f.diagonals + row) * f.width + col);
  }
  return a;
}

template <typename T, Kind kKind, bool kPair, int kCols>
__device__ inline void finish(const Finish& f, const Addend<kKind, kCols>& a, const Line& r, const Line (&c)[kCols],
                              int64_t batch, int row, int col, float (&v)[kCols]) {
#pragma unroll
  for (int e = 0; e < kCols; ++e) {
    v[e] = v[e] * c[e].sums * r.sums;
    if constexpr (kKind == kPoly) {
      const bool on = row == col + e;
      const float x = on ? r.left : (static_cast<float>(a.hi[e]) + static_cast<float>(a.lo[e])) * r.sums;
      v[e] = f.alpha * v[e] + (f.beta + f.alpha * (on ? r.left : r.left + c[e].left)) * x;
    } else if constexpr (kKind != kGram) {
      v[e] += (f.alpha + r.left) * a.hi[e];
    }
  }
  if constexpr (kKind == kLast) {
    T* out = static_cast<T*>(f.out) + batch * f.rows * f.cols;
    if (!f.tall && col + kCols <= f.cols) {
      typedef T Values __attribute__((ext_vector_type(kCols), aligned(sizeof(T))));
      Values t;
#pragma unroll
      for (int e = 0; e < kCols; ++e) t[e] = static_cast<T>(v[e]);
      if (row < f.rows) *reinterpret_cast<Values*>(out + row * f.cols + col) = t;
    } else {
#pragma unroll
      for (int e = 0; e < kCols; ++e) {
        const int i = f.tall ? col + e : row, j = f.tall ? row : col + e;
        if (i < f.rows && j < f.cols) out[i * f.cols + j] = static_cast<T>(v[e]);
      }
    }
  } else {
    typedef typename Addend<kKind, kCols>::Halves Halves;
    Halves h, l;
    if constexpr (kKind == kUpdate) {
      typename Addend<kKind, kCols>::Floats x;
#pragma unroll
      for (int e = 0; e < kCols; ++e) {
        x[e] = v[e];
        h[e] = static_cast<half>(v[e] * c[e].planes);
        l[e] = static_cast<half>(v[e] * c[e].planes - static_cast<float>(h[e]));
      }
      *reinterpret_cast<decltype(x)*>(f.x + (batch * f.diagonals + row) * f.width + col) = x;
      const int64_t at = batch * f.across.size + row * f.across.ld + col;
      *reinterpret_cast<Halves*>(f.across.hi + at) = h;
      if constexpr (kPair) *reinterpret_cast<Halves*>(f.across.lo + at) = l;
    }
#pragma unroll
    for (int e = 0; e < kCols; ++e) {
      if constexpr (kKind != kUpdate)
        if (row == col + e) {
          f.diagonal[batch * f.diagonals + row] = v[e];
          v[e] = 0.0f;
        }
      h[e] = static_cast<half>(v[e] * r.planes);
      l[e] = static_cast<half>(v[e] * r.planes - static_cast<float>(h[e]));
    }
    const int64_t at = batch * f.to.size + row * f.to.ld + col;
    *reinterpret_cast<Halves*>(f.to.hi + at) = h;
    if constexpr (kPair) *reinterpret_cast<Halves*>(f.to.lo + at) = l;
  }
}

// Finishes a tile's sums, kCount eights at a time: all of a batch's addends are
// loaded before the first is used.
// kBothWays: where `twice`, also across the diagonal.
template <typename T, Kind kKind, bool kPair, int kCount, bool kBothWays = false, typename S>
__device__ inline void finish_tile(const Finish& f, const S& s, int64_t batch, int r0, int c0, int m, int n,
                                   bool twice = false) {
  Line c[S::kGroups][8];
#pragma unroll
  for (int g = 0; g < S::kGroups; ++g) {
    const int col = c0 + s.group_col(g);
#pragma unroll
    for (int e = 0; e < 8; ++e) c[g][e] = column_of<kKind>(f, batch, col < n ? col + e : 0);
  }
#pragma unroll
  for (int b = 0; b < S::kEights / kCount; ++b) {
    Addend<kKind, 8> a[kCount];
    Line r[kCount];
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      const int row = r0 + s.row(b * kCount + k), col = c0 + s.col(b * kCount + k);
      const bool in = row < m && col < n;
      a[k] = load_addend<kKind, kPair, 8>(f, batch, in ? row : 0, in ? col : 0);
      r[k] = row_of<kKind>(f, batch, row < m ? row : 0);
    }
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      const int at = b * kCount + k, row = r0 + s.row(at), col = c0 + s.col(at);
      const f32x4 x = s.four(at, 0), y = s.four(at, 1);
      float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      if (row >= m || col >= n) continue;
      finish<T, kKind, kPair, 8>(f, a[k], r[k], c[S::group(at)], batch, row, col, v);
      if constexpr (kBothWays)
        if (twice)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int64_t to = batch * f.to.size + (col + e) * f.to.ld + row;
            const float scaled = v[e] * c[S::group(at)][e].planes;
            const half h = static_cast<half>(scaled);
            f.to.hi[to] = h;
            if constexpr (kPair) f.to.lo[to] = static_cast<half>(scaled - static_cast<float>(h));
          }
    }
  }
}

// The product of `left` [m][depth] with `right`, [n][depth], or [depth][n]
// where kTurned; extents are padded ones.
struct Product {
  Planes left, right;
  int m, n, depth;
  int splits;      // parts of the depth, each a sum of its own
  float* sums;     // [splits][batch][m][n] where there are several
};

__device__ inline mma::Operand<half> operand(const Planes& p, int64_t batch, int first, int most, int rows, int depth,
                                             bool turned) {
  const int64_t at = batch * p.size + (turned ? first : first * p.ld);
  return {p.hi + at, p.lo == nullptr ? nullptr : p.lo + at, p.ld, rows - first < most ? rows - first : most, depth};
}

// A and its polynomial are symmetric: the tiles below the diagonal are summed
// and stored both ways.
template <typename T, Kind kKind, bool kPair>
__global__ __launch_bounds__(mma::kThreads, 2) void product_large(Product p, Finish f) {
  constexpr bool kTurned = kKind == kUpdate || kKind == kLast;
  __shared__ __align__(1024) char lds[mma::kLdsBytes];
  const unsigned down = (p.m + mma::kTile - 1) / mma::kTile, across = (p.n + mma::kTile - 1) / mma::kTile;
  const unsigned each = kTurned ? down * across : down * (down + 1) / 2;
  const unsigned block = mma::run_of_xcd(blockIdx.x, gridDim.x), batch = block / each;
  unsigned i, j;
  if constexpr (kTurned) {
    mma::place_tile(block - batch * each, down, across, i, j);
  } else {
    const unsigned n = block - batch * each;
    i = static_cast<unsigned>((sqrtf(8.0f * static_cast<float>(n) + 1.0f) - 1.0f) * 0.5f);
    while (i * (i + 1) / 2 > n) --i;
    while ((i + 1) * (i + 2) / 2 <= n) ++i;
    j = n - i * (i + 1) / 2;
  }
  const int r0 = i * mma::kTile, c0 = j * mma::kTile;
  mma::Sums s;
  mma::multiply_tile<half, false, kTurned, kPair ? 3 : 1>(
      operand(p.left, batch, r0, mma::kTile, p.m, p.depth, false),
      operand(p.right, batch, c0, mma::kTile, p.n, p.depth, kTurned), lds, s);
  s.place();
  finish_tile<T, kKind, kPair, 4, !kTurned>(f, s, batch, r0, c0, p.m, p.n, r0 != c0);
}

// Splits of a matrix are further apart than its tiles.
template <typename T, Kind kKind, bool kPair, int kSide>
__global__ __launch_bounds__(mma::kThreads128, kSide == 64 ? 2 : 1) void product_small(Product p, Finish f) {
  constexpr bool kTurned = kKind == kUpdate || kKind == kLast;
  typedef mma::Ring<half, false, kTurned, kPair, kSide, kSide> Tile;
  __shared__ __align__(1024) char lds[Tile::kLdsBytes];
  const unsigned down = (p.m + kSide - 1) / kSide, across = (p.n + kSide - 1) / kSide;
  const unsigned block = mma::run_of_xcd(blockIdx.x, gridDim.x), matrix = block / (down * across);
  const unsigned batch = p.splits == 1 ? matrix : matrix / p.splits, split = matrix - batch * p.splits;
  unsigned i, j;
  mma::place_tile(block - matrix * (down * across), down, across, i, j);
  const int r0 = i * kSide, c0 = j * kSide;
  const unsigned steps = p.depth / Tile::kDepth;
  typename Tile::Sums s;
  s.clear();
  Tile::add(operand(p.left, batch, r0, kSide, p.m, p.depth, false),
            operand(p.right, batch, c0, kSide, p.n, p.depth, kTurned), lds,
            p.splits == 1 ? 0 : static_cast<int>(steps * split / p.splits),
            p.splits == 1 ? static_cast<int>(steps) : static_cast<int>(steps * (split + 1) / p.splits), s);
  s.place();
  if (p.splits == 1) {
    finish_tile<T, kKind, kPair, s.kEights>(f, s, batch, r0, c0, p.m, p.n);
    return;
  }
  const int64_t batches = gridDim.x / (down * across * p.splits);
  float* to = p.sums + (split * batches + batch) * p.m * p.n;
#pragma unroll
  for (int k = 0; k < s.kEights; ++k) {
    const int row = r0 + s.row(k), col = c0 + s.col(k);
    if (row < p.m && col < p.n)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<f32x4*>(to + static_cast<int64_t>(row) * p.n + col + 4 * h) = s.four(k, h);
  }
}

// Adds the splits' sums in order and finishes them.
template <typename T, Kind kKind, bool kPair>
__global__ __launch_bounds__(kThreads) void finish_sums(Product p, Finish f, int64_t batches) {
  const int64_t fours = static_cast<int64_t>(p.m) * p.n / 4, n = fours * batches;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    // one matrix's sums are below 2^32
    const int64_t batch = batches == 1 ? 0 : i / fours;
    const unsigned e = static_cast<unsigned>(i - batch * fours) * 4, row = e / p.n, col = e - row * p.n;
    const Addend<kKind, 4> a = load_addend<kKind, kPair, 4>(f, batch, row, col);
    const Line r = row_of<kKind>(f, batch, row);
    Line c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = column_of<kKind>(f, batch, col + k);
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int64_t k = 0; k < p.splits; ++k) s += *reinterpret_cast<const f32x4*>(p.sums + (k * n + i) * 4);
    float v[4] = {s[0], s[1], s[2], s[3]};
    finish<T, kKind, kPair, 4>(f, a, r, c, batch, row, col, v);
  }
}

// A whole matrix in one work-group: no launch between the products.  X stays in
// registers in fp32, each element with the lane that sums it; its planes lie in
// LDS, by rows for A and then by columns for the update, in lines of np + 8
// elements, and A and its polynomial (in A's place) in lines of mp + 8: an odd
// number of 16-byte pieces, so that the same piece of neighbouring lines lies in
// different banks.  A wave sums blocks of 32 x 32.  What bounds it is the LDS
// reads of one CU (8 KB for 12 matrix instructions) and the barriers.
constexpr int kInnerThreads = 512;
constexpr int kInnerWaves = kInnerThreads / 64;
constexpr int kInnerSteps = 16;   // most steps
// Most blocks of a wave: 40 of 1024 sums, and 16 where little LDS leaves room
// for a second work-group on a CU.
constexpr int kInnerBlocks = 5, kInnerBlocksFew = 2;
constexpr int kInnerLds = 160 * 1024 - 2048, kInnerLdsFew = 40 * 1024;
constexpr int kInnerMost = 128;   // most padded rows: two square matrices in kInnerLds
constexpr int kInnerSquares = 2;  // most blocks of a wave of a square one

struct InnerArgs {
  int64_t rows, cols;
  int m, n, mp, np;  // extents and padded ones, multiples of 32
  bool tall;
  int steps;
  double eps;
  float a[kInnerSteps], b[kInnerSteps], c[kInnerSteps];
  Levels levels[kInnerSteps + 1];
};

__host__ __device__ constexpr int64_t inner_bytes(int64_t mp, int64_t np) {
  return 4 * mp * (np + 8) + 4 * mp * (mp + 8);
}

// Two planes of a matrix in LDS.
struct InnerPlanes {
  half* hi;
  half* lo;
  int ld;
};

// Fragment for 32 k from k0 of 16 lines from `first` (k along them).
__device__ inline u32x4 inner_along(const half* p, int ld, int first, int k0, int lane) {
  return *reinterpret_cast<const u32x4*>(p + (first + (lane & 15)) * ld + k0 + (lane >> 4) * 8);
}
// The same of 16 columns from `first` (k across lines).
__device__ inline u32x4 inner_across(const half* p, int ld, int first, int k0, int lane) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
  mma::u32x2 h[2];
#pragma unroll
  for (int m = 0; m < 2; ++m)
    h[m] = __builtin_bit_cast(
        mma::u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(
                        p + (k0 + (lane >> 4) * 8 + m * 4 + ((lane & 15) >> 2)) * ld + first + (lane & 3) * 4)));
  return __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3);
}

typedef f32x4 InnerBlock[2][2];

// The block at (i0, j0) of left times right (turned: k across right's lines).
// Each instruction's large products are added in fp32, rounded.
template <bool kTurned>
__device__ inline void inner_product(const InnerPlanes& left, const InnerPlanes& right, int i0, int j0, int depth,
                                     InnerBlock& s) {
  const int lane = mma::thread_here() & 63;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) s[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  InnerBlock low = {};
  for (int k0 = 0; k0 < depth; k0 += 32) {
    u32x4 l[2][2], r[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        l[i][q] = inner_along(q == 0 ? left.hi : left.lo, left.ld, i0 + 16 * i, k0, lane);
        const half* p = q == 0 ? right.hi : right.lo;
        r[i][q] = kTurned ? inner_across(p, right.ld, j0 + 16 * i, k0, lane)
                          : inner_along(p, right.ld, j0 + 16 * i, k0, lane);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        low[i][j] = mma::multiply<half>(r[j][1], l[i][0], low[i][j]);
        s[i][j] += mma::multiply<half>(r[j][0], l[i][0], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        low[i][j] = mma::multiply<half>(r[j][0], l[i][1], low[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) s[i][j] += low[i][j];
}

// f(four sums, row, column of the first) for the wave's blocks.
template <int kBlocks, typename F>
__device__ inline void inner_each(InnerBlock (&s)[kBlocks], int blocks, int across, F f) {
  const int thread = mma::thread_here(), lane = thread & 63, wave = thread >> 6;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int block = wave + b * kInnerWaves;
    if (block >= blocks) break;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f(s[b][i][j], block / across * 32 + i * 16 + (lane & 15), block % across * 32 + j * 16 + (lane >> 4) * 4);
  }
}

__device__ inline void inner_store(const InnerPlanes& p, int row, int col, f32x4 v) {
  f16x4 h, l;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = static_cast<half>(v[e]);
    l[e] = static_cast<half>(v[e] - static_cast<float>(h[e]));
  }
  *reinterpret_cast<f16x4*>(p.hi + row * p.ld + col) = h;
  *reinterpret_cast<f16x4*>(p.lo + row * p.ld + col) = l;
}
__device__ inline f32x4 inner_load(const InnerPlanes& p, int row, int col) {
  const f16x4 h = *reinterpret_cast<const f16x4*>(p.hi + row * p.ld + col);
  const f16x4 l = *reinterpret_cast<const f16x4*>(p.lo + row * p.ld + col);
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(h[e]) + static_cast<float>(l[e]);
  return v;
}

// The largest of 16 neighbouring lanes' values: neighbours, pairs, and the
// halves of 8 and of 16 mirrored.
__device__ inline float largest_of_16(float v) {
  auto other = [&](auto control) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), decltype(control)::value, 0xf, 0xf, true));
  };
  v = fmaxf(v, other(std::integral_constant<int, 0xb1>()));
  v = fmaxf(v, other(std::integral_constant<int, 0x4e>()));
  v = fmaxf(v, other(std::integral_constant<int, 0x141>()));
  return fmaxf(v, other(std::integral_constant<int, 0x140>()));
}

// Exponents of four neighbouring lines, from `first`, a multiple of four.
struct InnerFour {
  int e[4];
  __device__ inline InnerFour(const signed char* exponents, int first) {
    const int four = *reinterpret_cast<const int*>(exponents + first);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = four << (24 - 8 * i) >> 24;
  }
};

// (The result may be the update: a work-group reads its matrix before it writes
// it.)
template <typename T, int kLds, int kBlocks>
__global__ __launch_bounds__(kInnerThreads) void orthogonalize_inner(InnerArgs a, const T* update, T* result) {
  __shared__ __align__(16) char lds[kLds];
  __shared__ double waves[kInnerWaves];
  __shared__ __align__(16) float diagonal[kInnerMost];  // of A, then of its polynomial, whose planes hold zeros there
  __shared__ __align__(4) signed char row_exponents[kInnerMost], col_exponents[kBlocks * kInnerWaves * 32];
  const int64_t elements = a.rows * a.cols;
  const T* u = update + blockIdx.x * elements;
  T* out = result + blockIdx.x * elements;
  const int cols = static_cast<int>(a.cols), lx = a.np + 8, la = a.mp + 8;
  half* p = reinterpret_cast<half*>(lds);
  const InnerPlanes planes{p, p + a.mp * lx, lx}, gram{p + 2 * a.mp * lx, p + 2 * a.mp * lx + a.mp * la, la};
  const int thread = threadIdx.x, lane = thread & 63;
  const int square = a.mp / 32 * (a.mp / 32), wide = a.mp / 32 * (a.np / 32);
  InnerBlock x[kBlocks], s[kInnerSquares];

  // The update, the sum of its squares, and the largest magnitudes of X's rows
  // and columns (as integers: the order does not matter), where the planes will
  // lie.
  unsigned* row_most = reinterpret_cast<unsigned*>(lds);
  unsigned* col_most = row_most + a.mp;
  for (int i = thread; i < a.mp + a.np; i += kInnerThreads) row_most[i] = 0;
  __syncthreads();
  double squares = 0.0;
  inner_each(x, wide, a.np / 32, [&](f32x4& v, int row, int col) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = row < a.m && col + e < a.n;
      const float loaded = static_cast<float>(u[in ? (a.tall ? (col + e) * cols + row : row * cols + col + e) : 0]);
      v[e] = in ? loaded : 0.0f;
    }
  });
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int block = (thread >> 6) + b * kInnerWaves, across = a.np / 32;
    if (block >= wide) break;
    float row[2] = {}, col[2][4] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = x[b][i][j][e];
          squares += static_cast<double>(v) * static_cast<double>(v);
          row[i] = fmaxf(row[i], fabsf(v));
          col[j][e] = fmaxf(col[j][e], fabsf(v));
        }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int d = 16; d < 64; d <<= 1) row[i] = fmaxf(row[i], __shfl_xor(row[i], d));
      if (lane < 16) atomicMax(row_most + block / across * 32 + i * 16 + lane, __builtin_bit_cast(unsigned, row[i]));
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float most = largest_of_16(col[j][e]);
        if ((lane & 15) == 0)
          atomicMax(col_most + block % across * 32 + j * 16 + (lane >> 4) * 4 + e, __builtin_bit_cast(unsigned, most));
      }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) squares += __shfl_xor(squares, d);
  if (lane == 0) waves[thread >> 6] = squares;
  __syncthreads();
  squares = 0.0;
#pragma unroll
  for (int w = 0; w < kInnerWaves; ++w) squares += waves[w];
  const double factor = 1.0 / (sqrt(squares) + a.eps);
  for (int i = thread; i < a.mp + a.np; i += kInnerThreads) {
    const int e = exponent_of(__builtin_bit_cast(float, row_most[i]) * factor, i < a.mp ? a.n : a.m);
    (i < a.mp ? row_exponents : col_exponents - a.mp)[i] = static_cast<signed char>(e);
  }
  inner_each(x, wide, a.np / 32, [&](f32x4& v, int, int) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(static_cast<double>(v[e]) * factor);
  });
  __syncthreads();

  auto store_by_row = [&](const Levels& l) {
    inner_each(x, wide, a.np / 32, [&](f32x4& v, int row, int col) {
      inner_store(planes, row, col, v * scale_of(level_x(l, row_exponents[row])));
    });
  };
  auto store_by_col = [&](const Levels& l) {
    inner_each(x, wide, a.np / 32, [&](f32x4& v, int row, int col) {
      const InnerFour at(col_exponents, col);
      f32x4 scaled;
#pragma unroll
      for (int e = 0; e < 4; ++e) scaled[e] = v[e] * scale_of(level_x(l, at.e[e]));
      inner_store(planes, row, col, scaled);
    });
  };
  // A or P, scaled by `scale`.
  auto store_square = [&](f32x4 v, int row, int col, float scale) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (row == col + e) {
        diagonal[row] = v[e];
        v[e] = 0.0f;
      }
    inner_store(gram, row, col, v * scale);
  };
  auto multiply_square = [&](const InnerPlanes& factor, int depth) {
    const int wave = mma::thread_here() >> 6, across = a.mp / 32;
#pragma unroll
    for (int b = 0; b < kInnerSquares; ++b) {
      const int block = wave + b * kInnerWaves;
      if (block >= square) break;
      inner_product<false>(factor, factor, block / across * 32, block % across * 32, depth, s[b]);
    }
  };
  store_by_row(a.levels[0]);
  __syncthreads();
  for (int t = 0; t < a.steps; ++t) {
    const Levels l = a.levels[t];
    multiply_square(planes, a.np);
    inner_each(s, square, a.mp / 32, [&](f32x4& v, int row, int col) {
      const int at = row_exponents[row];
      const InnerFour across(row_exponents, col);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = v[e] * unscale_of(level_x(l, across.e[e])) * unscale_of(level_x(l, at));
      store_square(v, row, col, scale_of(level_a(l, at)));
    });
    __syncthreads();  // X by rows has been read, too
    store_by_col(l);
    multiply_square(gram, a.mp);
    inner_each(s, square, a.mp / 32, [&](f32x4& v, int row, int col) {
      const f32x4 held = inner_load(gram, row, col), above = *reinterpret_cast<const f32x4*>(diagonal + col);
      const InnerFour across(row_exponents, col);
      const float left = diagonal[row], unscale = unscale_of(level_a(l, row_exponents[row]));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool on = row == col + e;
        const float w = a.b[t] + a.c[t] * (on ? left : left + above[e]);
        v[e] = a.c[t] * (v[e] * unscale_of(level_a(l, across.e[e])) * unscale) + w * (on ? left : held[e] * unscale);
      }
    });
    __syncthreads();  // all of A has been read
    inner_each(s, square, a.mp / 32, [&](f32x4& v, int row, int col) {
      store_square(v, row, col, scale_of(level_p(l, row_exponents[row])));
    });
    __syncthreads();
    const int thread_now = mma::thread_here(), wave = thread_now >> 6;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int block = wave + b * kInnerWaves;
      if (block >= wide) break;
      InnerBlock sum;
      inner_product<true>(gram, planes, block / (a.np / 32) * 32, block % (a.np / 32) * 32, a.mp, sum);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = block / (a.np / 32) * 32 + i * 16 + (thread_now & 15);
        const float unscale = unscale_of(level_p(l, row_exponents[row])), own = a.a[t] + diagonal[row];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const InnerFour at(col_exponents, block % (a.np / 32) * 32 + j * 16 + (thread_now >> 4 & 3) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[b][i][j][e] = sum[i][j][e] * unscale_of(level_x(l, at.e[e])) * unscale + own * x[b][i][j][e];
        }
      }
    }
    if (t + 1 == a.steps) break;
    __syncthreads();  // all of X has been read
    store_by_row(a.levels[t + 1]);
    __syncthreads();
  }
  inner_each(x, wide, a.np / 32, [&](f32x4& v, int row, int col) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (row < a.m && col + e < a.n) out[a.tall ? (col + e) * cols + row : row * cols + col + e] = static_cast<T>(v[e]);
  });
}

// Offsets inside a tile, and pieces of an operand, are counted in 32 bits.
constexpr int64_t kMostExtent = int64_t(1) << 22;

spmm_status check_desc(const spmm_orthogonalize_desc* d) {
  if (d == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null descriptor");
  if (!dense_type(d->value_type))
    return fail(SPMM_ERR_CONTRACT, "orthogonalize supports only FP16, BF16 and FP32 tensors");
  if (d->batch < 0 || d->rows < 0 || d->width < 0) return fail(SPMM_ERR_CONTRACT, "orthogonalize: negative extent");
  if (d->batch > 65535 || d->rows >= kMostExtent || d->width >= kMostExtent)
    return fail(SPMM_ERR_CONTRACT, "orthogonalize takes at most 65535 matrices with extents below 2^22");
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

// The least e with v < 2^e.
int exponent_above(double v) {
  if (!(v > 0.0)) return kLeast;
  if (std::isinf(v)) return kMost;
  int e;
  std::frexp(v, &e);
  return clamped(e);
}

// What the coefficients bound, step after step.
struct Bounds {
  double growth = 1.0, bound = 1.0;  // of X's rows and columns against X0's; of X's largest singular value

  // Of a step with the coefficients c.
  Levels levels(const double* c) const {
    const double high = std::fmax(std::fabs(c[1]), std::fabs(c[1] + c[2] * bound * bound));
    return {exponent_above(growth), exponent_above(bound), exponent_above(high)};
  }
  // After it.
  Levels step(const double* c) {
    const double t = bound * bound, turn = c[2] != 0.0 ? -c[1] / (2 * c[2]) : -1.0;
    // largest |a + b t + c t^2| on [0, bound^2]
    double grown = std::fmax(std::fabs(c[0]), std::fabs(c[0] + t * (c[1] + t * c[2])));
    if (turn > 0.0 && turn < t) grown = std::fmax(grown, std::fabs(c[0] + turn * (c[1] + turn * c[2])));
    growth = std::fmin(growth * grown, 1e300);
    bound = std::fmin(largest(c[0], c[1], c[2], bound), 1e60);
    return {exponent_above(growth), exponent_above(bound), kLeast};
  }
};

// How a product of smaller tiles is run: the tile's side and the parts of its
// depth.
struct Plan {
  int64_t side, splits;
};

// The plan that takes the least time by this count, in microseconds: a round of
// tiles takes 3 and its steps, 0.27 each, or where work-groups share a CU what
// each takes of it (128: 0.2, 64: 0.11; pairs 1.8 times that) if that is more;
// sums of parts cost a launch, 5, and 8 bytes each at 4 TB/s.  Measured on 12
// matrices of 512 x 512 x 1024: 14.8 us with 128, 17.0 with 64.
Plan plan_for(int64_t batch, int64_t rows, int64_t cols, int64_t depth, bool pair) {
  Plan best{64, 1};
  double least = 1e300;
  const int64_t steps = ceil_div(depth, 32);
  for (const int64_t side : {64, 128}) {
    const int64_t on_cu = side == 64 ? (pair ? 2 : 4) : (pair ? 1 : 2);
    const int64_t tiles = batch * ceil_div(rows, side) * ceil_div(cols, side);
    const double share = (side == 128 ? 0.2 : 0.11) * (pair ? 1.8 : 1.0);
    for (int64_t k = 1; k == 1 || (k <= 2 * kCus / tiles && 4 * k <= steps); ++k) {
      const int64_t each = ceil_div(steps, k), groups = tiles * k, rounds = ceil_div(groups, kCus * on_cu);
      const double beside = static_cast<double>(std::min(on_cu, ceil_div(groups, kCus)));
      const double time = static_cast<double>(rounds) * (3.0 + static_cast<double>(each) * std::fmax(0.27, beside * share)) +
                          (k > 1 ? 5.0 + static_cast<double>(k * batch * rows * cols) * 8.0 / 4e6 : 0.0);
      if (time < least) {
        least = time;
        best = {side, k};
      }
    }
  }
  return best;
}

// X in fp32, in planes by rows, and by columns twice (a step reads one and
// writes the other), A and P in planes, their diagonals, the exponents, what the
// first pass finds, and the sums of split products.
// m <= n: the matrix's extents, mp and np padded.
struct Layout {
  int64_t m, n, mp, np;
  int64_t down, across;  // tiles of the first pass
  bool pair;             // three products of planes; else one
  size_t x, gram, diagonal, row_exponents, col_exponents, factor, row_most, col_most, squares, sums;
  explicit Layout(const spmm_orthogonalize_desc* d) {
    m = d->rows < d->width ? d->rows : d->width;
    n = d->rows < d->width ? d->width : d->rows;
    mp = align_up(m, 64);
    np = align_up(n, 64);
    pair = d->value_type != SPMM_VALUE_BF16 || m < 128 || d->precise != 0;
    x = align_up(static_cast<size_t>(d->batch * mp * np) * sizeof(half), 256);
    gram = align_up(static_cast<size_t>(d->batch * mp * mp) * sizeof(half), 256);
    diagonal = align_up(static_cast<size_t>(d->batch * mp) * sizeof(float), 256);
    row_exponents = align_up(static_cast<size_t>(d->batch * mp) * sizeof(int), 256);
    col_exponents = align_up(static_cast<size_t>(d->batch * np) * sizeof(int), 256);
    factor = align_up(static_cast<size_t>(d->batch) * sizeof(double), 256);
    down = ceil_div(d->rows, kMeasureRows);
    across = ceil_div(d->width, d->value_type == SPMM_VALUE_F32 ? kMeasureCols<float> : kMeasureCols<half>);
    row_most = align_up(static_cast<size_t>(d->batch * d->rows * across) * sizeof(float), 256);
    col_most = align_up(static_cast<size_t>(d->batch * down * d->width) * sizeof(float), 256);
    squares = align_up(static_cast<size_t>(d->batch * down * across) * sizeof(double), 256);
    sums = 0;
    for (const bool wide : {false, true}) {
      const int64_t cols = wide ? np : mp, depth = wide ? mp : np, k = splits(d->batch, mp, cols, depth, pair);
      const size_t bytes = k > 1 ? static_cast<size_t>(k * d->batch * mp * cols) * sizeof(float) : 0;
      sums = sums > bytes ? sums : bytes;
    }
  }
  size_t total() const {
    const size_t planes = pair ? 2 : 1;
    return 2 * x + planes * (3 * x + 2 * gram) + 2 * diagonal + row_exponents + col_exponents + factor + row_most +
           col_most + squares + sums;
  }

  // The large tile where three quarters of the CUs get one, and fill it.
  static bool large(int64_t batch, int64_t rows, int64_t cols) {
    return rows > 128 && cols > 128 && batch * ceil_div(rows, mma::kTile) * ceil_div(cols, mma::kTile) >= kCus * 3 / 4;
  }
  static int64_t splits(int64_t batch, int64_t rows, int64_t cols, int64_t depth, bool pair) {
    if (batch == 0 || rows == 0 || cols == 0 || large(batch, rows, cols)) return 1;
    return plan_for(batch, rows, cols, depth, pair).splits;
  }
};

template <typename T, Kind kKind, bool kPair>
spmm_status multiply(Product p, const Finish& f, int64_t batch, hipStream_t s) {
  if (Layout::large(batch, p.m, p.n)) {
    const int64_t down = ceil_div(p.m, mma::kTile), across = ceil_div(p.n, mma::kTile);
    const bool turned = kKind == kUpdate || kKind == kLast;
    const unsigned tiles = static_cast<unsigned>((turned ? down * across : down * (down + 1) / 2) * batch);
    hipLaunchKernelGGL((product_large<T, kKind, kPair>), dim3(tiles), dim3(mma::kThreads), 0, s, p, f);
    return check_launch("orthogonalize product");
  }
  const Plan plan = plan_for(batch, p.m, p.n, p.depth, kPair);
  p.splits = static_cast<int>(plan.splits);
  const dim3 tiles(static_cast<unsigned>(ceil_div(p.m, plan.side) * ceil_div(p.n, plan.side) * batch * p.splits));
  const dim3 threads(mma::kThreads128);
  if (plan.side == 128)
    hipLaunchKernelGGL((product_small<T, kKind, kPair, 128>), tiles, threads, 0, s, p, f);
  else
    hipLaunchKernelGGL((product_small<T, kKind, kPair, 64>), tiles, threads, 0, s, p, f);
  if (spmm_status st = check_launch("orthogonalize product")) return st;
  if (p.splits == 1) return SPMM_OK;
  const int64_t blocks = ceil_div(static_cast<int64_t>(p.m) * p.n / 4 * batch, kThreads);
  hipLaunchKernelGGL((finish_sums<T, kKind, kPair>), dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)),
                     dim3(kThreads), 0, s, p, f, batch);
  return check_launch("orthogonalize sums");
}

// The update's type matters to the last product alone.
template <typename T, Kind kKind>
spmm_status multiply(const Product& p, const Finish& f, int64_t batch, bool pair, hipStream_t s) {
  if constexpr (kKind != kLast)
    return pair ? multiply<half, kKind, true>(p, f, batch, s) : multiply<half, kKind, false>(p, f, batch, s);
  else if constexpr (std::is_same_v<T, __bf16>)
    return pair ? multiply<T, kKind, true>(p, f, batch, s) : multiply<T, kKind, false>(p, f, batch, s);
  else
    return multiply<T, kKind, true>(p, f, batch, s);
}

// Whether a matrix and its Gram matrix fit a work-group's LDS.
bool inner_fits(const spmm_orthogonalize_desc* d) {
  const int64_t m = d->rows < d->width ? d->rows : d->width, n = d->rows < d->width ? d->width : d->rows;
  if (n > 4096 || d->steps < 1 || d->steps > kInnerSteps) return false;
  const int64_t mp = align_up(m, 32), np = align_up(n, 32);
  return inner_bytes(mp, np) <= kInnerLds && mp / 32 * (np / 32) <= kInnerBlocks * kInnerWaves;
}

template <typename T>
spmm_status run_inner(const spmm_orthogonalize_desc* d, const void* update, void* out, hipStream_t s) {
  InnerArgs a{};
  a.rows = d->rows;
  a.cols = d->width;
  a.tall = d->rows > d->width;
  a.m = static_cast<int>(a.tall ? d->width : d->rows);
  a.n = static_cast<int>(a.tall ? d->rows : d->width);
  a.mp = static_cast<int>(align_up(a.m, 32));
  a.np = static_cast<int>(align_up(a.n, 32));
  a.steps = static_cast<int>(d->steps);
  a.eps = d->eps;
  Bounds bounds;
  for (int i = 0; i < a.steps; ++i) {
    const double* c = d->coefficients + 3 * i;
    a.a[i] = static_cast<float>(c[0]);
    a.b[i] = static_cast<float>(c[1]);
    a.c[i] = static_cast<float>(c[2]);
    a.levels[i] = bounds.levels(c);
    a.levels[i + 1] = bounds.step(c);
  }
  const dim3 grid(static_cast<unsigned>(d->batch)), block(kInnerThreads);
  const T* u = static_cast<const T*>(update);
  if (inner_bytes(a.mp, a.np) <= kInnerLdsFew && a.mp / 32 * (a.np / 32) <= kInnerBlocksFew * kInnerWaves)
    hipLaunchKernelGGL((orthogonalize_inner<T, kInnerLdsFew, kInnerBlocksFew>), grid, block, 0, s, a, u,
                       static_cast<T*>(out));
  else
    hipLaunchKernelGGL((orthogonalize_inner<T, kInnerLds, kInnerBlocks>), grid, block, 0, s, a, u, static_cast<T*>(out));
  return check_launch("orthogonalize");
}

template <typename T>
spmm_status run(const spmm_orthogonalize_desc* d, const Layout& l, const void* update, void* out, char* ws,
                hipStream_t s) {
  const bool tall = d->rows > d->width;
  const int mp = static_cast<int>(l.mp), np = static_cast<int>(l.np);
  auto take = [&](size_t bytes) {
    char* p = ws;
    ws += bytes;
    return p;
  };
  auto planes = [&](size_t bytes, int64_t ld) {
    half* hi = reinterpret_cast<half*>(take(bytes));
    half* lo = l.pair ? reinterpret_cast<half*>(take(bytes)) : nullptr;
    return Planes{hi, lo, ld, l.mp * ld};
  };
  float* x = reinterpret_cast<float*>(take(2 * l.x));
  const Planes by_row = planes(l.x, l.np);
  Planes by_col = planes(l.x, l.np), by_col_next = planes(l.x, l.np);
  const Planes gram = planes(l.gram, l.mp), poly = planes(l.gram, l.mp);
  float* gram_diagonal = reinterpret_cast<float*>(take(l.diagonal));
  float* poly_diagonal = reinterpret_cast<float*>(take(l.diagonal));
  Exponents e;
  e.rows = reinterpret_cast<int*>(take(l.row_exponents));
  e.cols = reinterpret_cast<int*>(take(l.col_exponents));
  e.factor = reinterpret_cast<double*>(take(l.factor));
  Measures w;
  w.rows = reinterpret_cast<float*>(take(l.row_most));
  w.cols = reinterpret_cast<float*>(take(l.col_most));
  w.sums = reinterpret_cast<double*>(take(l.squares));
  float* sums = reinterpret_cast<float*>(ws);
  const T* u = static_cast<const T*>(update);
  const unsigned batch = static_cast<unsigned>(d->batch);
  Bounds bounds;
  hipLaunchKernelGGL(measure_update<T>, dim3(static_cast<unsigned>(l.down * l.across), batch), dim3(kThreads), 0, s, u,
                     d->rows, d->width, w);
  const int64_t rows_padded = tall ? l.np : l.mp, cols_padded = tall ? l.mp : l.np;
  hipLaunchKernelGGL(update_exponents,
                     dim3(static_cast<unsigned>(ceil_div(rows_padded, kThreads / 64) + ceil_div(cols_padded, 64)), batch),
                     dim3(kThreads), 0, s, w, d->rows, d->width, l.down, l.across, tall, d->eps, rows_padded,
                     cols_padded, e);
  if (spmm_status st = check_launch("orthogonalize measure")) return st;
  if (d->steps == 0) {
    const int64_t blocks = ceil_div(l.m * l.n, kThreads);
    hipLaunchKernelGGL(store_scaled<T>, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096), batch), dim3(kThreads), 0,
                       s, u, l.m * l.n, e.factor, static_cast<T*>(out));
    return check_launch("orthogonalize result");
  }
  hipLaunchKernelGGL(scale_update<T>, dim3(static_cast<unsigned>(l.np / 64), static_cast<unsigned>(l.mp / 64), batch),
                     dim3(kThreads), 0, s, u, d->rows, d->width, tall, e,
                     bounds.levels(d->coefficients), l.mp, l.np, x, by_row, by_col);
  if (spmm_status st = check_launch("orthogonalize scale")) return st;
  Finish f{};
  f.row_exponents = e.rows;
  f.col_exponents = e.cols;
  f.x = x;
  f.diagonals = l.mp;
  f.width = l.np;
  f.out = out;
  f.rows = d->rows;
  f.cols = d->width;
  f.tall = tall;
  for (int64_t i = 0; i < d->steps; ++i) {
    const double* c = d->coefficients + 3 * i;
    f.now = bounds.levels(c);
    f.next = bounds.step(c);
    f.to = gram;
    f.diagonal = gram_diagonal;
    if (spmm_status st = multiply<T, kGram>({by_row, by_row, mp, mp, np, 1, sums}, f, d->batch, l.pair, s)) return st;
    f.alpha = static_cast<float>(c[2]);
    f.beta = static_cast<float>(c[1]);
    f.add = gram;
    f.left = gram_diagonal;
    f.to = poly;
    f.diagonal = poly_diagonal;
    if (spmm_status st = multiply<T, kPoly>({gram, gram, mp, mp, mp, 1, sums}, f, d->batch, l.pair, s)) return st;
    f.alpha = static_cast<float>(c[0]);
    f.left = poly_diagonal;
    f.to = by_row;
    f.across = by_col_next;
    const Product p{poly, by_col, mp, np, mp, 1, sums};
    if (spmm_status st = i + 1 < d->steps ? multiply<T, kUpdate>(p, f, d->batch, l.pair, s)
                                          : multiply<T, kLast>(p, f, d->batch, l.pair, s))
      return st;
    std::swap(by_col, by_col_next);
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
  *bytes = inner_fits(d) ? 0 : Layout(d).total();
  return SPMM_OK;
}

spmm_status spmm_orthogonalize_run(const spmm_orthogonalize_desc* d, const void* update, void* out, void* workspace,
                                   size_t workspace_bytes, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_desc(d)) return st;
  if (d->batch == 0 || d->rows == 0 || d->width == 0) return SPMM_OK;
  if (update == nullptr || out == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "orthogonalize: null device pointer");
  hipStream_t s = as_stream(stream);
  if (inner_fits(d)) switch (d->value_type) {
      case SPMM_VALUE_F16: return run_inner<_Float16>(d, update, out, s);
      case SPMM_VALUE_BF16: return run_inner<__bf16>(d, update, out, s);
      default: return run_inner<float>(d, update, out, s);
    }
  const Layout l(d);
  if (workspace == nullptr || workspace_bytes < l.total())
    return fail(SPMM_ERR_CONTRACT, "orthogonalize: workspace too small: need " + std::to_string(l.total()) + " bytes");
  if (ceil_div(l.mp, 64) * ceil_div(l.np, 64) * d->batch > INT32_MAX / 64 || l.mp * l.np >= (int64_t(1) << 32))
    return fail(SPMM_ERR_OVERFLOW, "orthogonalize: too many tiles for one launch");
  char* ws = static_cast<char*>(workspace);
  switch (d->value_type) {
    case SPMM_VALUE_F16: return run<_Float16>(d, l, update, out, ws, s);
    case SPMM_VALUE_BF16: return run<__bf16>(d, l, update, out, ws, s);
    default: return run<float>(d, l, update, out, ws, s);
  }
}

}  // extern "C"
