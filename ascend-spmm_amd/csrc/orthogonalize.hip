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
// The diagonals of A and P, where most of these matrices lies, are carried in
// fp32 and are zeros in the planes: with D the diagonal, A A is taken as A' A' +
// D A' + A' D + D D, and P X as P' X + D X.  Matrix instructions cut their sums
// to fp32 (they do not round), always to the same side; without the large
// terms, and with products of low planes summed apart, little is lost.
//
// A bf16 update is rounded to 8 bits at the end, so its factors need fewer: one
// product of high planes, of 11 bits.  X keeps its low plane for a X, so that
// weak directions, which the steps raise most, are not lost beside strong ones.
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
constexpr int kNormParts = 512;  // work-groups that add up one matrix's squares
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
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kNormParts / 64; ++i) s += parts[i * 64 + (threadIdx.x & 63)];
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
// d[i]) * E(i, j), E the planes `add`; stored as planes or as the result.  d is
// the left factor's diagonal, which its planes hold as zeros: the polynomial's
// for the update of X; A's for the polynomial, where it counts on both sides.
enum Kind { kGram, kPoly, kUpdate, kLast };

struct Finish {
  float alpha, beta;
  Planes add;           // not for kGram
  const float* left;    // [batch][diagonals]: d; not for kGram
  Planes to;            // not for kLast
  float* diagonal;      // [batch][diagonals]: of the result of kGram and kPoly
  int64_t diagonals;
  void* out;            // kLast: the result, [rows][cols] of the update's type and shape
  int64_t rows, cols;
  bool tall;
};

// Neighbouring columns of a row of E, as they are loaded: fours or eights.
template <int kCols>
struct Addend {
  typedef half Halves __attribute__((ext_vector_type(kCols)));
  Halves hi, lo;
  float left, across[kCols];
};

template <Kind kKind, bool kPair, int kCols>
__device__ inline Addend<kCols> load_addend(const Finish& f, int64_t batch, int row, int col) {
  typedef typename Addend<kCols>::Halves Halves;
  Addend<kCols> a = {};
  if constexpr (kKind != kGram) {
    const int64_t at = batch * f.add.size + row * f.add.ld + col;
    a.hi = *reinterpret_cast<const Halves*>(f.add.hi + at);
    if constexpr (kPair || kKind != kPoly) a.lo = *reinterpret_cast<const Halves*>(f.add.lo + at);
    a.left = f.left[batch * f.diagonals + row];
    if constexpr (kKind == kPoly)
#pragma unroll
      for (int e = 0; e < kCols; ++e) a.across[e] = f.left[batch * f.diagonals + col + e];
  }
  return a;
}

template <typename T, Kind kKind, bool kPair, int kCols>
__device__ inline void finish(const Finish& f, const Addend<kCols>& a, int64_t batch, int row, int col,
                              float (&v)[kCols]) {
#pragma unroll
  for (int e = 0; e < kCols; ++e) v[e] *= f.alpha;
  if constexpr (kKind != kGram)
#pragma unroll
    for (int e = 0; e < kCols; ++e) {
      float x = static_cast<float>(a.hi[e]) + static_cast<float>(a.lo[e]);
      float w = f.beta + f.alpha * a.left;
      if constexpr (kKind == kPoly) {
        if (row == col + e) x = a.left;
        else w += f.alpha * a.across[e];
      }
      v[e] += w * x;
    }
  if constexpr (kKind == kLast) {
    T* out = static_cast<T*>(f.out) + batch * f.rows * f.cols;
    if (!f.tall && col + kCols <= f.cols) {
      typedef T Values __attribute__((ext_vector_type(kCols), aligned(sizeof(T))));
      Values r;
#pragma unroll
      for (int e = 0; e < kCols; ++e) r[e] = static_cast<T>(v[e]);
      if (row < f.rows) *reinterpret_cast<Values*>(out + row * f.cols + col) = r;
    } else {
#pragma unroll
      for (int e = 0; e < kCols; ++e) {
        const int i = f.tall ? col + e : row, j = f.tall ? row : col + e;
        if (i < f.rows && j < f.cols) out[i * f.cols + j] = static_cast<T>(v[e]);
      }
    }
  } else {
    typename Addend<kCols>::Halves h, l;
#pragma unroll
    for (int e = 0; e < kCols; ++e) {
      if constexpr (kKind != kUpdate)
        if (row == col + e) {
          f.diagonal[batch * f.diagonals + row] = v[e];
          v[e] = 0.0f;
        }
      h[e] = static_cast<half>(v[e]);
      l[e] = static_cast<half>(v[e] - static_cast<float>(h[e]));
    }
    const int64_t at = batch * f.to.size + row * f.to.ld + col;
    *reinterpret_cast<decltype(h)*>(f.to.hi + at) = h;
    if constexpr (kPair || kKind == kUpdate) *reinterpret_cast<decltype(h)*>(f.to.lo + at) = l;
  }
}

// Finishes a tile's sums, kCount eights at a time: all of a batch's addends are
// loaded before the first is used.
// kBothWays: where `twice`, also across the diagonal.
template <typename T, Kind kKind, bool kPair, int kCount, bool kBothWays = false, typename S>
__device__ inline void finish_tile(const Finish& f, const S& s, int64_t batch, int r0, int c0, int m, int n,
                                   bool twice = false) {
#pragma unroll
  for (int b = 0; b < S::kEights / kCount; ++b) {
    Addend<8> a[kCount];
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      const int row = r0 + s.row(b * kCount + k), col = c0 + s.col(b * kCount + k);
      const bool in = row < m && col < n;
      a[k] = load_addend<kKind, kPair, 8>(f, batch, in ? row : 0, in ? col : 0);
    }
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      const int row = r0 + s.row(b * kCount + k), col = c0 + s.col(b * kCount + k);
      const f32x4 x = s.four(b * kCount + k, 0), y = s.four(b * kCount + k, 1);
      float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      if (row >= m || col >= n) continue;
      finish<T, kKind, kPair, 8>(f, a[k], batch, row, col, v);
      if constexpr (kBothWays)
        if (twice)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int64_t at = batch * f.to.size + (col + e) * f.to.ld + row;
            const half h = static_cast<half>(v[e]);
            f.to.hi[at] = h;
            if constexpr (kPair) f.to.lo[at] = static_cast<half>(v[e] - static_cast<float>(h));
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
  finish_tile<T, kKind, kPair, 8, !kTurned>(f, s, batch, r0, c0, p.m, p.n, r0 != c0);
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
    const Addend<4> a = load_addend<kKind, kPair, 4>(f, batch, row, col);
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int64_t k = 0; k < p.splits; ++k) s += *reinterpret_cast<const f32x4*>(p.sums + (k * n + i) * 4);
    float v[4] = {s[0], s[1], s[2], s[3]};
    finish<T, kKind, kPair, 4>(f, a, batch, row, col, v);
  }
}

// X0 itself (no steps): the planes' sum, unscaled.
template <typename T>
__global__ __launch_bounds__(kThreads) void store_planes(Finish f, int64_t mp, int64_t batches) {
  const int64_t fours = mp * f.add.ld / 4;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < fours * batches;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t batch = i / fours, row = i % fours * 4 / f.add.ld, col = i % fours * 4 % f.add.ld;
    float v[4] = {};
    Addend<4> a = {};  // without a left factor
    a.hi = *reinterpret_cast<const f16x4*>(f.add.hi + batch * f.add.size + row * f.add.ld + col);
    a.lo = *reinterpret_cast<const f16x4*>(f.add.lo + batch * f.add.size + row * f.add.ld + col);
    finish<T, kLast, true, 4>(f, a, batch, row, col, v);
  }
}

// A whole matrix in one work-group, its planes in LDS: no launch between the
// products.  X lies in lines of np + 8 elements, A and its polynomial (in A's
// place) in lines of mp + 8: an odd number of 16-byte pieces, so that the same
// piece of neighbouring lines lies in different banks.  A wave sums blocks of
// 32 x 32.  What bounds it is the LDS reads of one CU (8 KB for 12 matrix
// instructions) and the barriers.
constexpr int kInnerThreads = 512;
constexpr int kInnerWaves = kInnerThreads / 64;
constexpr int kInnerSteps = 16;   // most steps
// Most blocks of a wave: 40 of 1024 sums, and 16 where little LDS leaves room
// for a second work-group on a CU.
constexpr int kInnerBlocks = 5, kInnerBlocksFew = 2;
constexpr int kInnerLds = 160 * 1024 - 1024, kInnerLdsFew = 40 * 1024;
constexpr int kInnerMost = 128;  // most padded rows: two square matrices in kInnerLds

struct InnerArgs {
  int64_t rows, cols;
  int m, n, mp, np;  // extents and padded ones, multiples of 32
  bool tall;
  int steps;
  double eps, scale;
  float gram[kInnerSteps], poly[kInnerSteps], poly_a[kInnerSteps], update[kInnerSteps], update_x[kInnerSteps];
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

// The wave's blocks of left times right (turned: k across right's lines).  Each
// instruction's large products are added in fp32, rounded.
template <bool kTurned, int kBlocks>
__device__ inline void inner_product(const InnerPlanes& left, const InnerPlanes& right, int blocks, int across, int depth,
                                     InnerBlock (&s)[kBlocks]) {
  const int thread = mma::thread_here(), lane = thread & 63, wave = thread >> 6;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int block = wave + b * kInnerWaves;
    if (block >= blocks) break;
    const int i0 = block / across * 32, j0 = block % across * 32;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) s[b][i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    InnerBlock low = {};
    for (int k0 = 0; k0 < depth; k0 += 32) {
      u32x4 l[2][2], r[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          l[i][q] = inner_along(q == 0 ? left.hi : left.lo, left.ld, i0 + 16 * i, k0, lane);
          const half* p = q == 0 ? right.hi : right.lo;
          r[i][q] = kTurned ? inner_across(p, right.ld, j0 + 16 * i, k0, lane) : inner_along(p, right.ld, j0 + 16 * i, k0, lane);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          low[i][j] = mma::multiply<half>(r[j][1], l[i][0], low[i][j]);
          s[b][i][j] += mma::multiply<half>(r[j][0], l[i][0], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
          low[i][j] = mma::multiply<half>(r[j][0], l[i][1], low[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) s[b][i][j] += low[i][j];
  }
}


// f(row, column, four sums) for the wave's blocks.
template <int kBlocks, typename F>
__device__ inline void inner_each(const InnerBlock (&s)[kBlocks], int blocks, int across, F f) {
  const int thread = mma::thread_here(), lane = thread & 63, wave = thread >> 6;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int block = wave + b * kInnerWaves;
    if (block >= blocks) break;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f(block / across * 32 + i * 16 + (lane & 15), block % across * 32 + j * 16 + (lane >> 4) * 4, s[b][i][j]);
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

// The wave's blocks as finish() takes them: times alpha, and a matrix times
// beta + alpha d, d the left factor's diagonal; kPoly: on both sides, of a
// matrix whose own diagonal it is.
template <bool kPoly, int kBlocks>
__device__ inline void inner_add(InnerBlock (&s)[kBlocks], int blocks, int across, float alpha, const InnerPlanes& p,
                                 float beta, const float* d) {
  const int thread = mma::thread_here(), lane = thread & 63, wave = thread >> 6;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int block = wave + b * kInnerWaves;
    if (block >= blocks) break;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = block / across * 32 + i * 16 + (lane & 15), col = block % across * 32 + j * 16 + (lane >> 4) * 4;
        const f32x4 x = inner_load(p, row, col);
        const float left = d[row];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float w = beta + alpha * left, v = x[e];
          if constexpr (kPoly) {
            if (row == col + e) v = left;
            else w += alpha * d[col + e];
          }
          s[b][i][j][e] = s[b][i][j][e] * alpha + w * v;
        }
      }
  }
}

template <typename T, int kLds, int kBlocks>
__global__ __launch_bounds__(kInnerThreads) void orthogonalize_inner(InnerArgs a, const T* __restrict__ update,
                                                                     T* __restrict__ result) {
  __shared__ __align__(16) char lds[kLds];
  __shared__ double waves[kInnerWaves];
  __shared__ float diagonal[kInnerMost];  // of A, then of its polynomial, whose planes hold zeros there
  const int64_t elements = a.rows * a.cols;
  const T* u = update + blockIdx.x * elements;
  T* out = result + blockIdx.x * elements;
  const int lx = a.np + 8, la = a.mp + 8;
  half* p = reinterpret_cast<half*>(lds);
  const InnerPlanes x{p, p + a.mp * lx, lx}, gram{p + 2 * a.mp * lx, p + 2 * a.mp * lx + a.mp * la, la};
  const int thread = threadIdx.x;

  double squares = 0.0;
  for (int i = thread; i < elements; i += kInnerThreads) {
    const double v = static_cast<double>(static_cast<float>(u[i]));
    squares += v * v;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) squares += __shfl_xor(squares, d);
  if ((thread & 63) == 0) waves[thread >> 6] = squares;
  for (int i = thread; i < a.mp * lx; i += kInnerThreads) x.hi[i] = x.lo[i] = static_cast<half>(0.0f);
  __syncthreads();
  squares = 0.0;
#pragma unroll
  for (int w = 0; w < kInnerWaves; ++w) squares += waves[w];
  const double factor = a.scale / (sqrt(squares) + a.eps);
  for (int i = thread; i < elements; i += kInnerThreads) {
    const int r = i / static_cast<int>(a.cols), c = i % static_cast<int>(a.cols);
    const int at = a.tall ? c * lx + r : r * lx + c;
    to_planes(static_cast<float>(static_cast<double>(static_cast<float>(u[i])) * factor), x.hi[at], x.lo[at]);
  }
  __syncthreads();

  const int square = a.mp / 32 * (a.mp / 32), wide = a.mp / 32 * (a.np / 32);
  InnerBlock s[kBlocks];
  auto store_square = [&](int row, int col, f32x4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (row == col + e) {
        diagonal[row] = v[e];
        v[e] = 0.0f;
      }
    inner_store(gram, row, col, v);
  };
  for (int t = 0; t < a.steps; ++t) {
    inner_product<false>(x, x, square, a.mp / 32, a.np, s);
    inner_each(s, square, a.mp / 32, [&](int row, int col, f32x4 v) { store_square(row, col, v * a.gram[t]); });
    __syncthreads();
    inner_product<false>(gram, gram, square, a.mp / 32, a.mp, s);
    inner_add<true>(s, square, a.mp / 32, a.poly[t], gram, a.poly_a[t], diagonal);
    __syncthreads();  // all of A has been read
    inner_each(s, square, a.mp / 32, store_square);
    __syncthreads();
    inner_product<true>(gram, x, wide, a.np / 32, a.mp, s);
    inner_add<false>(s, wide, a.np / 32, a.update[t], x, a.update_x[t], diagonal);
    if (t + 1 == a.steps) break;
    __syncthreads();  // all of X has been read
    inner_each(s, wide, a.np / 32, [&](int row, int col, f32x4 v) { inner_store(x, row, col, v); });
    __syncthreads();
  }
  inner_each(s, wide, a.np / 32, [&](int row, int col, f32x4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = a.tall ? col + e : row, j = a.tall ? row : col + e;
      if (i < a.rows && j < a.cols) out[i * static_cast<int>(a.cols) + j] = static_cast<T>(v[e]);
    }
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

// Power of two that takes entries of at most `most` to 2^13 .. 2^14: a quarter
// of fp16's range is left for rounding, and low planes stay clear of its least.
double scale_for(double most) {
  if (!(most > 1e-30)) most = 1e-30;
  return std::exp2(std::floor(std::log2(16384.0 / most)));
}

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

// X twice (a step reads one and writes the other), A and P in planes, their
// diagonals, the sums of squares, and the sums of split products.
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
      const int64_t cols = wide ? np : mp, depth = wide ? mp : np, k = splits(d->batch, mp, cols, depth, pair);
      const size_t bytes = k > 1 ? static_cast<size_t>(k * d->batch * mp * cols) * sizeof(float) : 0;
      sums = sums > bytes ? sums : bytes;
    }
  }
  size_t total() const { return 4 * x + 4 * gram + 2 * diagonal + parts + sums; }

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

// The factors of each step's products, for planes scaled by powers of two.
struct Scales {
  double gram, poly, poly_a, update, update_x;
};

// Of step i, from the bound on X's largest singular value, which becomes the
// bound after it.  The last step's result is not scaled.
Scales scales_of(const spmm_orthogonalize_desc* d, int64_t i, double& bound) {
  const double *c = d->coefficients + 3 * i, t = bound * bound, sx = scale_for(bound);
  // largest |b t + c t^2| on [0, bound^2]
  double high = std::fabs(c[1] * t + c[2] * t * t);
  if (c[2] != 0.0 && -c[1] / (2 * c[2]) > 0.0 && -c[1] / (2 * c[2]) < t)
    high = std::fmax(high, std::fabs(c[1] * c[1] / (4 * c[2])));
  const double sa = scale_for(t), sp = scale_for(high);
  bound = largest(c[0], c[1], c[2], bound);
  const double next = i + 1 < d->steps ? scale_for(bound) : 1.0;
  return {sa / (sx * sx), sp * c[2] / (sa * sa), sp * c[1] / sa, next / (sp * sx), next * c[0] / sx};
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
  a.scale = scale_for(1.0);
  double bound = 1.0;
  for (int i = 0; i < a.steps; ++i) {
    const Scales c = scales_of(d, i, bound);
    a.gram[i] = static_cast<float>(c.gram);
    a.poly[i] = static_cast<float>(c.poly);
    a.poly_a[i] = static_cast<float>(c.poly_a);
    a.update[i] = static_cast<float>(c.update);
    a.update_x[i] = static_cast<float>(c.update_x);
  }
  const dim3 grid(static_cast<unsigned>(d->batch)), block(kInnerThreads);
  const T* u = static_cast<const T*>(update);
  if (inner_bytes(a.mp, a.np) <= kInnerLdsFew && a.mp / 32 * (a.np / 32) <= kInnerBlocksFew * kInnerWaves)
    hipLaunchKernelGGL((orthogonalize_inner<T, kInnerLdsFew, kInnerBlocksFew>), grid, block, 0, s, a, u, static_cast<T*>(out));
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
  auto planes = [&](size_t bytes, int64_t ld, bool low) {
    half* hi = reinterpret_cast<half*>(take(bytes));
    half* lo = reinterpret_cast<half*>(take(bytes));
    return Planes{hi, low ? lo : nullptr, ld, l.mp * ld};
  };
  Planes x = planes(l.x, l.np, true), y = planes(l.x, l.np, true);
  const Planes gram = planes(l.gram, l.mp, l.pair), poly = planes(l.gram, l.mp, l.pair);
  float* gram_diagonal = reinterpret_cast<float*>(take(l.diagonal));
  float* poly_diagonal = reinterpret_cast<float*>(take(l.diagonal));
  double* parts = reinterpret_cast<double*>(take(l.parts));
  float* sums = reinterpret_cast<float*>(ws);
  const T* u = static_cast<const T*>(update);
  const unsigned batch = static_cast<unsigned>(d->batch);
  hipLaunchKernelGGL(square_sums<T>, dim3(kNormParts, batch), dim3(kThreads), 0, s, u, l.m * l.n, parts);
  hipLaunchKernelGGL(scale_update<T>, dim3(static_cast<unsigned>(l.np / 64), static_cast<unsigned>(l.mp / 64), batch),
                     dim3(kThreads), 0, s, u, d->rows, d->width, tall, d->eps, scale_for(1.0), parts, l.mp, l.np, x.hi,
                     x.lo);
  if (spmm_status st = check_launch("orthogonalize scale")) return st;
  Finish f{};
  f.diagonals = l.mp;
  f.out = out;
  f.rows = d->rows;
  f.cols = d->width;
  f.tall = tall;
  if (d->steps == 0) {
    f.beta = static_cast<float>(1.0 / scale_for(1.0));
    f.add = x;
    const int64_t blocks = ceil_div(l.mp * l.np / 4 * d->batch, kThreads);
    hipLaunchKernelGGL(store_planes<T>, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(kThreads), 0, s,
                       f, l.mp, d->batch);
    return check_launch("orthogonalize result");
  }
  double bound = 1.0;
  for (int64_t i = 0; i < d->steps; ++i) {
    const Scales c = scales_of(d, i, bound);
    f.alpha = static_cast<float>(c.gram);
    f.to = gram;
    f.diagonal = gram_diagonal;
    if (spmm_status st = multiply<T, kGram>({x, x, mp, mp, np, 1, sums}, f, d->batch, l.pair, s)) return st;
    f.alpha = static_cast<float>(c.poly);
    f.beta = static_cast<float>(c.poly_a);
    f.add = gram;
    f.left = gram_diagonal;
    f.to = poly;
    f.diagonal = poly_diagonal;
    if (spmm_status st = multiply<T, kPoly>({gram, gram, mp, mp, mp, 1, sums}, f, d->batch, l.pair, s)) return st;
    f.alpha = static_cast<float>(c.update);
    f.beta = static_cast<float>(c.update_x);
    f.add = x;
    f.left = poly_diagonal;
    f.to = y;
    const Product p{poly, x, mp, np, mp, 1, sums};
    if (spmm_status st = i + 1 < d->steps ? multiply<T, kUpdate>(p, f, d->batch, l.pair, s)
                                          : multiply<T, kLast>(p, f, d->batch, l.pair, s))
      return st;
    std::swap(x, y);
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
