// Matrix products grouped by row ranges: out[r] = x[r] W[g] for the rows r of
// group g, with dx[r] = grad[r] W[g]^T and dW[g] = x_g^T grad_g.
//
// All three are products of operands as they lie in memory: x and grad are
// read along their rows for out and dx and across them for dW, W either way,
// so nothing is turned first.  Tiles are those of mma_256.h and mma_ring.h
// (fp16 and bf16 whose pieces of 16 bytes are aligned) and mma_staged.h (fp32,
// any alignment, and groups of few rows).
//
// out and dx: one work-group per tile, none across a group's end; which group
// a tile belongs to is found on the device by a wave-wide search of offsets.
//
// dW: groups differ in length and there may be few tiles, so the rows of all
// groups are counted through and cut into equal ranges, and a work-group sums
// one tile over one range, group after group.  A group inside one range is
// written at once; the pieces of one that is cut go to the workspace in fp32
// and are added in order.
#include <climits>
#include <type_traits>
#include <utility>

#include "mma_ring.h"

namespace spmm {
namespace {

struct GroupedArgs {
  int rows, groups;
  int inner, width;  // of the product at hand: depth and output columns
  int64_t in_stride; // rows of its left operand
  int64_t weight_stride;
  const void* offsets;
  bool wide;         // offsets are int64
};

__device__ inline int edge(const GroupedArgs& a, int g) {
  const int64_t v = a.wide ? static_cast<const int64_t*>(a.offsets)[g] : static_cast<const int32_t*>(a.offsets)[g];
  return v < 0 ? 0 : v > a.rows ? a.rows : static_cast<int>(v);
}

// The last s of [0, top) with start(s) <= at, where start(0) <= at < start(top)
// and start ascends: 64 starts a round, three rounds for 262144.  Every lane of
// a wave calls it and gets the same answer.
template <typename F>
__device__ inline int find_start(int top, int at, F start) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = top;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) >> 6, probe = lo + (lane + 1) * step;
    const int f = __ffsll(__ballot(probe >= hi || start(probe) > at)) - 1;  // the last lane's probe is past hi
    const int next = lo + (f + 1) * step;
    hi = next < hi ? next : hi;
    lo += f * step;
  }
  return lo;
}

// The rows as segments: 0 is the rows before the first group, groups + 1 those
// behind the last; both are `group` -1.  Segment s is [bound(s), bound(s + 1)).
__device__ inline int bound(const GroupedArgs& a, int s) {
  return s == 0 ? 0 : s == a.groups + 2 ? a.rows : edge(a, s - 1);
}

struct RowRange {
  int first, rows, group;
};

// Tile `tile` of tiles of kHeight rows, none across a group's end; false where
// it has no rows.  Segment s has the tiles from bound(s) / kHeight + s on, at
// least as many as it needs, so that its first is known without a sum over the
// segments before it.
template <int kHeight>
__device__ inline bool find_rows(const GroupedArgs& a, int tile, RowRange& r) {
  auto start = [&](int s) { return static_cast<int>(static_cast<unsigned>(bound(a, s)) / kHeight) + s; };
  if (tile >= a.rows / kHeight + a.groups + 2) return false;
  const int s = find_start(a.groups + 2, tile, start);
  r.first = bound(a, s) + (tile - start(s)) * kHeight;
  const int left = bound(a, s + 1) - r.first;
  r.rows = left < kHeight ? left : kHeight;
  r.group = s == 0 || s == a.groups + 1 ? -1 : s - 1;
  return left > 0;
}

// The same of the tiles that have rows, counted through: what work-groups that
// stay share out evenly.  `marks` (LDS, kMarks) takes the tiles ahead of every
// 64th segment.
constexpr int kMarks = 256;
template <int kHeight>
struct CountedRows {
  const GroupedArgs& a;
  int* marks;
  int tiles;  // in all

  __device__ inline int size(int s) const {
    const int n = s < a.groups + 2 ? bound(a, s + 1) - bound(a, s) : 0;
    return n > 0 ? (n + kHeight - 1) / kHeight : 0;
  }
  // `upto`: the tiles of the window's segments up to the lane's own.
  __device__ inline int window(int w, int& upto) const {
    const int lane = threadIdx.x & 63, mine = size(w * 64 + lane);
    upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    return mine;
  }

  __device__ inline CountedRows(const GroupedArgs& a, int* marks) : a(a), marks(marks) {
    const int most = a.rows / kHeight + a.groups + 2;  // more only where offsets do not ascend
    int before = 0;
    for (int w = 0; w * 64 < a.groups + 2; ++w) {
      if (threadIdx.x == 0) marks[w] = before;
      int upto;
      window(w, upto);
      before += __builtin_amdgcn_readlane(upto, 63);
      before = before < most ? before : most;
    }
    tiles = before;
    __syncthreads();
  }

  // 0 <= tile < tiles.  (False only where offsets do not ascend.)
  __device__ inline bool find(int tile, RowRange& r) const {
    const int lane = threadIdx.x & 63, windows = (a.groups + 2 + 63) >> 6;
    int w = 0;
    for (int w0 = 0; w0 < windows; w0 += 64) {
      const unsigned long long ahead = __ballot(w0 + lane < windows && marks[w0 + lane] <= tile);
      if (ahead == 0) break;
      w = w0 + 63 - __clzll(ahead);
    }
    int upto;
    const int mine = window(w, upto), before = __builtin_amdgcn_readfirstlane(marks[w]);
    const unsigned long long past = __ballot(before + upto > tile);
    if (past == 0) return false;
    const int found = __ffsll(past) - 1, s = w * 64 + found;
    r.first = bound(a, s) + (tile - before - __builtin_amdgcn_readlane(upto - mine, found)) * kHeight;
    const int left = bound(a, s + 1) - r.first;
    r.rows = left < kHeight ? left : kHeight;
    r.group = s == 0 || s == a.groups + 1 ? -1 : s - 1;
    return left > 0;
  }
};

// Neighbouring sums of one row, rounded; `cols`: of the row from the first of
// them.
template <typename T>
__device__ inline void store_four(T* to, int cols, f32x4 v) {
  typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (cols >= 4) {
    *reinterpret_cast<four*>(to) =
        four{static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < cols) to[e] = static_cast<T>(v[e]);
  }
}
template <typename T>
__device__ inline void store_eight(T* to, int cols, f32x4 v, f32x4 w) {
  if constexpr (sizeof(T) == 2) {
    if (cols >= 8) {
      piece_t<T> p;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = static_cast<T>(v[e]);
        p[e + 4] = static_cast<T>(w[e]);
      }
      *reinterpret_cast<piece_t<T>*>(to) = p;
      return;
    }
  }
  store_four(to, cols, v);
  if (cols > 4) store_four(to + 4, cols - 4, w);
}

// Calls f(row, column, eight sums of neighbouring columns) for the lane's part
// of a tile.
template <typename S, typename F>
__device__ inline void each_eight(S& s, F f) {
  s.place();
#pragma unroll
  for (int k = 0; k < S::kEights; ++k) f(s.row(k), s.col(k), s.four(k, 0), s.four(k, 1));
}

// The engines of one product: Large of mma_256.h, Middle of mma_ring.h, Small of
// mma_staged.h.
template <typename T, bool kAC, bool kBC>
struct Large {
  typedef T Value;
  static constexpr int kRows = mma::kTile, kCols = mma::kTile, kThreads = mma::kThreads;
  static constexpr int kLds = mma::kLdsBytes, kPerCu = 1;
  mma::Sums s;
  __device__ inline void sum(const mma::Operand<T>& a, const mma::Operand<T>& b, char* lds) {
    mma::multiply_tile<T, kAC, kBC, 1>(a, b, lds, s);
  }
  template <typename F>
  __device__ inline void each(F f) {
    each_eight(s, f);
  }
};

template <typename T, bool kAC, bool kBC, int kHeight, bool kAligned>
struct Small {
  typedef T Value;
  static constexpr int kRows = kHeight, kCols = kHeight == 32 ? 128 : 64, kThreads = mma::kThreads128;
  typedef mma::Staged<T, kAC, kBC, kRows, kCols, kAligned> Tile;
  static constexpr int kLds = Tile::kLdsBytes, kPerCu = 4;
  typename Tile::Sums s;
  __device__ inline void sum(const mma::Operand<T>& a, const mma::Operand<T>& b, char* lds) { Tile::sum(a, b, lds, s); }
  template <typename F>
  __device__ inline void each(F f) {
    each_eight(s, f);
  }
};

template <typename T, bool kAC, bool kBC>
struct Middle {
  typedef T Value;
  typedef mma::Ring<T, kAC, kBC, false, 128, 128> Tile;
  static constexpr int kRows = 128, kCols = 128, kThreads = mma::kThreads128, kStep = Tile::kDepth;
  static constexpr int kLds = Tile::kLdsBytes, kPerCu = 2;
  typename Tile::Sums s;
  __device__ inline void sum(const mma::Operand<T>& a, const mma::Operand<T>& b, char* lds) {
    s.clear();
    Tile::add(a, b, lds, 0, static_cast<int>((a.depth + kStep - 1) / kStep), s);
  }
  template <typename F>
  __device__ inline void each(F f) {
    each_eight(s, f);
  }
};

// out or dx; kTurned: the weights' depth is their contiguous extent.
template <typename E, bool kTurned>
__global__ __launch_bounds__(E::kThreads, E::kPerCu* E::kThreads / 256) void grouped_rows(
    GroupedArgs a, const typename E::Value* __restrict__ in, const typename E::Value* __restrict__ weight,
    typename E::Value* __restrict__ out, unsigned down) {
  typedef typename E::Value T;
  __shared__ __align__(1024) char lds[E::kLds];
  const unsigned across = (a.width + E::kCols - 1) / E::kCols;
  unsigned i, j;
  mma::place_tile(mma::run_of_xcd(blockIdx.x, gridDim.x), down, across, i, j);
  RowRange r;
  if (!find_rows<E::kRows>(a, i, r)) return;
  const int c0 = j * E::kCols, cols = a.width - c0 < E::kCols ? a.width - c0 : E::kCols;
  T* to = out + static_cast<int64_t>(r.first) * a.width + c0;
  E e;
  const T* w = weight + (r.group < 0 ? 0 : r.group) * a.weight_stride + (kTurned ? static_cast<int64_t>(c0) * a.inner : c0);
  // outside the groups: an empty sum
  const int depth = r.group < 0 ? 0 : a.inner;
  e.sum({in + r.first * a.in_stride, nullptr, a.in_stride, r.rows, depth},
        {w, nullptr, kTurned ? a.inner : a.width, cols, depth}, lds);
  e.each([&](int row, int col, f32x4 v, f32x4 w) {
    if (row < r.rows && col < cols) store_eight(to + static_cast<int64_t>(row) * a.width + col, cols - col, v, w);
  });
}

// The same by 256 work-groups that stay, on large tiles: a tile's first copies
// are started before the last one's sums are stored, so that neither the one's
// latency nor the other's burst of stores leaves the matrix cores idle.  An
// XCD's work-groups take neighbouring tiles of its run; runs are of the tiles
// that there are (the host knows only how many at most).
template <typename T, bool kTurned>
__global__ __launch_bounds__(mma::kThreads, 2) void grouped_rows_large(GroupedArgs a, const T* __restrict__ in,
                                                                       const T* __restrict__ weight,
                                                                       T* __restrict__ out) {
  constexpr int kTile = mma::kTile, kStores = mma::Sums::kEights;
  typedef mma::Tile256<T, false, !kTurned, 1> Tile;
  __shared__ __align__(1024) char lds[mma::kLdsBytes];
  __shared__ int marks[kMarks];
  const CountedRows<kTile> counted(a, marks);
  const unsigned down = counted.tiles, across = (a.width + kTile - 1) / kTile, tiles = down * across;
  const unsigned x = blockIdx.x % kXcds, rest = tiles % kXcds;
  const unsigned begin = x * (tiles / kXcds) + (x < rest ? x : rest), end = begin + tiles / kXcds + (x < rest ? 1 : 0);
  const unsigned stride = gridDim.x / kXcds;

  struct Place {
    RowRange r;
    int c0, cols;
  };
  // tile n; false past the run
  auto find = [&](unsigned n, Place& p) {
    if (n >= end) return false;
    unsigned i, j;
    mma::place_tile(n, down, across, i, j);
    if (!counted.find(i, p.r)) return false;
    p.c0 = j * kTile;
    p.cols = a.width - p.c0 < kTile ? a.width - p.c0 : kTile;
    return true;
  };
  auto tile_at = [&](const Place& p) {
    const T* w = weight + (p.r.group < 0 ? 0 : p.r.group) * a.weight_stride +
                 (kTurned ? static_cast<int64_t>(p.c0) * a.inner : p.c0);
    const int depth = p.r.group < 0 ? 0 : a.inner;  // outside the groups: an empty sum
    return Tile({in + p.r.first * a.in_stride, nullptr, a.in_stride, p.r.rows, depth},
                {w, nullptr, kTurned ? a.inner : a.width, p.cols, depth}, lds, mma::thread_here());
  };

  unsigned n = begin + blockIdx.x / kXcds;
  Place here, next;
  if (!find(n, here)) return;
  Tile t = tile_at(here);
  t.start();
  mma::wait_copies<0>();  // no stores are under way yet: what run() lets pass must have arrived
  for (;;) {
    mma::Sums s;
    t.template run<kStores>(lds, s);
    n += stride;
    const bool more = find(n, next);  // nothing is under way here that its loads would wait for
    if (more) {
      t = tile_at(next);
      t.start();
    }
    s.place();
    // Every wave issues kStores stores; the buffer's end and the offset past it
    // drop what lies outside.
    T* to = out + static_cast<int64_t>(here.r.first) * a.width + here.c0;
    const int bytes = static_cast<int>(sizeof(T)) * ((here.r.rows - 1) * a.width + here.cols);
    const __amdgpu_buffer_rsrc_t b = __builtin_amdgcn_make_buffer_rsrc(to, static_cast<short>(0), bytes, 0x00020000);
#pragma unroll
    for (int k = 0; k < kStores; ++k) {
      const f32x4 v = s.four(k, 0), w = s.four(k, 1);
      typedef T Eight __attribute__((ext_vector_type(8)));
      Eight p;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = static_cast<T>(v[e]);
        p[e + 4] = static_cast<T>(w[e]);
      }
      const unsigned at = s.col(k) < here.cols ? static_cast<unsigned>(sizeof(T)) * (s.row(k) * a.width + s.col(k)) : 0x80000000u;
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, p), b, static_cast<int>(at), 0, 0);
    }
    if (!more) return;
    here = next;
  }
}

// dW's sums run over the rows of all groups, counted in steps of 64 (every
// group has one at least, and may have one that adds nothing) and cut into
// `parts` equal ranges.  The cuts depend on sizes alone, so every engine adds
// in the same order.  Group g's steps are [steps.start(g), steps.start(g + 1)).
constexpr int kRowStep = 64;
struct Steps {
  const GroupedArgs& a;
  int origin, total;
  __device__ inline explicit Steps(const GroupedArgs& a) : a(a), origin(edge(a, 0) / kRowStep) { total = start(a.groups); }
  __device__ inline int start(int g) const { return static_cast<int>(static_cast<unsigned>(edge(a, g)) / kRowStep) + g - origin; }
  // 0 <= at < total
  __device__ inline int find(int at) const {
    return find_start(a.groups, at, [&](int g) { return start(g); });
  }
};
__device__ inline int part_start(int total, int part, int parts) {
  return static_cast<int>(static_cast<int64_t>(total) * part / parts);
}

// A work-group sums one tile over one range; tiles of a range are neighbours,
// which share its rows in their XCD's L2.  The pieces of groups that a range
// cuts go to pieces [parts][tiles][2][tile] in fp32: a range's first group to
// the first place, its last one to the second.
template <typename E>
__global__ __launch_bounds__(E::kThreads, E::kPerCu* E::kThreads / 256) void grouped_weights(
    GroupedArgs a, const typename E::Value* __restrict__ left, int64_t left_stride,
    const typename E::Value* __restrict__ right, int64_t right_stride, typename E::Value* __restrict__ dweight,
    int parts, float* __restrict__ pieces) {
  typedef typename E::Value T;
  __shared__ __align__(1024) char lds[E::kLds];
  const unsigned across = (a.width + E::kCols - 1) / E::kCols, down = (a.inner + E::kRows - 1) / E::kRows;
  const Steps steps(a);
  const unsigned block = mma::run_of_xcd(blockIdx.x, gridDim.x);
  const int part = block / (across * down);
  unsigned i, j;
  mma::place_tile(block - part * (across * down), down, across, i, j);
  if (parts > steps.total) parts = steps.total;  // of which the host knows only how many at most
  if (part >= parts) return;
  const int i0 = i * E::kRows, j0 = j * E::kCols;
  const int rows = a.inner - i0 < E::kRows ? a.inner - i0 : E::kRows;
  const int cols = a.width - j0 < E::kCols ? a.width - j0 : E::kCols;
  const int u0 = part_start(steps.total, part, parts), u1 = part_start(steps.total, part + 1, parts);
  int g = steps.find(u0), before = steps.start(g);
  for (int u = u0; u < u1 && g < a.groups; ++g) {
    const int lo = edge(a, g), hi = edge(a, g + 1), n = steps.start(g + 1) - before;
    const int s0 = u - before, s1 = n - s0 < u1 - u ? n : s0 + (u1 - u);
    const int first = lo + s0 * kRowStep, last = hi - lo > s1 * kRowStep ? lo + s1 * kRowStep : hi;
    const int depth = last > first ? last - first : 0;
    E e;
    e.sum({left + first * left_stride + i0, nullptr, left_stride, rows, depth},
          {right + first * right_stride + j0, nullptr, right_stride, cols, depth}, lds);
    if (s0 == 0 && s1 == n) {
      T* to = dweight + (static_cast<int64_t>(g) * a.inner + i0) * a.width + j0;
      e.each([&](int row, int col, f32x4 v, f32x4 w) {
        if (row < rows && col < cols) store_eight(to + static_cast<int64_t>(row) * a.width + col, cols - col, v, w);
      });
    } else {
      float* to = pieces + (2 * static_cast<int64_t>(block) + (u == u0 ? 0 : 1)) * E::kRows * E::kCols;
      e.each([&](int row, int col, f32x4 v, f32x4 w) {
        *reinterpret_cast<f32x4*>(to + row * E::kCols + col) = v;
        *reinterpret_cast<f32x4*>(to + row * E::kCols + col + 4) = w;
      });
    }
    u += s1 > s0 ? s1 - s0 : 1;
    before += n;
  }
}

// Adds the pieces of the groups that were cut; a work-group takes kJoin sums of
// a group's tile.  by_cut: of the group that holds the cut before range n + 1,
// where that is the group's first cut; else of group n.
template <typename T, int kJoin>
__global__ __launch_bounds__(256) void join_pieces(GroupedArgs a, int tile_rows, int tile_cols, int parts, bool by_cut,
                                                   const float* __restrict__ pieces, T* __restrict__ dweight) {
  const unsigned across = (a.width + tile_cols - 1) / tile_cols, down = (a.inner + tile_rows - 1) / tile_rows;
  const unsigned tiles = across * down, size = tile_rows * tile_cols, slices = size / kJoin;
  const unsigned each = blockIdx.x / slices, n = each / tiles, tile = each - n * tiles;
  const Steps steps(a);
  const int total = steps.total;
  if (parts > total) parts = total;
  if (parts <= 0) return;
  int g, u0, part;  // the group, its first step, and the range that holds it
  if (by_cut) {
    if (n + 1 >= static_cast<unsigned>(parts)) return;
    const int cut = part_start(total, n + 1, parts);
    g = steps.find(cut);
    u0 = steps.start(g);
    if (cut == u0 || part_start(total, n, parts) > u0) return;
    part = n;
  } else {
    g = n;
    u0 = steps.start(g);
    if (u0 < 0 || u0 >= total) return;  // (offsets that do not ascend)
    part = static_cast<int>(static_cast<int64_t>(u0) * parts / total);
    while (part > 0 && part_start(total, part, parts) > u0) --part;
    while (part + 1 < parts && part_start(total, part + 1, parts) <= u0) ++part;
  }
  const int u_end = steps.start(g + 1), u1 = u_end < total ? u_end : total;
  if (u1 <= u0 || part_start(total, part + 1, parts) >= u1) return;  // written whole
  // ranges that start inside the group
  int end = static_cast<int>(static_cast<int64_t>(u1) * parts / total);
  while (end > part + 1 && part_start(total, end - 1, parts) >= u1) --end;
  while (end < parts && part_start(total, end, parts) < u1) ++end;
  const int64_t range = static_cast<int64_t>(tiles) * 2 * size;
  const float* from = pieces + static_cast<int64_t>(tile) * 2 * size + (blockIdx.x - each * slices) * kJoin + threadIdx.x * 4;
  f32x4 s[kJoin / 1024];
#pragma unroll
  for (int k = 0; k < kJoin / 1024; ++k)
    s[k] = *reinterpret_cast<const f32x4*>(from + part * range + (part_start(total, part, parts) < u0 ? size : 0) + 1024 * k);
#pragma unroll 8192 / kJoin
  for (++part; part < end; ++part)
#pragma unroll
    for (int k = 0; k < kJoin / 1024; ++k) s[k] += *reinterpret_cast<const f32x4*>(from + part * range + 1024 * k);
  unsigned i, j;
  mma::place_tile(tile, down, across, i, j);
#pragma unroll
  for (int k = 0; k < kJoin / 1024; ++k) {
    const unsigned e = (blockIdx.x - each * slices) * kJoin + 1024 * k + threadIdx.x * 4;
    const int row = i * tile_rows + e / tile_cols, col = j * tile_cols + e % tile_cols;
    if (row < a.inner && col < a.width)
      store_four(dweight + (static_cast<int64_t>(g) * a.inner + row) * a.width + col, a.width - col, s[k]);
  }
}

constexpr int64_t kMostStride = int64_t(1) << 22;

spmm_status check_grouped_desc(const spmm_grouped_desc* d, const char* op) {
  if (d == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null descriptor");
  if (d->index_type != SPMM_INDEX_I32 && d->index_type != SPMM_INDEX_I64)
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": offsets must be int32 or int64");
  if (!dense_type(d->value_type))
    return fail(SPMM_ERR_CONTRACT, std::string(op) + " supports only FP16, BF16 and FP32 tensors");
  if (d->rows < 0 || d->groups < 0 || d->inner < 0 || d->width < 0)
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": negative extent");
  if (d->rows > INT32_MAX - 512 || d->groups > (1 << 24))
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": rows must be below 2^31 and groups at most 2^24");
  // offsets inside a tile are 32-bit
  if (d->inner >= kMostStride || d->width >= kMostStride || (d->rows > 1 && d->x_stride >= kMostStride))
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": inner, width and row strides must be below 2^22");
  if (d->rows > 1 && d->x_stride < d->inner) return fail(SPMM_ERR_CONTRACT, std::string(op) + ": rows of x overlap");
  if (d->groups > 1 && d->weight_stride < d->inner * d->width)
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": matrices of weight overlap");
  return SPMM_OK;
}

// Work-groups of a launch: a grid's limit, 2^32 work-items, is an error, not a
// wrapped count.
spmm_status check_grid(int64_t blocks, int64_t threads, const char* op) {
  if (blocks * threads > UINT32_MAX) return fail(SPMM_ERR_OVERFLOW, std::string(op) + ": too many tiles for one launch");
  return SPMM_OK;
}

// Whether 16-byte pieces of the operands can be copied as they lie.
bool pieces_aligned(const spmm_grouped_desc* d, const void* x, const void* weight, const void* grad) {
  const int64_t size = dense_type_bytes(d->value_type);
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(grad);
  return at % 16 == 0 && d->inner % 8 == 0 && d->width % 8 == 0 && (d->rows <= 1 || d->x_stride * size % 16 == 0) &&
         (grad == nullptr || d->rows <= 1 || d->grad_stride * size % 16 == 0) &&
         (d->groups <= 1 || d->weight_stride * size % 16 == 0);
}

constexpr int64_t kCus = 256;

// The large tile for out and dx, where three quarters of the CUs get one and the
// groups' average fills half of it: 65536 rows in 8 groups, 1024 x 2048 bf16,
// 300 and 310 us against 444 and 459 with tiles of 128; at the rule's edges,
// 49152 rows of 256 x 256, 17 against 20, and 192 groups of 128 rows, 1024 x
// 1024, 138 against 179.  More groups than its marks hold go to tiles of 128.
bool large_rows(const GroupedArgs& a) {
  return a.width > 128 && a.inner >= 2 * mma::kDepth && a.rows / mma::kTile * ceil_div(a.width, mma::kTile) >= kCus * 3 / 4 &&
         a.rows / (mma::kTile / 2) >= a.groups && a.groups + 2 <= 64 * kMarks;
}

// The low tile where the groups' average leaves most of a tile of 128 empty: 13
// rows in 8 groups, 512 x 512 bf16, 6.8 us against 9.4; at the edge, 42 groups
// of 48 rows, 10.1 against 10.9.
bool low_rows(const GroupedArgs& a) { return a.rows / 48 < a.groups; }

// Copies count an operand's pieces in 32 bits.
bool small_counts(const GroupedArgs& a, int64_t stride, int64_t other) {
  return static_cast<int64_t>(a.rows) * (stride > other ? stride : other) < (int64_t(1) << 33);
}

// The large tile for dW, where the groups' average keeps it busy for 8 steps:
// 8 groups of 8192 rows, 1024 x 2048 bf16, 262 us against 342 with tiles of
// 128; 60 groups of 273 rows, 1024 x 1024, 105 against 100.
bool large_weights(const GroupedArgs& a) {
  return a.inner > 128 && a.width > 128 && a.rows / (8 * mma::kDepth) >= a.groups;
}

// Ranges that dW's rows are cut into: the number that takes the least time by
// this count, in microseconds.  A round of work-groups takes 1.6 a step for the
// large tile (4096 x 4096 x 4096: 108 us), 0.8 for two of 128 on a CU, and 4.6
// for four of fp32's (the same product: 1150 us); a cut costs a piece of each
// tile written and read at 4 TB/s, and joining a launch.
int64_t weight_parts(const GroupedArgs& a, bool fp32) {
  const bool large = !fp32 && large_weights(a);
  const int64_t side = large ? mma::kTile : fp32 ? 64 : 128, at_once = kCus * (large ? 1 : fp32 ? 4 : 2);
  const int64_t tiles = ceil_div(a.inner, side) * ceil_div(a.width, side);
  const int64_t steps = a.rows / kRowStep + a.groups;
  if (tiles == 0 || steps == 0) return 1;
  const double step = large ? 1.6 : fp32 ? 4.6 : 0.8, piece = static_cast<double>(tiles * side * side) * 8.0 / 4e6;
  int64_t best = 1;
  double least = 1e300;
  auto consider = [&](int64_t parts) {
    if (parts < 1 || parts > steps) return;
    const double time = static_cast<double>(ceil_div(parts * tiles, at_once) * ceil_div(steps, parts)) * step +
                        (parts > 1 ? static_cast<double>(parts) * piece + 4.0 : 0.0);
    if (time < least) {
      least = time;
      best = parts;
    }
  };
  for (int64_t p = 1; p <= 4; ++p) consider(p);
  for (int64_t k = 1; k <= 32; ++k) consider(at_once * k / (8 * tiles));
  return best;
}
template <typename E>
size_t weight_bytes(const GroupedArgs& a) {
  const int64_t parts = weight_parts(a, std::is_same_v<typename E::Value, float>);
  const int64_t tiles = ceil_div(a.inner, E::kRows) * ceil_div(a.width, E::kCols);
  return parts == 1 ? 0 : static_cast<size_t>(parts * tiles) * 2 * E::kRows * E::kCols * sizeof(float);
}

// Calls f with null pointers of the value type.
template <typename F>
spmm_status with_type(int32_t value_type, F f) {
  switch (value_type) {
    case SPMM_VALUE_F16: return f(static_cast<_Float16*>(nullptr));
    case SPMM_VALUE_BF16: return f(static_cast<__bf16*>(nullptr));
    default: return f(static_cast<float*>(nullptr));
  }
}
template <typename P>
using value_of = std::remove_pointer_t<P>;

template <typename E, bool kTurned>
spmm_status launch_rows(const GroupedArgs& a, const void* in, const void* weight, void* out, hipStream_t s,
                        const char* op) {
  typedef typename E::Value T;
  const int64_t down = ceil_div(a.rows, E::kRows) + a.groups + 1;
  const int64_t blocks = down * ceil_div(a.width, E::kCols);
  if (spmm_status st = check_grid(blocks, E::kThreads, op)) return st;
  hipLaunchKernelGGL((grouped_rows<E, kTurned>), dim3(static_cast<unsigned>(blocks)), dim3(E::kThreads), 0, s, a,
                     static_cast<const T*>(in), static_cast<const T*>(weight), static_cast<T*>(out), static_cast<unsigned>(down));
  return check_launch(op);
}

// in [rows, depth] times each group's matrix, whose depth is contiguous where
// kTurned.
template <typename T, bool kTurned>
spmm_status run_rows(const GroupedArgs& a, bool aligned, const void* in, const void* weight, void* out, hipStream_t s,
                     const char* op) {
  if (a.rows == 0 || a.width == 0) return SPMM_OK;
  // (copies count a matrix's pieces in 32 bits)
  aligned = aligned && static_cast<int64_t>(a.inner) * a.width < (int64_t(1) << 33);
  if constexpr (sizeof(T) == 2)
    // Its buffer stores are of whole, aligned pieces; the other tiles store at any
    // element.
    if (aligned && reinterpret_cast<uintptr_t>(out) % 16 == 0 && large_rows(a)) {
      // (the kernel counts its tiles in 32 bits)
      const int64_t down = ceil_div(a.rows, mma::kTile) + a.groups + 1;
      if (spmm_status st = check_grid(down * ceil_div(a.width, mma::kTile), 1, op)) return st;
      hipLaunchKernelGGL((grouped_rows_large<T, kTurned>), dim3(kCus), dim3(mma::kThreads), 0, s, a,
                         static_cast<const T*>(in), static_cast<const T*>(weight), static_cast<T*>(out));
      return check_launch(op);
    }
  if (low_rows(a))
    return aligned ? launch_rows<Small<T, false, !kTurned, 32, true>, kTurned>(a, in, weight, out, s, op)
                   : launch_rows<Small<T, false, !kTurned, 32, false>, kTurned>(a, in, weight, out, s, op);
  if constexpr (sizeof(T) == 2)
    if (aligned) return launch_rows<Middle<T, false, !kTurned>, kTurned>(a, in, weight, out, s, op);
  if constexpr (sizeof(T) == 4)
    if (aligned) return launch_rows<Small<T, false, !kTurned, 64, true>, kTurned>(a, in, weight, out, s, op);
  return launch_rows<Small<T, false, !kTurned, 64, false>, kTurned>(a, in, weight, out, s, op);
}

template <typename E>
spmm_status launch_weights(const GroupedArgs& a, const void* left, int64_t left_stride, const void* right,
                           int64_t right_stride, void* dweight, void* ws, size_t ws_bytes, hipStream_t s,
                           const char* op) {
  typedef typename E::Value T;
  const size_t need = weight_bytes<E>(a);
  if (need > 0 && (ws == nullptr || ws_bytes < need))
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": workspace too small: need " + std::to_string(need) + " bytes");
  const int64_t parts = weight_parts(a, std::is_same_v<typename E::Value, float>);
  const int64_t tiles = ceil_div(a.inner, E::kRows) * ceil_div(a.width, E::kCols);
  // Joined by groups or by cuts, whichever are fewer.
  const bool by_cut = parts - 1 < a.groups;
  const int64_t sums = (by_cut ? parts - 1 : a.groups) * tiles * (E::kRows * E::kCols);
  if (spmm_status st = check_grid(parts * tiles, E::kThreads, op)) return st;
  if (spmm_status st = check_grid(sums / 1024, 256, op)) return st;
  hipLaunchKernelGGL(grouped_weights<E>, dim3(static_cast<unsigned>(parts * tiles)), dim3(E::kThreads), 0, s, a,
                     static_cast<const T*>(left), left_stride, static_cast<const T*>(right), right_stride,
                     static_cast<T*>(dweight), static_cast<int>(parts), static_cast<float*>(ws));
  if (spmm_status st = check_launch(op)) return st;
  if (parts == 1) return SPMM_OK;
  // A work-group takes 4096 sums where that leaves eight for each CU (8 groups
  // of 1024 x 2048: 28 us, 62 with 1024), else 1024 (12 of 128 x 128: 6.5, 10).
  auto join = [&](auto size) {
    constexpr int kJoin = decltype(size)::value;
    hipLaunchKernelGGL((join_pieces<T, kJoin>), dim3(static_cast<unsigned>(sums / kJoin)), dim3(256), 0, s, a, E::kRows,
                       E::kCols, static_cast<int>(parts), by_cut, static_cast<const float*>(ws),
                       static_cast<T*>(dweight));
  };
  if (sums >= 8 * kCus * 4096)
    join(std::integral_constant<int, 4096>());
  else
    join(std::integral_constant<int, 1024>());
  return check_launch(op);
}

// The stride of an operand's rows.  A single row's is not looked at by the
// checks and may be anything, but where rows are a product's depth, lines past
// the last one are kept out by lying past the operand's end: at least as far
// apart as they are wide, and in whole pieces as every stride there.
int64_t stride_of(const spmm_grouped_desc* d, int64_t stride, int64_t columns) {
  return d->rows > 1 ? stride : static_cast<int64_t>(align_up(static_cast<size_t>(columns), 8));
}

GroupedArgs grouped_args(const spmm_grouped_desc* d, const void* offsets) {
  return {static_cast<int>(d->rows), static_cast<int>(d->groups), static_cast<int>(d->inner),
          static_cast<int>(d->width), stride_of(d, d->x_stride, d->inner), d->weight_stride, offsets,
          d->index_type == SPMM_INDEX_I64};
}

// dW's operands, in the order of weight's storage.
struct WeightSides {
  GroupedArgs a;
  const void *left, *right;
  int64_t left_stride, right_stride;
  WeightSides(const spmm_grouped_desc* d, const void* offsets, const void* x, const void* grad)
      : a(grouped_args(d, offsets)),
        left(x),
        right(grad),
        left_stride(stride_of(d, d->x_stride, d->inner)),
        right_stride(stride_of(d, d->grad_stride, d->width)) {
    if (d->weight_transposed) {
      std::swap(a.inner, a.width);
      std::swap(left, right);
      std::swap(left_stride, right_stride);
    }
  }
};

template <typename T, typename F>
spmm_status with_weight_engine(const GroupedArgs& a, bool aligned, int64_t stride, int64_t other, F f) {
  if constexpr (sizeof(T) == 2)
    if (aligned && small_counts(a, stride, other))
      return large_weights(a) ? f(static_cast<Large<T, true, true>*>(nullptr))
                              : f(static_cast<Middle<T, true, true>*>(nullptr));
  if constexpr (sizeof(T) == 4)
    if (aligned) return f(static_cast<Small<T, true, true, 64, true>*>(nullptr));
  return f(static_cast<Small<T, true, true, 64, false>*>(nullptr));
}

}  // namespace
}  // namespace spmm

using namespace spmm;

extern "C" {

spmm_status spmm_grouped_workspace(const spmm_grouped_desc* d, size_t* bytes) {
  clear_error();
  if (bytes == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null argument");
  if (spmm_status st = check_grouped_desc(d, "grouped_matmul")) return st;
  *bytes = 0;
  return SPMM_OK;
}

spmm_status spmm_grouped_run(const spmm_grouped_desc* d, const void* x, const void* weight, const void* offsets,
                             void* out, void* workspace, size_t workspace_bytes, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_grouped_desc(d, "grouped_matmul")) return st;
  if (d->rows == 0 || d->width == 0) return SPMM_OK;
  if (offsets == nullptr || out == nullptr ||
      (d->inner > 0 && (x == nullptr || (d->groups > 0 && weight == nullptr))))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "grouped_matmul: null device pointer");
  (void)workspace;
  (void)workspace_bytes;
  const GroupedArgs a = grouped_args(d, offsets);
  const bool aligned = pieces_aligned(d, x, weight, nullptr);
  hipStream_t s = as_stream(stream);
  return with_type(d->value_type, [&](auto* t) {
    using T = value_of<decltype(t)>;
    return d->weight_transposed ? run_rows<T, true>(a, aligned, x, weight, out, s, "grouped_matmul")
                                : run_rows<T, false>(a, aligned, x, weight, out, s, "grouped_matmul");
  });
}

spmm_status spmm_grouped_grad_workspace(const spmm_grouped_desc* d, size_t* bytes) {
  clear_error();
  if (bytes == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null argument");
  if (spmm_status st = check_grouped_desc(d, "grouped_matmul")) return st;
  // of whichever engine the pointers' alignment leads to
  const WeightSides w(d, nullptr, nullptr, nullptr);
  return with_type(d->value_type, [&](auto* t) {
    size_t most = 0;
    for (bool aligned : {false, true})
      with_weight_engine<value_of<decltype(t)>>(w.a, aligned, w.left_stride, w.right_stride, [&](auto* e) {
        const size_t need = weight_bytes<value_of<decltype(e)>>(w.a);
        most = need > most ? need : most;
        return SPMM_OK;
      });
    *bytes = most;
    return SPMM_OK;
  });
}

spmm_status spmm_grouped_grad_run(const spmm_grouped_desc* d, const void* x, const void* weight, const void* offsets,
                                  const void* grad, void* dx, void* dweight, void* workspace, size_t workspace_bytes,
                                  spmm_stream stream) {
  const char* op = "grouped_matmul gradient";
  clear_error();
  if (spmm_status st = check_grouped_desc(d, "grouped_matmul")) return st;
  if (d->rows > 1 && d->grad_stride < d->width)
    return fail(SPMM_ERR_CONTRACT, "grouped_matmul: rows of grad overlap");
  if (d->rows > 1 && d->grad_stride >= kMostStride)
    return fail(SPMM_ERR_CONTRACT, "grouped_matmul: inner, width and row strides must be below 2^22");
  if (offsets == nullptr || (d->rows > 0 && d->width > 0 && grad == nullptr) ||
      (dx != nullptr && d->groups > 0 && d->inner > 0 && d->width > 0 && weight == nullptr) ||
      (dweight != nullptr && d->rows > 0 && d->inner > 0 && x == nullptr))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "grouped_matmul: null device pointer");
  const bool aligned = pieces_aligned(d, x, weight, grad);
  hipStream_t s = as_stream(stream);
  return with_type(d->value_type, [&](auto* t) {
    using T = value_of<decltype(t)>;
    if (dx != nullptr) {
      GroupedArgs a = grouped_args(d, offsets);
      std::swap(a.inner, a.width);
      a.in_stride = stride_of(d, d->grad_stride, d->width);
      // W^T: its depth is W's columns, contiguous unless W is transposed
      if (spmm_status st = d->weight_transposed ? run_rows<T, false>(a, aligned, grad, weight, dx, s, op)
                                                : run_rows<T, true>(a, aligned, grad, weight, dx, s, op))
        return st;
    }
    if (dweight == nullptr || d->groups == 0 || d->inner == 0 || d->width == 0) return SPMM_OK;
    const WeightSides w(d, offsets, x, grad);
    return with_weight_engine<T>(w.a, aligned, w.left_stride, w.right_stride, [&](auto* e) {
      return launch_weights<value_of<decltype(e)>>(w.a, w.left, w.left_stride, w.right, w.right_stride, dweight,
                                                   workspace, workspace_bytes, s, op);
    });
  });
}

}  // extern "C"
