// Log probabilities of given classes under a softmax over each row of logits,
// the entropy, and the best classes; and the gradient of the first two.
//
// With m the row's maximum, z = x - m, s = sum e^z and ls = log s:
//   logp = z_t - ls,   H = ls - sum e^z z / s,
//   dx_i = a ([i = t] - p_i) - h p_i (log p_i + H),   p_i = e^(z_i - ls),
// for incoming gradients a of logp and h of H.  H is a sum of two terms of one
// sign, so it keeps its digits where it is small.
//
// All of it is fp32 and in powers of two: y = fma(x, log2(e), -c), c = m log2(e)
// rounded, rounds once for each logit.  c need not be exact, as every y has the
// same c: it is taken out again as a whole.  But y of the maximum is what c was
// rounded by, so c has to be small enough that this is next to nothing: beyond
// |m| = 2^20, y = (x - m) log2(e), which rounds twice.
#include <cfloat>
#include <cmath>

#include "lane_reduce.h"
#include "row_pieces.h"

namespace spmm {
namespace {

constexpr int kThreads = 256;
constexpr int kWideThreads = 512;
constexpr int kMaxTop = 64;
constexpr int kMaxParts = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
// A greater maximum has a c that will not do.  Up to it c is below 2^21, and
// rounded by 2^-4 at most.
constexpr float kFar = 0x1p20f;
constexpr float kFloor = -300.0f;  // below it 2^y is zero; a finite stand-in for an infinite y

// The product by itself: contracted with a difference of two of them it would
// leave their rounding, and equal origins would not be equal.
__device__ inline float origin_of(float m) {
#pragma clang fp contract(off)
  return fmaxf(m, -kFar) * kLog2e;
}

// What the logits of a row are measured from.
struct Origin {
  float m, c;
  bool far;
  __device__ inline explicit Origin(float max)
      : m(max), c(origin_of(max)), far(!(fabsf(max) <= kFar)) {}
  __device__ inline float near(float x) const { return __builtin_fmaf(x, kLog2e, -c); }
  __device__ inline float operator()(float x) const { return far ? (x - m) * kLog2e : near(x); }
  // log p of a logit, given log2 s.  So far below the maximum that its y may overflow where its
  // distance does not (a type's lowest value), it is the distance: log s is nothing against it,
  // unless it is NaN.
  __device__ inline float log_p(float x, float ls) const {
    const float y = (*this)(x);
    return y < -1e30f ? (x - m) - ls : (y - ls) * kLn2;
  }
};

struct LogArgs {
  int64_t rows, classes, stride;
  int32_t top;
  bool index64;
};

__device__ inline int64_t target_of(const void* targets, bool index64, int64_t r) {
  return index64 ? static_cast<const int64_t*>(targets)[r] : static_cast<const int32_t*>(targets)[r];
}

struct RowOut {
  float* logp;
  float* entropy;
  float* top_values;
  int32_t* top_ids;
  float* stats;  // [rows][2]: m and log2 s, or null
};

// What a row's maximum, s = sum 2^y and t = sum 2^y y say, by one thread: returns
// log2 s.  A row whose logits are all -inf has s = 0: logp -inf, no entropy, and
// an infinite log2 s, which makes every p of the gradient zero.
__device__ inline float finish_row(const LogArgs& a, const RowOut& out, int64_t r, int64_t target, float xt,
                                   const Origin& o, float s, float t) {
  const float ls = s == 0.0f ? INFINITY : log2f(s);
  const bool named = static_cast<uint64_t>(target) < static_cast<uint64_t>(a.classes);
  out.logp[r] = named ? (s == 0.0f ? -INFINITY : o.log_p(xt, ls)) : 0.0f;
  out.entropy[r] = s == 0.0f ? 0.0f : (ls - t / s) * kLn2;
  if (out.stats != nullptr) {
    out.stats[2 * r] = o.m;
    out.stats[2 * r + 1] = ls;
  }
  return ls;
}

__device__ inline float best_value(uint32_t key, const Origin& o, float ls) {
  return key > kKeyOfMinusInf ? o.log_p(key_value(key), ls) : -INFINITY;
}

// A logit's key among the best classes: NaN is none of them.
__device__ inline uint32_t class_key(float v) { return v != v ? 0u : order_key(v); }

// The rows that fit the registers of L lanes, I pieces of 16 bytes each.  The
// next row's loads are under way while a row is summed.  100000 x 47 fp32, top 1:
// 8.5 us (2.6 TB/s; 5.9 where the logits are in cache), bound by latency.
template <typename T, int L, int I, bool Narrow>
__global__ __launch_bounds__(kThreads) void log_probs_rows(LogArgs a, const T* __restrict__ x,
                                                           const void* __restrict__ targets, RowOut out) {
  using Piece = RowPiece<T, Narrow>;
  constexpr int V = kPiece<T>, kGroups = kThreads / L;
  const int lane = threadIdx.x % L;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / L;
  if (r >= a.rows) return;
  piece_t<T> raw[I];
  int64_t target;
  float xt;
  auto column = [&](int i) { return static_cast<int64_t>(i * L + lane) * V; };
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < I; ++i) raw[i] = Piece::load(x + row * a.stride, column(i), a.classes);
    target = target_of(targets, a.index64, row);
    const bool named = static_cast<uint64_t>(target) < static_cast<uint64_t>(a.classes);
    xt = static_cast<float>(x[row * a.stride + (named ? target : 0)]);
  };
  fetch(r);
  for (; r < a.rows; r += step) {
    float v[I][V], m = -INFINITY, s = 0.0f, t = 0.0f;
    const int64_t mine = target;
    const float xm = xt;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int64_t first = Narrow ? 0 : Piece::shift(column(i), a.classes), count = Narrow ? a.classes - column(i) : V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = j >= first && j < count ? static_cast<float>(raw[i][j]) : -INFINITY;
        m = fmaxf(m, v[i][j]);
      }
    }
    if (r + step < a.rows) fetch(r + step);
    const Origin o(fmaxf(lane_max<L>(m), -FLT_MAX));
    auto add = [&](float y) {
      const float e = __builtin_amdgcn_exp2f(y);
      s += e;
      t = __builtin_fmaf(e, fmaxf(y, kFloor), t);
    };
    if (o.far) {
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) add((v[i][j] - o.m) * kLog2e);
    } else {
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) add(o.near(v[i][j]));
    }
    s = lane_sum<L>(s);
    t = lane_sum<L>(t);
    float ls = 0.0f;
    if (lane == 0) ls = finish_row(a, out, r, mine, xm, o, s, t);
    if (a.top == 0) continue;
    // Logits of 16 bits: the upper 19 bits of their order hold all of them, and 13 are left for the
    // index, so that a maximum finds both.  No two such keys are equal: the next one is the nearest
    // below the last, the greatest difference to it modulo 2^32 (from zero at first).
    constexpr bool kPacked = sizeof(T) == 2;
    constexpr uint32_t kFine = 0x1FFF;
    uint32_t key[I][V], best = 0;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        key[i][j] = class_key(v[i][j]);
        if constexpr (kPacked)
          key[i][j] = (key[i][j] & ~kFine) | (kFine - static_cast<uint32_t>(Piece::begin(column(i), a.classes) + j));
      }
#pragma unroll 1
    for (int q = 0; q < a.top; ++q) {
      uint32_t own = 0, win, value;
      if constexpr (kPacked) {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) own = key[i][j] - best > own ? key[i][j] - best : own;
        best += lane_max<L>(own);
        win = kFine - (best & kFine);
        value = (best & 0x80000000u) != 0 ? best & ~kFine : best | kFine;
      } else {
        uint32_t at = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) own = key[i][j] > own ? key[i][j] : own;
        // The greatest key, then the lowest index that has it.
        best = value = lane_max<L>(own);
#pragma unroll
        for (int i = I - 1; i >= 0; --i)
#pragma unroll
          for (int j = V - 1; j >= 0; --j)
            at = key[i][j] == best ? static_cast<uint32_t>(Piece::begin(column(i), a.classes)) + j : at;
        win = lane_min<L>(at);
#pragma unroll
        for (int i = 0; i < I; ++i) {
          const uint32_t j0 = win - static_cast<uint32_t>(Piece::begin(column(i), a.classes));
#pragma unroll
          for (int j = 0; j < V; ++j) key[i][j] = j0 == static_cast<uint32_t>(j) ? 0 : key[i][j];
        }
      }
      if (lane == 0) {
        out.top_values[r * a.top + q] = best_value(value, o, ls);
        out.top_ids[r * a.top + q] = value > kKeyOfMinusInf ? static_cast<int32_t>(win) : -1;
      }
    }
  }
}

// Best classes as (key, ~index): the greatest is the likeliest, ties by the
// lowest index.
__device__ inline uint64_t pair_of(uint32_t key, uint32_t index) {
  return (static_cast<uint64_t>(key) << 32) | (0xFFFFFFFFu - index);
}

template <int L>
__device__ inline uint64_t lane_max_pair(uint64_t p) {
  const uint32_t high = lane_max<L>(static_cast<uint32_t>(p >> 32));
  const uint32_t low = lane_max<L>(static_cast<uint32_t>(p >> 32) == high ? static_cast<uint32_t>(p) : 0u);
  return (static_cast<uint64_t>(high) << 32) | low;
}

struct Part {
  float m, s, t;
};

// y of one origin - y of another: 2^shift is the factor that takes sums from
// `from` to `to`, the shift what t takes besides.  Sums from far below vanish.  A
// far origin is m log2(e) itself, the others are c.
__device__ inline float origin_shift(const Origin& from, const Origin& to) {
  if (to.far) return from.far ? (from.m - to.m) * kLog2e : -from.near(to.m);
  return from.far ? to.near(from.m) : from.c - to.c;
}

// Wider rows: a work-group streams one part of a row, each thread with a
// running maximum and sums relative to it, and joins them at the end.
//
// The best classes cost the stream nothing: each thread's maximum is there
// anyway.  The top-th greatest of them is a bound that at least `top` logits
// reach, and only the threads whose maximum reaches it have such logits: their
// elements are read again (cache), some top * classes / threads of them, and
// those that reach the bound are ranked against each other.  Where more do than
// the buffer holds (many equal logits), the row is gone through once for each
// best class instead.
//
// 4096 x 131072 bf16, top 4: 197 us (5.5 TB/s), vector units 87% busy: the
// exponential, and six instructions more for each logit.  One such row: 6.4 us,
// and 4.5 of the join.  Rows far from zero are read a second time for their sums:
// 328 us for 168 with top 0.
constexpr int kCandidates = 1024;

template <typename T>
__global__ __launch_bounds__(kWideThreads) void log_probs_wide(LogArgs a, const T* __restrict__ x,
                                                               const void* __restrict__ targets, RowOut out, int parts,
                                                               Part* part_sums, uint64_t* part_best) {
  using Piece = RowPiece<T, false>;
  constexpr int V = kPiece<T>, W = kWideThreads / 64, U = 4;
  __shared__ float red[3][W];
  __shared__ uint32_t keys[kWideThreads];
  __shared__ uint64_t cand[kCandidates];
  __shared__ uint64_t best[kMaxTop];
  __shared__ uint32_t bound, reached, found;
  const int64_t r = blockIdx.x / static_cast<unsigned>(parts);
  const int part = blockIdx.x % static_cast<unsigned>(parts);
  const T* row = x + r * a.stride;
  const int64_t pieces = (a.classes + V - 1) / V, whole = a.classes / V;
  const int64_t p0 = pieces * part / parts, p1 = pieces * (part + 1) / parts;
  const int tid = threadIdx.x;

  // Sums relative to a maximum no lower than -kFar: logits far below it alone leave s zero.
  float m = -INFINITY, s = 0.0f, t = 0.0f;
  auto add = [&](auto N, const float (&v)[decltype(N)::value]) {
    float top = m;
#pragma unroll
    for (int j = 0; j < decltype(N)::value; ++j) top = fmaxf(top, v[j]);
    const float c = origin_of(top), shift = origin_of(m) - c;
    const float f = __builtin_amdgcn_exp2f(shift);
    t = f * __builtin_fmaf(s, fmaxf(shift, kFloor), t);
    s *= f;
    m = top;
#pragma unroll
    for (int j = 0; j < decltype(N)::value; ++j) {
      const float y = __builtin_fmaf(v[j], kLog2e, -c), e = __builtin_amdgcn_exp2f(y);
      s += e;
      t = __builtin_fmaf(e, fmaxf(y, kFloor), t);
    }
  };
  // take(N, v) for the part's logits, N at a time.
  auto stream = [&](auto take) {
    int64_t p = p0 + tid;
    const int64_t end = p1 < whole ? p1 : whole;
    for (; p + (U - 1) * kWideThreads < end; p += U * kWideThreads) {
      piece_t<T> raw[U];
      float v[U * V];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = Piece::template load<true>(row, (p + u * kWideThreads) * V, a.classes);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) v[u * V + j] = static_cast<float>(raw[u][j]);
      take(std::integral_constant<int, U * V>(), v);
    }
    for (; p < p1; p += kWideThreads) {
      const piece_t<T> raw = Piece::template load<true>(row, p * V, a.classes);
      const int first = Piece::shift(p * V, a.classes);
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = j >= first ? static_cast<float>(raw[j]) : -INFINITY;
      take(std::integral_constant<int, V>(), v);
    }
  };
  stream(add);

  const Origin o(fmaxf(block_max<W>(m, red[0]), -FLT_MAX));
  if (o.far) {
    s = t = 0.0f;
    stream([&](auto N, const float (&v)[decltype(N)::value]) {
#pragma unroll
      for (int j = 0; j < decltype(N)::value; ++j) {
        const float y = o(v[j]), e = __builtin_amdgcn_exp2f(y);
        s += e;
        t = __builtin_fmaf(e, fmaxf(y, kFloor), t);
      }
    });
  } else {
    const float shift = origin_of(m) - o.c, f = __builtin_amdgcn_exp2f(shift);
    t = f * __builtin_fmaf(s, fmaxf(shift, kFloor), t);
    s *= f;
  }
  s = lane_sum<64>(s);
  t = lane_sum<64>(t);
  if ((tid & 63) == 0) {
    red[1][tid >> 6] = s;
    red[2][tid >> 6] = t;
  }
  const uint32_t own_key = order_key(fmaxf(m, -FLT_MAX));
  keys[tid] = own_key;
  if (tid == 0) reached = found = 0;
  __syncthreads();
  s = t = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    s += red[1][w];
    t += red[2][w];
  }
  float ls = 0.0f;
  if (tid == 0) {
    if (parts > 1) {
      part_sums[blockIdx.x] = {o.m, s, t};
    } else {
      const int64_t target = target_of(targets, a.index64, r);
      const bool named = static_cast<uint64_t>(target) < static_cast<uint64_t>(a.classes);
      ls = finish_row(a, out, r, target, named ? static_cast<float>(row[target]) : 0.0f, o, s, t);
    }
  }
  if (a.top == 0) return;

  if (tid < 64) {  // the top-th greatest of the threads' maxima
    uint32_t mine[W];
#pragma unroll
    for (int w = 0; w < W; ++w) mine[w] = keys[w * 64 + tid];
    uint32_t limit = 0;
    for (int q = 0; q < a.top; ++q) {
      uint32_t own = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) own = mine[w] > own ? mine[w] : own;
      limit = lane_max<64>(own);
      const uint64_t has = __ballot(own == limit);
      if (tid == __builtin_ctzll(has)) {
        bool gone = false;
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (!gone && mine[w] == limit) {
            mine[w] = 0;
            gone = true;
          }
      }
    }
    if (tid == 0) bound = limit > kKeyOfMinusInf ? limit : kKeyOfMinusInf + 1;
  }
  __syncthreads();
  const uint32_t limit = bound;
  // A thread without a finite logit has its starting maximum for a key, which no logit is below:
  // at worst the bound is that, and all are candidates.
  uint32_t* list = keys;  // the maxima are read
  if (own_key >= limit) list[atomicAdd(&reached, 1u)] = tid;
  __syncthreads();
  const uint32_t lists = reached;
  for (uint32_t e = tid >> 6; e < lists; e += W) {
    const int64_t first = p0 + list[e];
    const int lane = tid & 63;
    for (int64_t q = first + static_cast<int64_t>(lane / V) * kWideThreads; q < p1; q += (64 / V) * kWideThreads) {
      const int64_t c = q * V + lane % V;
      if (c < a.classes) {
        const uint32_t key = class_key(static_cast<float>(row[c]));
        if (key >= limit) {
          const uint32_t at = atomicAdd(&found, 1u);
          if (at < kCandidates) cand[at] = pair_of(key, static_cast<uint32_t>(c));
        }
      }
    }
  }
  if (tid < kMaxTop) best[tid] = 0;
  __syncthreads();
  const uint32_t count = found;
  if (count <= kCandidates) {
    for (uint32_t c = tid; c < count; c += kWideThreads) {
      const uint64_t mine = cand[c];
      uint32_t rank = 0;
      for (uint32_t o = 0; o < count; ++o) rank += cand[o] > mine;
      if (rank < static_cast<uint32_t>(a.top)) best[rank] = mine;
    }
  } else {
    uint64_t last = ~uint64_t(0);
    for (int q = 0; q < a.top; ++q) {
      uint64_t mine = 0;
      for (int64_t c = p0 * V + tid; c < p1 * V && c < a.classes; c += kWideThreads) {
        const uint32_t key = class_key(static_cast<float>(row[c]));
        const uint64_t pair = pair_of(key, static_cast<uint32_t>(c));
        if (key > kKeyOfMinusInf && pair < last && pair > mine) mine = pair;
      }
      mine = lane_max_pair<64>(mine);
      __syncthreads();  // cand is free: readers of the last round are done
      if ((tid & 63) == 0) cand[tid >> 6] = mine;
      __syncthreads();
      mine = cand[0];
      for (int w = 1; w < W; ++w) mine = cand[w] > mine ? cand[w] : mine;
      if (tid == 0) best[q] = mine;
      if (mine == 0) break;
      last = mine;
    }
  }
  __syncthreads();
  if (tid >= 64) return;
  ls = as_float(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(as_bits(ls)))));
  if (tid < a.top) {
    const uint64_t pair = best[tid];
    if (parts > 1) {
      part_best[static_cast<int64_t>(blockIdx.x) * a.top + tid] = pair;
    } else {
      const uint32_t key = static_cast<uint32_t>(pair >> 32);
      out.top_values[r * a.top + tid] = best_value(key, o, ls);
      out.top_ids[r * a.top + tid] =
          key > kKeyOfMinusInf ? static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(pair)) : -1;
    }
  }
}

// Joins a row's parts: one wave a row, a lane a part.  Each part's best classes
// are in order, so the row's are taken from the heads of the lists.
template <typename T>
__global__ __launch_bounds__(64) void log_probs_join(LogArgs a, const T* __restrict__ x,
                                                     const void* __restrict__ targets, RowOut out, int parts,
                                                     const Part* __restrict__ part_sums,
                                                     const uint64_t* __restrict__ part_best) {
  extern __shared__ uint64_t heads[];  // the parts' lists
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x;
  for (int k = lane; k < parts * a.top; k += 64) heads[k] = part_best[r * parts * a.top + k];
  const int64_t target = target_of(targets, a.index64, r);
  const bool named = static_cast<uint64_t>(target) < static_cast<uint64_t>(a.classes);
  const float xt = named ? static_cast<float>(x[r * a.stride + target]) : 0.0f;
  Part mine = {-FLT_MAX, 0.0f, 0.0f};
  if (lane < parts) mine = part_sums[r * parts + lane];
  __syncthreads();
  int taken = 0;
  uint64_t head = lane < parts && a.top > 0 ? heads[lane * a.top] : 0;
  const Origin o(lane_max<64>(mine.m));
  const float shift = origin_shift(Origin(mine.m), o), f = __builtin_amdgcn_exp2f(shift);
  const float t = lane_sum<64>(f * __builtin_fmaf(mine.s, fmaxf(shift, kFloor), mine.t)), s = lane_sum<64>(mine.s * f);
  float ls = 0.0f;
  if (lane == 0) ls = finish_row(a, out, r, target, xt, o, s, t);
  for (int q = 0; q < a.top; ++q) {
    const uint64_t pair = lane_max_pair<64>(head);
    if (lane == 0) {
      const uint32_t key = static_cast<uint32_t>(pair >> 32);
      out.top_values[r * a.top + q] = best_value(key, o, ls);
      out.top_ids[r * a.top + q] =
          key > kKeyOfMinusInf ? static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(pair)) : -1;
    }
    // Pairs differ by their index: one lane at most has this one, but for the empty pair.
    if (head == pair && pair != 0) head = ++taken < a.top ? heads[lane * a.top + taken] : 0;
  }
}

// dlogits, each group of L lanes (256: the work-group) walking the pieces
// [p0, p1) of a row; rows over blockIdx.x, parts of a row over blockIdx.y.  Bound
// by memory: 4096 x 131072 bf16 396 us (5.4 TB/s), 100000 x 47 fp32 11.0 (3.4).
template <typename T, int L, bool Narrow>
__global__ __launch_bounds__(kThreads) void log_probs_grad(LogArgs a, const T* __restrict__ x,
                                                           const void* __restrict__ targets,
                                                           const float* __restrict__ stats,
                                                           const float* __restrict__ entropy,
                                                           const float* __restrict__ grad_logp,
                                                           const float* __restrict__ grad_entropy,
                                                           T* __restrict__ dx) {
  using Piece = RowPiece<T, Narrow>;
  constexpr int V = kPiece<T>, kGroups = kThreads / L, U = L == 256 ? 4 : 1;
  const int lane = threadIdx.x % L;
  const int64_t pieces = (a.classes + V - 1) / V, step = static_cast<int64_t>(gridDim.x) * kGroups;
  const int64_t p0 = pieces * blockIdx.y / gridDim.y, p1 = pieces * (blockIdx.y + 1) / gridDim.y;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / L; r < a.rows; r += step) {
    const int64_t target = target_of(targets, a.index64, r);
    const Origin o(stats[2 * r]);
    const float ls = stats[2 * r + 1];
    const bool named = static_cast<uint64_t>(target) < static_cast<uint64_t>(a.classes) && ls != INFINITY;
    const float ga = named && grad_logp != nullptr ? grad_logp[r] : 0.0f;
    const float gh = grad_entropy != nullptr ? grad_entropy[r] : 0.0f;
    // -(a + h (log p + H)), with log p in powers of two.
    const float factor = -gh * kLn2, rest = -__builtin_fmaf(gh, entropy[r], ga);
    const T* row = x + r * a.stride;
    T* out = dx + r * a.classes;
    auto walk = [&](auto y) {
      auto piece = [&](int64_t p, const piece_t<T>& raw) {
        const int64_t c = Piece::begin(p * V, a.classes);
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float lp = y(static_cast<float>(raw[j])) - ls;
          v[j] = __builtin_amdgcn_exp2f(lp) * __builtin_fmaf(factor, fmaxf(lp, kFloor), rest);
        }
        if (static_cast<uint64_t>(target - c) < V)
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] += c + j == target ? ga : 0.0f;
        Piece::template store<(L == 256)>(out, p * V, a.classes, v);
      };
      int64_t p = p0 + lane;
      for (; p + (U - 1) * L < p1; p += U * L) {
        piece_t<T> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = Piece::template load<(L == 256)>(row, (p + u * L) * V, a.classes);
#pragma unroll
        for (int u = 0; u < U; ++u) piece(p + u * L, raw[u]);
      }
      for (; p < p1; p += L) piece(p, Piece::load(row, p * V, a.classes));
    };
    if (o.far) walk([&](float v) { return (v - o.m) * kLog2e; });
    else walk([&](float v) { return o.near(v); });
  }
}

spmm_status check_log_desc(const spmm_log_probs_desc* d) {
  if (d == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null descriptor");
  if (!dense_type(d->value_type))
    return fail(SPMM_ERR_CONTRACT, "log_probs supports only FP16, BF16 and FP32 tensors");
  if (d->index_type != SPMM_INDEX_I32 && d->index_type != SPMM_INDEX_I64)
    return fail(SPMM_ERR_CONTRACT, "log_probs: targets must be int32 or int64");
  if (d->rows < 0 || d->rows > INT32_MAX)
    return fail(SPMM_ERR_CONTRACT,
                "log_probs: rows must be at least 0 and below 2^31, but got " + std::to_string(d->rows));
  if (d->classes < 1 || d->classes > INT32_MAX)
    return fail(SPMM_ERR_CONTRACT, "log_probs requires 1 <= classes < 2^31, but got " + std::to_string(d->classes));
  if (d->rows > 1 && d->logits_stride < d->classes)
    return fail(SPMM_ERR_CONTRACT, "log_probs: rows of logits overlap");
  if (d->top < 0 || d->top > kMaxTop || d->top > d->classes)
    return fail(SPMM_ERR_INVALID_ARGUMENT,
                "log_probs: top must be at least 0, at most 64 and at most the classes, but got " +
                    std::to_string(d->top));
  return SPMM_OK;
}

LogArgs log_args(const spmm_log_probs_desc* d) {
  return {d->rows, d->classes, d->logits_stride, static_cast<int32_t>(d->top), d->index_type == SPMM_INDEX_I64};
}

// f(L, I, Narrow) for rows that a wave's registers hold; false where they are
// wider.  Four pieces a lane, so that what a row does once is shared by more rows
// of a wave, where there are rows for four waves a CU all the same; else the most
// lanes (100000 x 47 fp32, top 1: 5.9 us against 9.7; 64 x 1000 bf16, top 5: 6.5
// against 4.7).
template <typename T, typename F>
bool with_lanes(int64_t rows, int64_t classes, F f) {
  const int64_t pieces = ceil_div(classes, kPiece<T>);
  if (classes < kPiece<T>)
    return f(std::integral_constant<int, 2>(), std::integral_constant<int, 1>(), std::true_type()), true;
#define SPMM_TILE(L, I) \
  if (pieces <= (L) * (I) && (I == 1 || L == 64 || rows * (L) >= 64 * 1024)) \
  return f(std::integral_constant<int, L>(), std::integral_constant<int, I>(), std::false_type()), true
  SPMM_TILE(2, 1);
  SPMM_TILE(4, 1);
  SPMM_TILE(4, 2);
  SPMM_TILE(4, 3);
  SPMM_TILE(4, 4);
  SPMM_TILE(8, 4);
  SPMM_TILE(16, 4);
  SPMM_TILE(32, 4);
  SPMM_TILE(8, 1);
  SPMM_TILE(16, 1);
  SPMM_TILE(32, 1);
  SPMM_TILE(64, 1);
  SPMM_TILE(64, 2);
  SPMM_TILE(64, 4);
#undef SPMM_TILE
  return false;
}

bool in_registers(const spmm_log_probs_desc* d) {
  return ceil_div(d->classes, 16 / dense_type_bytes(d->value_type)) <= 256;
}

// Parts of a row: as many as give the chip four work-groups a CU, each with a
// piece for every thread at least.
int row_parts(const spmm_log_probs_desc* d) {
  const int64_t pieces = ceil_div(d->classes, 16 / dense_type_bytes(d->value_type));
  int64_t parts = d->rows > 0 ? 1024 / d->rows : 1;
  if (parts > pieces / kWideThreads) parts = pieces / kWideThreads;
  if (parts > kMaxParts) parts = kMaxParts;
  return static_cast<int>(parts < 1 ? 1 : parts);
}

size_t part_sums_bytes(const spmm_log_probs_desc* d, int parts) {
  return align_up(static_cast<size_t>(d->rows) * parts * sizeof(Part), 256);
}

size_t log_workspace(const spmm_log_probs_desc* d) {
  if (in_registers(d) || d->rows == 0) return 0;
  const int parts = row_parts(d);
  if (parts == 1) return 0;
  return part_sums_bytes(d, parts) + static_cast<size_t>(d->rows) * parts * d->top * sizeof(uint64_t);
}

// A launch has fewer than 2^32 work-items: so many wide rows go into one.
constexpr int64_t kWideRows = int64_t(1) << 22;

template <typename T>
spmm_status run_forward(const spmm_log_probs_desc* d, const void* logits, const void* targets, const RowOut& out,
                        void* workspace, hipStream_t s) {
  LogArgs a = log_args(d);
  const T* x = static_cast<const T*>(logits);
  const bool held = with_lanes<T>(d->rows, d->classes, [&](auto L, auto I, auto Narrow) {
    const int64_t blocks = ceil_div(d->rows, kThreads / decltype(L)::value);
    hipLaunchKernelGGL((log_probs_rows<T, decltype(L)::value, decltype(I)::value, decltype(Narrow)::value>),
                       dim3(static_cast<unsigned>(blocks < 2048 ? blocks : 2048)), dim3(kThreads), 0, s, a, x, targets,
                       out);
  });
  if (held) return check_launch("log_probs");
  const int parts = row_parts(d);
  Part* sums = static_cast<Part*>(workspace);
  uint64_t* best = parts > 1 ? reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + part_sums_bytes(d, parts))
                             : nullptr;
  for (int64_t r = 0; r < d->rows; r += kWideRows) {
    a.rows = d->rows - r < kWideRows ? d->rows - r : kWideRows;
    const RowOut part = {out.logp + r, out.entropy + r, out.top_values + r * a.top, out.top_ids + r * a.top,
                         out.stats == nullptr ? nullptr : out.stats + 2 * r};
    hipLaunchKernelGGL(log_probs_wide<T>, dim3(static_cast<unsigned>(a.rows * parts)), dim3(kWideThreads), 0, s, a,
                       x + r * a.stride, static_cast<const char*>(targets) + r * (a.index64 ? 8 : 4), part, parts,
                       sums, best);
    if (spmm_status st = check_launch("log_probs")) return st;
  }
  if (parts == 1) return SPMM_OK;
  hipLaunchKernelGGL(log_probs_join<T>, dim3(static_cast<unsigned>(d->rows)), dim3(64),
                     static_cast<size_t>(parts) * a.top * sizeof(uint64_t), s, a, x, targets, out, parts, sums, best);
  return check_launch("log_probs join");
}

template <typename T>
spmm_status run_backward(const spmm_log_probs_desc* d, const void* logits, const void* targets, const float* stats,
                         const float* entropy, const float* grad_logp, const float* grad_entropy, void* dlogits,
                         hipStream_t s) {
  const LogArgs a = log_args(d);
  const int64_t pieces = ceil_div(d->classes, kPiece<T>);
  auto launch = [&](auto L, auto Narrow) {
    constexpr int kGroups = kThreads / decltype(L)::value;
    int64_t blocks = ceil_div(d->rows, kGroups);
    // Few rows: in parts of four pieces a lane or more.
    int64_t parts = blocks < 2048 ? ceil_div(2048, blocks) : 1;
    const int64_t most = ceil_div(pieces, 4 * decltype(L)::value);
    if (parts > most) parts = most;
    if (blocks > 65536) blocks = 65536;
    hipLaunchKernelGGL((log_probs_grad<T, decltype(L)::value, decltype(Narrow)::value>),
                       dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(parts)), dim3(kThreads), 0, s, a,
                       static_cast<const T*>(logits), targets, stats, entropy, grad_logp, grad_entropy,
                       static_cast<T*>(dlogits));
  };
  if (d->classes < kPiece<T>) launch(std::integral_constant<int, 4>(), std::true_type());
  else if (pieces <= 4) launch(std::integral_constant<int, 4>(), std::false_type());
  else if (pieces <= 16) launch(std::integral_constant<int, 16>(), std::false_type());
  else if (pieces <= 256) launch(std::integral_constant<int, 64>(), std::false_type());
  else launch(std::integral_constant<int, 256>(), std::false_type());
  return check_launch("log_probs_grad");
}

}  // namespace
}  // namespace spmm

using namespace spmm;

extern "C" {

spmm_status spmm_log_probs_workspace(const spmm_log_probs_desc* d, size_t* bytes) {
  clear_error();
  if (bytes == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null argument");
  if (spmm_status st = check_log_desc(d)) return st;
  *bytes = log_workspace(d);
  return SPMM_OK;
}

spmm_status spmm_log_probs_run(const spmm_log_probs_desc* d, const void* logits, const void* targets, float* logp,
                               float* entropy, float* top_values, int32_t* top_ids, float* stats, void* workspace,
                               size_t workspace_bytes, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_log_desc(d)) return st;
  if (d->rows == 0) return SPMM_OK;
  if (logits == nullptr || targets == nullptr || logp == nullptr || entropy == nullptr ||
      (d->top > 0 && (top_values == nullptr || top_ids == nullptr)))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "log_probs: null device pointer");
  const size_t need = log_workspace(d);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(SPMM_ERR_CONTRACT, "log_probs: workspace too small: need " + std::to_string(need) + " bytes");
  const RowOut out = {logp, entropy, top_values, top_ids, stats};
  hipStream_t s = as_stream(stream);
  switch (d->value_type) {
    case SPMM_VALUE_F16: return run_forward<_Float16>(d, logits, targets, out, workspace, s);
    case SPMM_VALUE_BF16: return run_forward<__bf16>(d, logits, targets, out, workspace, s);
    default: return run_forward<float>(d, logits, targets, out, workspace, s);
  }
}

spmm_status spmm_log_probs_grad_run(const spmm_log_probs_desc* d, const void* logits, const void* targets,
                                    const float* stats, const float* entropy, const float* grad_logp,
                                    const float* grad_entropy, void* dlogits, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_log_desc(d)) return st;
  if (d->rows == 0) return SPMM_OK;
  if (logits == nullptr || targets == nullptr || stats == nullptr || entropy == nullptr || dlogits == nullptr)
    return fail(SPMM_ERR_INVALID_ARGUMENT, "log_probs: null device pointer");
  hipStream_t s = as_stream(stream);
  switch (d->value_type) {
    case SPMM_VALUE_F16:
      return run_backward<_Float16>(d, logits, targets, stats, entropy, grad_logp, grad_entropy, dlogits, s);
    case SPMM_VALUE_BF16:
      return run_backward<__bf16>(d, logits, targets, stats, entropy, grad_logp, grad_entropy, dlogits, s);
    default: return run_backward<float>(d, logits, targets, stats, entropy, grad_logp, grad_entropy, dlogits, s);
  }
}

}  // extern "C"
