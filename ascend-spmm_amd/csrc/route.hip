// Routing of rows to experts from a router's logits.
//
// With l_i the log score of expert i, x_i - log sum e^x (softmax) or
// -log(1 + e^-x_i) (sigmoid), the k chosen experts are those of the greatest
// selection values e^l_i + bias_i, and their weights are
//   w_j = scale * e^l_j,  or  scale * e^l_j / sum over the chosen of e^l
// where they are renormalised (computed as a softmax over the chosen l, which
// neither overflows nor divides zero by zero).  Gradient, with u_j = w_j g_j:
//   dl_j = u_j,  or  w_j (g_j - sum u / scale);
//   dx_i = dl_i - p_i sum dl  (softmax; p drops out where dl sums to zero, as it
//   does renormalised),  dx_i = dl_i / (1 + e^x_i)  (sigmoid).
//
// Which experts are chosen is decided without rounding that could turn a close
// pair: by the logits themselves where there is neither a bias nor groups (the
// scores grow with them), else by values in 64 bits.
#include <cfloat>
#include <cmath>

#include "lane_reduce.h"
#include "row_pieces.h"

namespace spmm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxExperts = 1024, kMaxTopK = 64, kMaxGroups = 64;

struct RouteArgs {
  int64_t rows, stride;
  int32_t experts, k, groups, top_groups;
  float scale;
  bool sigmoid, renormalize;
};

__device__ inline float log_sigmoid(float x) { return fminf(x, 0.0f) - log1pf(expf(-fabsf(x))); }

// Order of doubles and floats as whole numbers; NaN above all, so that it is
// chosen and seen, and zero below all, for what is taken.
__device__ inline uint64_t key_of(double v) {
  if (v != v) return ~uint64_t(0);
  const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
  return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}
__device__ inline uint32_t key_of(float v) { return v != v ? 0xFFFFFFFFu : order_key(v); }
constexpr uint64_t kWideMinusInf = 0x000FFFFFFFFFFFFFull;
constexpr double kInf64 = __builtin_huge_val();
constexpr float kLog2e = 1.44269504088896340736f;

template <int L>
__device__ inline uint32_t best_index(uint64_t own, uint32_t at, uint64_t& best) {
  const uint32_t high = lane_max<L>(static_cast<uint32_t>(own >> 32));
  const uint32_t low = lane_max<L>(static_cast<uint32_t>(own >> 32) == high ? static_cast<uint32_t>(own) : 0u);
  best = (static_cast<uint64_t>(high) << 32) | low;
  return lane_min<L>(own == best ? at : 0xFFFFFFFFu);
}

// The two greatest values.
template <typename F>
struct BestTwo {
  F first, second;
  bool nan;
  __device__ inline void add(F a, F b) {  // a >= b
    second = fmax(fmin(first, a), fmax(second, b));
    first = fmax(first, a);
  }
};

// What the lanes of a row share when they look for its open groups: evenly many
// lanes a group, each of which looks through a part of it.
template <int L>
struct GroupLanes {
  int shift, each, group, size;  // each: 2^shift
  __device__ inline explicit GroupLanes(const RouteArgs& a) : shift(0), size(a.experts / a.groups) {
    while ((2 << shift) * a.groups <= L) ++shift;
    each = 1 << shift;
    group = threadIdx.x % L >> shift;
  }
  template <typename F>
  __device__ inline BestTwo<F> best(const RouteArgs& a, const F* values) const {
    const F none = -static_cast<F>(INFINITY);
    BestTwo<F> b = {none, none, false};
    if (group < a.groups)
      for (int e = threadIdx.x % each; e < size; e += each) {
        const F v = values[group * size + e];
        b.nan |= v != v;
        b.add(v, none);
      }
    for (int d = 1; d < each; d <<= 1) {
      const F first = __shfl_xor(b.first, d, L), second = __shfl_xor(b.second, d, L);
      b.nan |= __shfl_xor(static_cast<int>(b.nan), d, L) != 0;
      b.add(first, second);
    }
    return b;
  }
  // The same of groups of whole pieces of four, in aligned LDS, but for a NaN only
  // its own lane knows of.  Groups start at different pieces, so that their lanes
  // read different banks: 65536 x 256 in 8 groups 40.0 us, 46.7 as above.
  __device__ inline BestTwo<float> best_of_pieces(const RouteArgs& a, const float* values) const {
    BestTwo<float> b = {-INFINITY, -INFINITY, false};
    const int first = threadIdx.x & (each - 1), pieces = size / 4, n = (pieces - first + each - 1) >> shift;
    if (group < a.groups) {
      int t = group * pieces >> 4;
      t = t < n ? t : 0;
      for (int u = 0; u < n; ++u) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(values + group * size + 4 * (first + (t << shift)));
        t = t + 1 < n ? t + 1 : 0;
        b.nan |= __builtin_isunordered(v[0], v[1]) || __builtin_isunordered(v[2], v[3]);
        b.add(fmaxf(v[0], v[1]), fminf(v[0], v[1]));
        b.add(fmaxf(v[2], v[3]), fminf(v[2], v[3]));
      }
    }
    if (each > 1) join<1>(b);
    if (each > 2) join<2>(b);
    if (each > 4) join<4>(b);
    if (each > 8) join<8>(b);
    if (each > 16) join<16>(b);
    if (each > 32) join<32>(b);
    return b;
  }
  template <int D>
  __device__ static inline void join(BestTwo<float>& b) {
    uint32_t mine[2], other[2];
    reduce_step<D>(as_bits(b.first), [&](uint32_t x, uint32_t y) { return mine[0] = x, other[0] = y, x; });
    reduce_step<D>(as_bits(b.second), [&](uint32_t x, uint32_t y) { return mine[1] = x, other[1] = y, x; });
    b.first = as_float(mine[0]);
    b.second = as_float(mine[1]);
    b.add(as_float(other[0]), as_float(other[1]));
  }
  // A bit for each lane of the row, from its group's answer; of one group; the first with a bit.
  __device__ inline uint64_t bits(const RouteArgs& a, bool open) const {
    return __ballot(group < a.groups && open) >> (threadIdx.x & 63 & ~(L - 1)) & (~uint64_t(0) >> (64 - L));
  }
  __device__ inline bool has(uint64_t bits, int g) const { return (bits >> (g << shift & 63)) & 1u; }
  __device__ inline int first(uint64_t bits) const { return bits != 0 ? __builtin_ctzll(bits) >> shift : 0; }
};

// Exact choice of one row by a wave, in 64 bits: for rows whose choice 32 bits do
// not decide, about one in 2000 of random logits with biases of the scores' size,
// and nearly all where a bias is far beyond them or all values are equal (the
// kernel's 42 us below are 182 then).  It takes the row's logits and leaves
// ids[0..k) (-1 where no expert is left); values: `experts` doubles of the wave's
// own LDS.  Returns whether a softmax's values are no numbers, as a NaN or an
// infinity is among its logits.
template <typename T>
__device__ inline bool choose_exactly(const RouteArgs& a, const T* row, const float* bias, double* values,
                                      int32_t* ids) {
  constexpr int L = 64;
  const int lane = threadIdx.x % L;
  double m = -kInf64, total = 0.0;
  if (!a.sigmoid) {
#pragma unroll 4
    for (int e = lane; e < a.experts; e += L) m = fmax(m, static_cast<double>(static_cast<float>(row[e])));
    for (int d = 1; d < L; d <<= 1) m = fmax(m, __shfl_xor(m, d, L));
#pragma unroll 4
    for (int e = lane; e < a.experts; e += L) {
      const float x = static_cast<float>(row[e]);
      if (x != -INFINITY) total += exp(static_cast<double>(x) - m);
    }
    for (int d = 1; d < L; d <<= 1) total += __shfl_xor(total, d, L);
  }
#pragma unroll 4
  for (int e = lane; e < a.experts; e += L) {
    const float x = static_cast<float>(row[e]), b = bias != nullptr ? bias[e] : 0.0f;
    const double score = a.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(x)))
                                   : exp(static_cast<double>(x) - m) / total;
    values[e] = x == -INFINITY || b == -INFINITY ? -kInf64 : score + b;
  }
  // A wave's LDS accesses are performed in order.
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (a.groups > 1) {
    const GroupLanes<L> lanes(a);
    const BestTwo<double> best = lanes.best(a, values);
    const double sum = best.second == -kInf64 ? best.first : best.first + best.second;
    const uint64_t key = best.nan ? ~uint64_t(0) : key_of(sum);
    int rank = 0;
    for (int o = 0; o < a.groups; ++o) {
      const uint64_t other = __shfl(key, o * lanes.each, L);
      rank += other > key || (other == key && o < lanes.group);
    }
    const uint64_t open = lanes.bits(a, rank < a.top_groups);
#pragma unroll 4
    for (int e = lane; e < a.experts; e += L)
      if (!lanes.has(open, e / lanes.size)) values[e] = -kInf64;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
#pragma unroll 1
  for (int q = 0; q < a.k; ++q) {
    uint64_t own = 0, best;
    uint32_t at = 0xFFFFFFFFu;
#pragma unroll 4
    for (int e = lane; e < a.experts; e += L) {
      const uint64_t key = key_of(values[e]);
      if (key > own) {
        own = key;
        at = e;
      }
    }
    const uint32_t win = best_index<L>(own, at, best);
    if (lane == 0) ids[q] = best > kWideMinusInf ? static_cast<int32_t>(win) : -1;
    if (best > kWideMinusInf && win % L == static_cast<uint32_t>(lane)) values[win] = -kInf64;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return total != total;
}

// How far apart two selection values in 32 bits have to be for their order to be
// the exact one.  With e = 2^-24: y = x log2(e) is off by 1.25 |x| e (in units of
// log e), 2^y by 2 e more.  A sigmoid 1 / (1 + 2^y) is then off by s (1 - s) times
// that, 0.8 e at most, and by 3 e for its two roundings.  A softmax's sum of up to
// 1024 terms is off by 1.25 sum p |z| e + 24 e, below 32 e; its logarithm, of up
// to 10, by 11 e; p = 2^(y - log2 s) in all by (52 + 2.25 |z|) e of itself, with
// p |z| < 0.4.  A value with its bias rounds by e times the row's greatest value.
// Two values: twice that.  Two sums of two: a softmax's four scores are at most 1
// together, and there are three roundings more.
__device__ inline float pair_margin(bool sigmoid, float scores, float most) {
  return (sigmoid ? 0x1p-20f : 0x1p-18f * scores) + 0x1p-22f * most;
}
__device__ inline float group_margin(bool sigmoid, float most) {
  return (sigmoid ? 0x1p-19f : 0x1p-18f) + 0x1p-20f * most;
}

// Rows of whole pieces; rows whose last piece is moved back to end with them;
// rows narrower than a piece.
enum class RowShape { kWhole, kMoved, kNarrow };

// The keys in which a row's best are found, the greatest first and of equal ones
// the lowest index.  kPacked: value and index in one word, so that a maximum
// finds both.
//  - logits of 16 bits: the upper 19 bits of their order hold all of them, 13 are
//    left for the index;
//  - values with a bias: steps of 2^-22 of the row's range (which the
//    check of neighbours counts in), and 10 bits for the index.
// Logits of 32 bits without a bias take a word for the value alone, and the index
// is looked for.
constexpr uint32_t kFine = 0x1FFF, kCoarse = 0x3FF;
constexpr float kSteps = 4194300.0f;  // below 2^22
constexpr float kLargest = 1e38f;     // of a value in 32 bits: two of them add up to a finite one
constexpr float kFar = 0x1p20f;       // of a logit that a softmax in 32 bits starts from

// L lanes a row, which hold I pieces of 16 bytes of it each.  The k best are taken
// one after another.  Without a bias the logits are the keys, and exact.  With one
// (Biased) the keys are selection values in 32 bits, and two more than k are
// taken: where neighbours among them are closer than pair_margin, and not of the
// same logit and bias, or the groups at the border are as close, the row's choice
// is made again in 64 bits.  In groups without a bias the keys are the logits, and
// 64 bits decide where two that differ may have the same score.  Bound by vector
// instructions, most of them of the k rounds.  65536 rows of 256 fp32 logits in 8
// groups, bias, k = 8: 42 to 45 us (1.6 TB/s, vector units always busy); all in 64
// bits 132, one wave a row 233, value and index apart 113.
template <typename T, int L, int I, RowShape Shape, bool Biased, bool Grouped>
__global__ __launch_bounds__(kThreads, 4) void route_rows(RouteArgs a, const T* __restrict__ logits,
                                                          const float* __restrict__ bias, float* __restrict__ weights,
                                                          int32_t* __restrict__ chosen, float* stats) {
  constexpr bool Narrow = Shape == RowShape::kNarrow, Whole = Shape == RowShape::kWhole;
  using Piece = RowPiece<T, Narrow>;
  constexpr int V = kPiece<T>, kGroups = kThreads / L;
  constexpr bool kChecked = Biased || Grouped, kPacked = Biased || sizeof(T) == 2;
  constexpr uint32_t kIndex = Biased ? kCoarse : kFine, kNone = Biased ? kCoarse : kKeyOfMinusInf;
  extern __shared__ __align__(16) double lds[];  // read as pieces of 16 bytes too
  // 64-bit values for one row of each wave; the row's own values where there are groups; its choices' ids and scores.
  double* exact = lds + (threadIdx.x >> 6) * a.experts;
  float* all_values = reinterpret_cast<float*>(lds + (kChecked ? kThreads / 64 * a.experts : 0));
  const int per_row = Grouped ? (a.experts + 3) / 4 * 4 : 0;
  float* values = all_values + (threadIdx.x / L) * per_row;
  int32_t* all_ids = reinterpret_cast<int32_t*>(all_values + kGroups * per_row);
  int32_t* ids = all_ids + (threadIdx.x / L) * (2 * a.k + 2);
  float* scores = reinterpret_cast<float*>(ids + a.k + 2);
  const int lane = threadIdx.x % L;
  int begin[I], first[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int column = (i * L + lane) * V;
    begin[i] = Whole ? column : static_cast<int>(Piece::begin(column, a.experts));
    // Elements before it are another piece's, or past the row.
    first[i] = Narrow ? 0 : Whole ? (column < a.experts ? 0 : V) : Piece::shift(column, a.experts);
  }
  const int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / L;
  const bool live = r < a.rows;  // lanes without a row go along with the last one
  const T* row = logits + (live ? r : a.rows - 1) * a.stride;
  float x[I][V], m = -FLT_MAX, ls = 0.0f, c = 0.0f, l2s = 0.0f;
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const piece_t<T> raw = Piece::load(row, (i * L + lane) * V, a.experts);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool in = Whole ? first[i] == 0 : j >= first[i] && (!Narrow || begin[i] + j < a.experts);
      x[i][j] = in ? static_cast<float>(raw[j]) : -INFINITY;
      m = fmaxf(m, x[i][j]);
    }
  }
  if (!a.sigmoid && (kChecked || !a.renormalize)) m = lane_max<L>(m);
  if (!a.sigmoid && !a.renormalize) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s += expf(x[i][j] - m);
    ls = logf(lane_sum<L>(s));
  }
  bool close = false;
  if (kChecked && !a.sigmoid) {
    float s = 0.0f;
    c = m * kLog2e;
    // 64 bits decide where c is rounded by more than 2^-4.  (Of -FLT_MAX, which is also the maximum
    // of a row without any expert, the scores are NaN, which no check below lets pass.)
    close = !(fabsf(m) <= kFar) && m > -FLT_MAX;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s += __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][j], kLog2e, -c));
    l2s = __builtin_amdgcn_logf(lane_sum<L>(s));
  }
  // A score in 32 bits: of the choice alone, not of the weights.
  auto sigmoid = [&](float v) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v * kLog2e)); };
  auto softmax = [&](float v) { return __builtin_amdgcn_exp2f(__builtin_fmaf(v, kLog2e, -c) - l2s); };
  auto score = [&](float v) { return a.sigmoid ? sigmoid(v) : softmax(v); };
  auto selected = [&](float s, float v, float b) { return v == -INFINITY || b == -INFINITY ? -INFINITY : s + b; };
  float v[I][V], least = INFINITY, most = -INFINITY;
  float seen = 0.0f;
  if constexpr (Biased) {
    float b[I][V];
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        if constexpr (Narrow) {
#pragma unroll
          for (int u = 0; u < 4; ++u) b[i][j + u] = bias[begin[i] + j + u < a.experts ? begin[i] + j + u : 0];
        } else {
          const float* from = bias + (Whole && first[i] != 0 ? 0 : begin[i]) + j;
          const piece_t<float> four = *reinterpret_cast<const piece_t<float>*>(from);
#pragma unroll
          for (int u = 0; u < 4; ++u) b[i][j + u] = four[u];
        }
      }
    if (a.sigmoid) {
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = sigmoid(x[i][j]);
    } else {
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = softmax(x[i][j]);
    }
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const float one = v[i][j] + b[i][j], two = v[i][j + 1] + b[i][j + 1];
        // Of experts without a logit too: their score is zero, which widens the range at worst.
        least = fminf(fminf(least, one), two);
        most = fmaxf(fmaxf(most, one), two);
        close |= __builtin_isunordered(one, two);
        v[i][j] = x[i][j] == -INFINITY ? -INFINITY : one;
        v[i][j + 1] = x[i][j + 1] == -INFINITY ? -INFINITY : two;
      }
  } else {
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = x[i][j];
  }
  uint32_t key[I][V];
  float step_of_key = 0.0f, largest = 1.0f;  // the row's greatest value by size
  if constexpr (Biased) {
    least = lane_min_value<L>(least);
    most = lane_max<L>(most);
    if (__ballot(least == -INFINITY) != 0) {  // of a bias
      least = INFINITY;
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) least = fminf(least, v[i][j] == -INFINITY ? INFINITY : v[i][j]);
      least = lane_min_value<L>(least);
    }
    largest = fmaxf(fabsf(least), fabsf(most));
    // Greater values' range, or the sum of two, may overflow: 64 bits decide.
    close |= !(largest <= kLargest);
    const float range = most - least, steps = range > 0.0f ? kSteps / range : 0.0f;
    step_of_key = range > 0.0f ? range / kSteps : 0.0f;
    // A range so small that this overflows has no keys.
    close |= !(steps <= FLT_MAX);
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // From 1 on; 0, and so a key that counts as none, for -inf.
        const uint32_t place = static_cast<uint32_t>(fmaxf(__builtin_fmaf(v[i][j] - least, steps, 1.0f), 0.0f));
        key[i][j] = (place << 10) | (kCoarse - (begin[i] + j));
      }
  } else {
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        key[i][j] = key_of(v[i][j]);
        if constexpr (kPacked) key[i][j] = (key[i][j] & ~kFine) | (kFine - (begin[i] + j));
      }
  }
  if constexpr (Grouped) {
    const int size = a.experts / a.groups;
    if constexpr (Whole) {
#pragma unroll
      for (int i = 0; i < I; ++i)
        if (first[i] == 0)
#pragma unroll
          for (int j = 0; j < V; j += 4)
            *reinterpret_cast<f32x4*>(values + begin[i] + j) = f32x4{v[i][j], v[i][j + 1], v[i][j + 2], v[i][j + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j >= first[i] && begin[i] + j < a.experts) values[begin[i] + j] = v[i][j];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const GroupLanes<L> lanes(a);
    const BestTwo<float> best = size % 4 == 0 ? lanes.best_of_pieces(a, values) : lanes.best(a, values);
    close |= best.nan;
    // Without a bias the two best logits have the two best scores.
    const float one = Biased || best.first == -INFINITY ? best.first : score(best.first);
    const float two = best.second == -INFINITY ? 0.0f : Biased ? best.second : score(best.second);
    const float sum = one == -INFINITY ? -INFINITY : one + two;
    // The sums take the place of the values.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lanes.group < a.groups && lane % lanes.each == 0) values[lanes.group] = sum;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    int rank = 0;
    for (int o = 0; o < a.groups; ++o) {
      const float other = values[o];
      rank += other > sum || (other == sum && o < lanes.group);
    }
    const uint64_t open = lanes.bits(a, rank < a.top_groups);
    if (a.top_groups < a.groups) {
      // The last open group and the first closed one: ranks differ, unless a sum is no number.
      const int g = lanes.first(lanes.bits(a, rank == a.top_groups - 1));
      const int h = lanes.first(lanes.bits(a, rank == a.top_groups));
      const bool same = !Biased && __shfl(best.first, g * lanes.each, L) == __shfl(best.first, h * lanes.each, L) &&
                        __shfl(best.second, g * lanes.each, L) == __shfl(best.second, h * lanes.each, L);
      close |= !same && values[h] != -INFINITY && !(values[g] - values[h] > group_margin(a.sigmoid, largest));
      // Behind two that are the same, a third could be greater by less than 32 bits show.
      for (int o = 0; o < a.groups; ++o)
        close |= same && o != g && o != h && values[o] != -INFINITY &&
                 !(fabsf(values[o] - values[g]) > group_margin(a.sigmoid, largest));
    }
    // The group of an expert: half a step from a border at least, so the product decides it.
    const float inverse = static_cast<float>(a.groups) / static_cast<float>(a.experts);
    auto is_open = [&](int expert) {
      return lanes.has(open, static_cast<int>((static_cast<float>(expert) + 0.5f) * inverse));
    };
    if (Whole && size % V == 0) {
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const bool in = is_open(begin[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) key[i][j] = in ? key[i][j] : 0;
      }
    } else {
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (!is_open(begin[i] + j)) key[i][j] = 0;
    }
  }
  const int rounds = Biased ? (a.k + 2 < a.experts ? a.k + 2 : a.experts) : a.k;
  uint32_t best = 0;
#pragma unroll 1
  for (int q = 0; q < rounds; ++q) {
    uint32_t win;
    if constexpr (kPacked) {
      // No two keys are equal: the next one is the nearest below the last, the greatest
      // difference to it modulo 2^32 (from zero at first), and none has to be struck out.
      uint32_t next = 0;
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) next = key[i][j] - best > next ? key[i][j] - best : next;
      best = q > 0 && best == 0 ? 0 : best + lane_max<L>(next);  // zero: none is left
      win = kIndex - (best & kIndex);
    } else {
      uint32_t own = 0, at = 0xFFFFFFFFu;
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) own = key[i][j] > own ? key[i][j] : own;
      best = lane_max<L>(own);
#pragma unroll
      for (int i = I - 1; i >= 0; --i)
#pragma unroll
        for (int j = V - 1; j >= 0; --j) at = key[i][j] == best ? begin[i] + j : at;
      win = lane_min<L>(at);
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const uint32_t j0 = win - begin[i];
#pragma unroll
        for (int j = 0; j < V; ++j) key[i][j] = j0 == static_cast<uint32_t>(j) ? 0 : key[i][j];
      }
    }
    if (lane == 0) ids[q] = best > kNone ? static_cast<int32_t>(win) : -1;
  }
  // Of groups without a bias: whether a logit below x may differ from it and have its score in 64 bits.
  // The nearest is |x| 2^-24 away or more.  Over a gap in x a softmax changes by gap of itself, and its
  // x - m is rounded besides, a sigmoid by (1 - s) gap, at least min(1, e^-x) gap / 2: beyond x = 2^-24
  // and up to 14, where x e^-x is 2^-24 at least, that is more than a few roundings.
  auto may_tie = [&](float x) {
    return a.sigmoid ? !(x < 14.0f && fabsf(x) > 0x1p-24f) : !(fabsf(x) > 0x1p-24f * (1.0f + (m - x)));
  };
  auto ties = [&](float x, float gap) {
    return !(a.sigmoid ? gap * fminf(expf(-x), 1.0f) > 0x1p-49f : gap > 0x1p-49f * (1.0f + (m - x)));
  };
  float below = -INFINITY;  // the greatest logit that is lower than the last one chosen, where it may tie
  if constexpr (Grouped && !Biased) {
    constexpr uint32_t kValue = kPacked ? ~kFine : ~0u;
    auto logit = [&](uint32_t key) { return key_value(kPacked && key < 0x80000000u ? key | kFine : key & kValue); };
    if (__ballot(best > kNone && may_tie(logit(best))) != 0) {
      uint32_t own = 0;
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const uint32_t value = key[i][j] & kValue;
          own = value < (best & kValue) && value > own ? value : own;
        }
      own = lane_max<L>(own);
      if (own > (kNone & kValue)) below = logit(own);
    }
  }
  // A wave's LDS accesses are performed in order, and a row's lanes are of one wave.
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if constexpr (Biased) {
    auto clear = [&](int32_t i, int32_t j) {
      const float xi = static_cast<float>(row[i]), xj = static_cast<float>(row[j]), si = score(xi), sj = score(xj);
      return selected(si, xi, bias[i]) - selected(sj, xj, bias[j]) >
             pair_margin(a.sigmoid, si + sj, largest) + 4.0f * step_of_key;
    };
    // Neighbours among the k and the next one have to be clear of each other, or the same.
    for (int q = lane; q < a.k && q + 1 < rounds; q += L) {
      const int32_t i = ids[q], j = ids[q + 1];
      if (j < 0) continue;  // none is left
      close |= !clear(i, j) && !(row[i] == row[j] && bias[i] == bias[j]);
    }
    // Where the last chosen and the next one are the same, one behind them could yet be greater.
    if (rounds == a.k + 2 && ids[a.k + 1] >= 0) {
      const int32_t i = ids[a.k - 1], j = ids[a.k], n = ids[a.k + 1];
      close |= row[i] == row[j] && bias[i] == bias[j] && !clear(j, n);
    }
  } else if constexpr (Grouped) {
    // Where logits differ and their scores in 64 bits do not, the scores decide: those next to zero, and
    // neighbours among the k and the next one.
    for (int q = lane; q < a.k; q += L) scores[q] = ids[q] < 0 ? -INFINITY : static_cast<float>(row[ids[q]]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int q = lane; q < a.k; q += L) {
      const float x0 = scores[q], x1 = q + 1 == a.k ? below : scores[q + 1];
      if (x0 == -INFINITY) continue;  // none is left
      close |= !((a.sigmoid ? x0 : x0 - m) > -700.0f);
      if (may_tie(x0) && x0 != x1 && ties(x0, x0 - x1)) close = true;
    }
  }
  if constexpr (kChecked) {
    uint64_t rows = __ballot(close && live);
    while (rows != 0) {
      // The whole wave takes one such row after another.
      const int group = __builtin_ctzll(rows) / L;
      rows &= ~((~uint64_t(0) >> (64 - L)) << (group * L));
      const int64_t which = static_cast<int64_t>(blockIdx.x) * kGroups + (threadIdx.x >> 6) * (64 / L) + group;
      int32_t* into = all_ids + ((threadIdx.x >> 6) * (64 / L) + group) * (2 * a.k + 2);
      // With values that are no numbers, the chosen may be others than the NaN: it is to be seen all the same.
      if (choose_exactly(a, logits + which * a.stride, bias, exact, into) && (threadIdx.x & 63) / L == group)
        seen = NAN;
    }
  }
  most = -INFINITY;
  least = INFINITY;
  float sum = 0.0f;
#pragma unroll 1
  for (int q = lane; q < a.k; q += L) {
    const int32_t id = ids[q];
    scores[q] = id < 0 ? -INFINITY : static_cast<float>(row[id]);
    most = fmaxf(most, scores[q]);
    if (id >= 0) least = fminf(least, scores[q]);
  }
  most = lane_max<L>(most);
  // Sigmoids that fp32 does not hold keep their ratios as logarithms.
  const bool tiny = a.sigmoid && a.renormalize && lane_min_value<L>(least) < -80.0f;
  if (tiny) most = log_sigmoid(most);
#pragma unroll 1
  for (int q = lane; q < a.k; q += L) {
    const float xj = scores[q];
    float e;
    if (a.sigmoid && !tiny) e = 1.0f / (1.0f + expf(-xj));
    else e = expf(a.sigmoid ? log_sigmoid(xj) - most : a.renormalize ? xj - most : (xj - m) - ls);
    scores[q] = ids[q] < 0 ? 0.0f : e + seen;
    sum += scores[q];
  }
  const float over = a.renormalize ? lane_sum<L>(sum) : 1.0f;
#pragma unroll 1
  for (int q = lane; q < a.k && live; q += L) {
    weights[r * a.k + q] = ids[q] < 0 ? 0.0f : a.scale * (scores[q] / over);
    chosen[r * a.k + q] = ids[q];
  }
  if (stats != nullptr && lane == 0 && live) {
    stats[2 * r] = m;
    stats[2 * r + 1] = ls;
  }
}

// dlogits of kTile / experts rows a work-group, put together in LDS: what every
// expert has of it (softmax that is not renormalised), then the chosen.  65536 x
// 256 fp32, k = 8: 20.6 us (5.2 TB/s); 100000 x 12 fp16, k = 2,
// 7.0.
constexpr int kTile = 2048;
template <typename T, bool Narrow>
__global__ __launch_bounds__(kThreads) void route_grad(RouteArgs a, const T* __restrict__ logits,
                                                       const int32_t* __restrict__ chosen,
                                                       const float* __restrict__ weights,
                                                       const float* __restrict__ stats, const float* __restrict__ grad,
                                                       T* __restrict__ dlogits) {
  using Piece = RowPiece<T, Narrow>;
  constexpr int V = kPiece<T>;
  alignas(16) __shared__ float out[kTile + V];
  __shared__ float parts[kTile], sums[kTile];  // by choice, by row
  const int tile = kTile / a.experts;
  const bool dense = !a.sigmoid && !a.renormalize;
  const int64_t step = static_cast<int64_t>(gridDim.x) * tile;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * tile; r0 < a.rows; r0 += step) {
    const int rows = static_cast<int>(a.rows - r0 < tile ? a.rows - r0 : tile);
    const int choices = rows * a.k, all = rows * a.experts;
    for (int q = threadIdx.x; q < choices; q += kThreads) {
      const int64_t at = r0 * a.k + q;
      const float w = a.renormalize ? weights[at] / a.scale : weights[at], g = grad[at];
      parts[q] = static_cast<uint32_t>(chosen[at]) < static_cast<uint32_t>(a.experts) ? w * g : 0.0f;
    }
    __syncthreads();
    for (int q = threadIdx.x; q < rows; q += kThreads) {
      float sum = 0.0f;
      for (int j = 0; j < a.k; ++j) sum += parts[q * a.k + j];
      sums[q] = sum;
    }
    if (!dense)
      for (int q = threadIdx.x * 4; q < all; q += kThreads * 4) *reinterpret_cast<f32x4*>(out + q) = f32x4{};
    __syncthreads();
    if (dense) {
      const int pieces = (a.experts + V - 1) / V;
      for (int q = threadIdx.x; q < rows * pieces; q += kThreads) {
        const int row = q / pieces, column = (q - row * pieces) * V;
        const piece_t<T> raw = Piece::load(logits + (r0 + row) * a.stride, column, a.experts);
        const int begin = static_cast<int>(Piece::begin(column, a.experts));
        const float m = stats[2 * (r0 + row)], ls = stats[2 * (r0 + row) + 1], sum = sums[row];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (Narrow && column + j >= a.experts) break;
          const float x = static_cast<float>(raw[j]);
          out[row * a.experts + begin + j] = x == -INFINITY ? 0.0f : -expf((x - m) - ls) * sum;
        }
      }
      __syncthreads();
    }
    for (int q = threadIdx.x; q < choices; q += kThreads) {
      const int64_t at = r0 * a.k + q;
      const int32_t e = chosen[at];
      if (static_cast<uint32_t>(e) >= static_cast<uint32_t>(a.experts)) continue;
      const int row = q / a.k;
      const float w = weights[at], g = grad[at];
      // Renormalised, the gradient's mean under the weights: equal gradients cancel, a single one exactly.
      float v = a.renormalize ? w * (g - sums[row]) : w * g;
      if (a.sigmoid) v /= 1.0f + expf(static_cast<float>(logits[(r0 + row) * a.stride + e]));
      out[row * a.experts + e] += v;
    }
    __syncthreads();
    for (int q = threadIdx.x * V; q < all; q += kThreads * V) {
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = out[q + j];
      store_piece(dlogits + r0 * a.experts + q, all - q, v);
    }
    __syncthreads();
  }
}

spmm_status check_route_desc(const spmm_route_desc* d) {
  if (d == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null descriptor");
  if (!dense_type(d->value_type)) return fail(SPMM_ERR_CONTRACT, "route supports only FP16, BF16 and FP32 tensors");
  if (d->score != SPMM_SCORE_SOFTMAX && d->score != SPMM_SCORE_SIGMOID)
    return fail(SPMM_ERR_INVALID_ARGUMENT, "route: score must be softmax or sigmoid");
  if (d->rows < 0) return fail(SPMM_ERR_CONTRACT, "route: negative extent");
  if (d->experts < 1 || d->experts > kMaxExperts)
    return fail(SPMM_ERR_CONTRACT, "route takes 1 to 1024 experts, but got " + std::to_string(d->experts));
  if (d->rows > 1 && d->logits_stride < d->experts) return fail(SPMM_ERR_CONTRACT, "route: rows of logits overlap");
  if (d->groups < 1 || d->groups > kMaxGroups || d->experts % d->groups != 0)
    return fail(SPMM_ERR_INVALID_ARGUMENT, "route: groups must be 1 to 64 and divide the experts, but got " +
                                               std::to_string(d->groups));
  if (d->top_groups < 1 || d->top_groups > d->groups)
    return fail(SPMM_ERR_INVALID_ARGUMENT, "route: top_groups must be 1 to groups, but got " +
                                               std::to_string(d->top_groups));
  const int64_t open = d->experts / d->groups * d->top_groups;
  if (d->top_k < 1 || d->top_k > kMaxTopK || d->top_k > open)
    return fail(SPMM_ERR_INVALID_ARGUMENT, "route: top_k must be 1 to 64 and at most the experts of top_groups groups (" +
                                               std::to_string(open) + "), but got " + std::to_string(d->top_k));
  if (!(d->scale >= FLT_MIN) || !(d->scale <= FLT_MAX))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "route: scale must be a positive FP32 number");
  return SPMM_OK;
}

RouteArgs route_args(const spmm_route_desc* d) {
  return {d->rows,
          d->logits_stride,
          static_cast<int32_t>(d->experts),
          static_cast<int32_t>(d->top_k),
          static_cast<int32_t>(d->groups),
          static_cast<int32_t>(d->top_groups),
          static_cast<float>(d->scale),
          d->score == SPMM_SCORE_SIGMOID,
          d->renormalize != 0};
}

template <typename T>
spmm_status run_route(const spmm_route_desc* d, const void* logits, const float* bias, float* weights, int32_t* chosen,
                      float* stats, hipStream_t s) {
  const RouteArgs a = route_args(d);
  constexpr int V = kPiece<T>;
  auto launch = [&](auto L, auto I, auto Shape) {
    constexpr int kL = decltype(L)::value, kI = decltype(I)::value, kGroups = kThreads / kL;
    constexpr RowShape kShape = decltype(Shape)::value;
    const dim3 grid(static_cast<unsigned>(ceil_div(a.rows, kGroups)));
    const size_t exact = bias != nullptr || a.groups > 1 ? static_cast<size_t>(a.experts) * 8 * (kThreads / 64) : 0;
    const size_t values = a.groups > 1 ? align_up(static_cast<size_t>(a.experts), 4) * 4 : 0;
    const size_t lds = exact + kGroups * (values + (2 * static_cast<size_t>(a.k) + 2) * 4);
    const T* x = static_cast<const T*>(logits);
    if (bias != nullptr && a.groups > 1)
      hipLaunchKernelGGL((route_rows<T, kL, kI, kShape, true, true>), grid, dim3(kThreads), lds, s, a, x, bias,
                         weights, chosen, stats);
    else if (bias != nullptr)
      hipLaunchKernelGGL((route_rows<T, kL, kI, kShape, true, false>), grid, dim3(kThreads), lds, s, a, x, bias,
                         weights, chosen, stats);
    else if (a.groups > 1)
      hipLaunchKernelGGL((route_rows<T, kL, kI, kShape, false, true>), grid, dim3(kThreads), lds, s, a, x, bias,
                         weights, chosen, stats);
    else
      hipLaunchKernelGGL((route_rows<T, kL, kI, kShape, false, false>), grid, dim3(kThreads), lds, s, a, x, bias,
                         weights, chosen, stats);
  };
  using std::integral_constant;
  auto with_shape = [&](auto L, auto I) {
    if (d->experts % V == 0) launch(L, I, integral_constant<RowShape, RowShape::kWhole>());
    else launch(L, I, integral_constant<RowShape, RowShape::kMoved>());
  };
  const int64_t pieces = ceil_div(d->experts, V);
  // A launch has fewer than 2^32 work-items.
  constexpr int64_t kMost = int64_t(1) << 24;
  if (d->rows > kMost) {
    for (int64_t r = 0; r < d->rows; r += kMost) {
      spmm_route_desc part = *d;
      part.rows = d->rows - r < kMost ? d->rows - r : kMost;
      if (spmm_status st = run_route<T>(&part, static_cast<const T*>(logits) + r * d->logits_stride, bias,
                                        weights + r * d->top_k, chosen + r * d->top_k,
                                        stats == nullptr ? nullptr : stats + 2 * r, s))
        return st;
    }
    return SPMM_OK;
  }
  // The fewest lanes that hold the row in one piece each, or in 16 logits each, and a lane a group at least.
  constexpr integral_constant<int, 1> one;
  constexpr integral_constant<int, 16 / V> more;
  if (d->experts < V) launch(integral_constant<int, 8>(), one, integral_constant<RowShape, RowShape::kNarrow>());
  else if (pieces <= 4 && d->groups <= 4) with_shape(integral_constant<int, 4>(), one);
  else if (pieces <= 8 && d->groups <= 8) with_shape(integral_constant<int, 8>(), one);
  else if (pieces <= 16 && d->groups <= 16) with_shape(integral_constant<int, 16>(), one);
  else if (pieces <= 16 * more.value && d->groups <= 16) with_shape(integral_constant<int, 16>(), more);
  else if (pieces <= 32 * more.value && d->groups <= 32) with_shape(integral_constant<int, 32>(), more);
  else if (pieces <= 64) with_shape(integral_constant<int, 64>(), one);
  else with_shape(integral_constant<int, 64>(), more);
  return check_launch("route");
}

template <typename T>
spmm_status run_route_grad(const spmm_route_desc* d, const void* logits, const int32_t* chosen, const float* weights,
                           const float* stats, const float* grad, void* dlogits, hipStream_t s) {
  const RouteArgs a = route_args(d);
  const int64_t blocks = ceil_div(d->rows, kTile / d->experts);
  const dim3 grid(static_cast<unsigned>(blocks < 16384 ? blocks : 16384));
  if (d->experts < kPiece<T>)
    hipLaunchKernelGGL((route_grad<T, true>), grid, dim3(kThreads), 0, s, a, static_cast<const T*>(logits), chosen,
                       weights, stats, grad, static_cast<T*>(dlogits));
  else
    hipLaunchKernelGGL((route_grad<T, false>), grid, dim3(kThreads), 0, s, a, static_cast<const T*>(logits), chosen,
                       weights, stats, grad, static_cast<T*>(dlogits));
  return check_launch("route_grad");
}

}  // namespace
}  // namespace spmm

using namespace spmm;

extern "C" {

spmm_status spmm_route_run(const spmm_route_desc* d, const void* logits, const float* bias, float* weights,
                           int32_t* chosen, float* stats, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_route_desc(d)) return st;
  if (d->rows == 0) return SPMM_OK;
  if (logits == nullptr || weights == nullptr || chosen == nullptr)
    return fail(SPMM_ERR_INVALID_ARGUMENT, "route: null device pointer");
  hipStream_t s = as_stream(stream);
  switch (d->value_type) {
    case SPMM_VALUE_F16: return run_route<_Float16>(d, logits, bias, weights, chosen, stats, s);
    case SPMM_VALUE_BF16: return run_route<__bf16>(d, logits, bias, weights, chosen, stats, s);
    default: return run_route<float>(d, logits, bias, weights, chosen, stats, s);
  }
}

spmm_status spmm_route_grad_run(const spmm_route_desc* d, const void* logits, const int32_t* chosen,
                                const float* weights, const float* stats, const float* grad, void* dlogits,
                                spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_route_desc(d)) return st;
  if (d->rows == 0) return SPMM_OK;
  const bool dense = d->score == SPMM_SCORE_SOFTMAX && d->renormalize == 0;
  if (logits == nullptr || chosen == nullptr || weights == nullptr || grad == nullptr || dlogits == nullptr ||
      (dense && stats == nullptr))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "route: null device pointer");
  hipStream_t s = as_stream(stream);
  switch (d->value_type) {
    case SPMM_VALUE_F16: return run_route_grad<_Float16>(d, logits, chosen, weights, stats, grad, dlogits, s);
    case SPMM_VALUE_BF16: return run_route_grad<__bf16>(d, logits, chosen, weights, stats, grad, dlogits, s);
    default: return run_route_grad<float>(d, logits, chosen, weights, stats, grad, dlogits, s);
  }
}

}  // extern "C"
