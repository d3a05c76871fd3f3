// Rows of a table by ids, scaled, and the gradient of the table.
//
//   out[i] = scale * weight[ids[i]],   dweight[v] = scale * sum of grad[i] over ids[i] = v
//
// An id outside the table gives a row of zeros and adds to none.  The gradient's
// sums are fp32, in the order of the positions, so that they repeat exactly: the
// ids are sorted (stably) and each run of equal ones is summed.
#include <cfloat>
#include <cmath>

#include "lane_reduce.h"
#include "row_pieces.h"
#include "sort_ids.h"

namespace spmm {
namespace {

constexpr int kThreads = 256;

struct TableArgs {
  int64_t count, table, width, weight_stride, grad_stride;
  float scale;
  bool index64;
};

__device__ inline int64_t id_at(const void* ids, bool index64, int64_t i) {
  return index64 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// A group of L lanes takes kRows rows of the output at a time, whose loads are
// under way together.  Ids outside the table read a row of it all the same (the
// table has one) and keep nothing of it.  Bound by memory: 262144 popular ids of a
// table of 131072 x 1024 bf16 153 us (5.3 TB/s), 100000 x 128 fp32 17.6 (5.8).
// Two rows and eight at a time: the same.
constexpr int kRows = 4;
template <typename T, int L, bool Narrow>
__global__ __launch_bounds__(kThreads) void gather_table(TableArgs a, const T* __restrict__ weight,
                                                         const void* __restrict__ ids, T* __restrict__ out) {
  using Piece = RowPiece<T, Narrow>;
  constexpr int V = kPiece<T>, kGroups = kThreads / L;
  const int lane = threadIdx.x % L;
  int64_t group = static_cast<int64_t>(blockIdx.x) * kGroups;
  if constexpr (L == 64) group += __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  else group += threadIdx.x / L;
  for (int64_t i = group * kRows; i < a.count; i += static_cast<int64_t>(gridDim.x) * kGroups * kRows) {
    int64_t id[kRows];
    bool present[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) id[u] = id_at(ids, a.index64, i + u < a.count ? i + u : a.count - 1);
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      present[u] = static_cast<uint64_t>(id[u]) < static_cast<uint64_t>(a.table);
      if (!present[u]) id[u] = 0;
    }
    for (int64_t c = lane * V; c < a.width; c += L * V) {
      piece_t<T> raw[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) raw[u] = Piece::load(weight + id[u] * a.weight_stride, c, a.width);
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        if (i + u >= a.count) break;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = present[u] ? static_cast<float>(raw[u][j]) * a.scale : 0.0f;
        Piece::template store<true>(out + (i + u) * a.width, c, a.width, v);
      }
    }
  }
}

// An empty table: zeros.
template <typename T>
__global__ __launch_bounds__(kThreads) void zero_rows(int64_t n, T* out) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads)
    out[i] = static_cast<T>(0.0f);
}

// The keys of the sort: an id, or the table's rows for one outside of it.
struct IdKeys {
  const void* ids;
  bool index64;
  int64_t table;
  __device__ inline uint32_t operator()(int64_t i) const {
    const int64_t id = id_at(ids, index64, i);
    return static_cast<uint32_t>(static_cast<uint64_t>(id) < static_cast<uint64_t>(table) ? id : table);
  }
};
struct SortedKeys {
  const uint32_t* keys;
  __device__ inline uint32_t operator()(int64_t i) const { return keys[i]; }
};
// Keys and positions at their places; `from` holds the positions so far (null: i itself).
struct PutPairs {
  const uint32_t* from;
  uint32_t *keys, *order;
  __device__ inline void operator()(int64_t i, uint32_t key, uint32_t place) const {
    keys[place] = key;
    order[place] = from == nullptr ? static_cast<uint32_t>(i) : from[i];
  }
};
// The count of the runs over several ranges starts at zero: cleared by the sort, as it runs before the sums.
struct ClearRuns {
  uint32_t* runs;
  __device__ inline void operator()(int b, uint32_t) const {
    if (b == 0) *runs = 0;
  }
};

// A group of lanes sums the rows of `range` sorted positions, loading kBatch of
// them at a time.  A run of one id that lies in one range is stored at once; each
// part of a longer run goes to a slot: [2 * range] for a run that began before
// the range, [2 * range + 1] for one that begins in it.  Bound by memory, each
// row of the gradient read once: 262144 x 1024 bf16 168 us (5.0 TB/s), 100000 x 128
// fp32 22.4 (4.6).
constexpr int kBatch = 8;

// Positions of a range: 32, so that the slots of long runs stay few against
// their rows, down to 8 where that leaves less than 8192 waves.
inline int range_of(int64_t count, int64_t pieces) {
  int range = 32;
  const int64_t lanes = pieces < 64 ? (pieces < 4 ? 4 : pieces) : ceil_div(pieces, 64) * 64;
  while (range > kBatch && count / range * lanes < int64_t(8192) * 64) range /= 2;
  return range;
}

struct SumArgs {
  TableArgs a;
  const uint32_t *keys, *order;
  float* slots;
  uint32_t* runs;  // [0]: runs over several ranges so far; then the range in which each begins
  int64_t range, ranges, zero_blocks, pieces;
};

template <typename T, int L, bool Narrow>
__global__ __launch_bounds__(kThreads) void sum_runs(SumArgs s, const T* __restrict__ grad, T* __restrict__ dweight) {
  using Piece = RowPiece<T, Narrow>;
  constexpr int V = kPiece<T>, kGroups = kThreads / L;
  const TableArgs& a = s.a;
  const int64_t n = a.count;
  if (static_cast<int64_t>(blockIdx.x) < s.zero_blocks) {
    // Rows of the table that no id names become zero: a wave looks 64 of them up.
    if (blockIdx.y != 0) return;
    const int lane = threadIdx.x & 63;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6)) * 64;
    const int64_t v = first + lane;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (s.keys[mid] < v) lo = mid + 1;
      else hi = mid;
    }
    uint64_t absent = __ballot(v < a.table && (lo >= n || s.keys[lo] != v));
    const piece_t<T> zero = {};
    while (absent != 0) {
      const int64_t row = first + __builtin_ctzll(absent);
      absent &= absent - 1;
      for (int64_t c = lane * V; c < a.width; c += 64 * V)
        Piece::template store<true>(dweight + row * a.width, c, a.width, zero);
    }
    return;
  }
  const int64_t block = static_cast<int64_t>(blockIdx.x) - s.zero_blocks;
  int64_t range = block * kGroups;
  if constexpr (L == 64) range += __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  else range += threadIdx.x / L;
  const int64_t p = static_cast<int64_t>(blockIdx.y) * L + threadIdx.x % L, c = p * V;
  if (range >= s.ranges || p >= s.pieces) return;
  const int64_t begin = range * s.range, end = begin + s.range < n ? begin + s.range : n;
  const uint32_t before = begin > 0 ? s.keys[begin - 1] : ~0u, after = end < n ? s.keys[end] : ~0u;
  float sum[V] = {};
  uint32_t key = s.keys[begin];
  bool head = key == before;
  auto flush = [&](bool tail) {
    if (key >= a.table) return;
    if (head || tail) {
      float* slot = s.slots + ((2 * range + (head ? 0 : 1)) * s.pieces + p) * V;
#pragma unroll
      for (int j = 0; j < V; j += 4)
        *reinterpret_cast<f32x4*>(slot + j) = f32x4{sum[j], sum[j + 1], sum[j + 2], sum[j + 3]};
      if (!head && p == 0) s.runs[1 + atomicAdd(s.runs, 1u)] = static_cast<uint32_t>(range);
    } else {
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = sum[j] * a.scale;
      Piece::template store<true>(dweight + static_cast<int64_t>(key) * a.width, c, a.width, v);
    }
  };
  // Keys and positions are read one batch ahead of the rows.
  uint32_t k[kBatch], at[kBatch];
  auto fetch = [&](int64_t i) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      k[u] = s.keys[i + u < end ? i + u : end - 1];
      at[u] = s.order[i + u < end ? i + u : end - 1];
    }
  };
  fetch(begin);
  for (int64_t i = begin; i < end; i += kBatch) {
    uint32_t now[kBatch];
    piece_t<T> raw[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      now[u] = k[u];
      raw[u] = Piece::template load<true>(grad + static_cast<int64_t>(at[u]) * a.grad_stride, c, a.width);
    }
    if (i + kBatch < end) fetch(i + kBatch);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (i + u >= end) break;
      if (now[u] != key) {
        flush(false);
        key = now[u];
        head = false;
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += static_cast<float>(raw[u][j]);
    }
  }
  flush(key == after);
}

// Adds the slots of the runs over several ranges, 64 pieces of their columns a
// work-group.  A run of up to kShort ranges is added by one wave, a longer one by
// all waves of the work-group: each adds consecutive ranges, and the waves' sums
// are added in order.  The 1400 runs of 262144 popular ids of width 1024, most of
// them short: 21 us, and 54 with a work-group for each, one after another.
constexpr int kJoinWaves = 16, kShort = 32;

// Ranges of the run that begins in range `first`: 64 probes at a time for one
// past the last range whose first key is the run's.
__device__ inline int64_t run_ranges(const SumArgs& s, int64_t first, uint32_t key) {
  const int lane = threadIdx.x & 63;
  int64_t lo = first + 2, hi = s.ranges, ahead = 64;
  // Most runs are short: the next 64 ranges first.
  if (hi - lo > ahead) {
    const uint64_t more = __ballot(s.keys[(lo + lane) * s.range] != key);
    if (more != 0) return lo + __builtin_ctzll(more) - first;
    lo += ahead;
  }
  while (lo < hi) {
    const int64_t step = (hi - lo + 63) / 64, probe = lo + lane * step;
    const uint64_t more = __ballot(probe < hi && s.keys[probe * s.range] != key);
    if (more == 0) {
      lo += (hi - 1 - lo) / step * step + 1;  // past the last probe
    } else {
      const int at = __builtin_ctzll(more);
      hi = lo + at * step;
      lo = at == 0 ? hi : lo + (at - 1) * step + 1;
    }
  }
  return lo - first;
}

template <typename T, bool Narrow>
__global__ __launch_bounds__(64 * kJoinWaves) void join_runs(SumArgs s, T* __restrict__ dweight) {
  constexpr int V = kPiece<T>;
  __shared__ float part[kJoinWaves][64 * V];
  __shared__ uint32_t longer[kJoinWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t p = static_cast<int64_t>(blockIdx.y) * 64 + lane, c = p * V;
  const bool live = p < s.pieces;
  const uint32_t runs = s.runs[0];
  auto add = [&](int64_t first, int64_t k0, int64_t k1, float (&sum)[V]) {
#pragma unroll 8
    for (int64_t k = k0; k < k1; ++k) {
      const float* slot = s.slots + ((2 * (first + k) + (k == 0 ? 1 : 0)) * s.pieces + p) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += slot[j];
    }
  };
  auto store = [&](uint32_t key, const float (&sum)[V]) {
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = sum[j] * s.a.scale;
    RowPiece<T, Narrow>::store(dweight + static_cast<int64_t>(key) * s.a.width, c, s.a.width, v);
  };
  for (uint32_t q0 = blockIdx.x * kJoinWaves; q0 < runs; q0 += gridDim.x * kJoinWaves) {
    const uint32_t q = q0 + wave;
    int64_t ranges = 0;
    if (q < runs) {
      const int64_t first = s.runs[1 + q];
      const uint32_t key = s.keys[(first + 1) * s.range];
      ranges = run_ranges(s, first, key);
      if (ranges <= kShort && live) {
        float sum[V] = {};
        add(first, 0, ranges, sum);
        store(key, sum);
      }
    }
    if (lane == 0) longer[wave] = ranges > kShort ? static_cast<uint32_t>(ranges) : 0;
    __syncthreads();
    for (int w = 0; w < kJoinWaves; ++w) {
      const int64_t all = longer[w];
      if (all == 0) continue;
      const int64_t first = s.runs[1 + q0 + w];
      float sum[V] = {};
      if (live) add(first, all * wave / kJoinWaves, all * (wave + 1) / kJoinWaves, sum);
#pragma unroll
      for (int j = 0; j < V; ++j) part[wave][lane * V + j] = sum[j];
      __syncthreads();
      if (wave == 0 && live) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          sum[j] = 0.0f;
#pragma unroll
          for (int k = 0; k < kJoinWaves; ++k) sum[j] += part[k][lane * V + j];
        }
        store(s.keys[(first + 1) * s.range], sum);
      }
      __syncthreads();
    }
    __syncthreads();  // the list is read
  }
}

spmm_status check_embedding_desc(const spmm_embedding_desc* d) {
  if (d == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null descriptor");
  if (!dense_type(d->value_type)) return fail(SPMM_ERR_CONTRACT, "embedding supports only FP16, BF16 and FP32 tensors");
  if (d->index_type != SPMM_INDEX_I32 && d->index_type != SPMM_INDEX_I64)
    return fail(SPMM_ERR_CONTRACT, "embedding: ids must be int32 or int64");
  if (d->count < 0 || d->table_rows < 0 || d->width < 0) return fail(SPMM_ERR_CONTRACT, "embedding: negative extent");
  if (d->count >= (1 << 30) || d->table_rows >= (1 << 30) || d->width >= (1 << 22))
    return fail(SPMM_ERR_CONTRACT, "embedding: ids and rows of the table must be below 2^30, the width below 2^22");
  if (d->table_rows > 1 && d->weight_stride < d->width)
    return fail(SPMM_ERR_CONTRACT, "embedding: rows of weight overlap");
  if (!(std::fabs(d->scale) <= FLT_MAX))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "embedding: scale must be finite in FP32");
  return SPMM_OK;
}

TableArgs table_args(const spmm_embedding_desc* d) {
  return {d->count,       d->table_rows, d->width, d->weight_stride, d->grad_stride, static_cast<float>(d->scale),
          d->index_type == SPMM_INDEX_I64};
}

// f(L, Narrow): lanes of a row, one piece of 16 bytes each.
template <typename T, typename F>
void with_row_lanes(int64_t width, F f) {
  using std::integral_constant;
  const int64_t pieces = ceil_div(width, kPiece<T>);
  if (width < kPiece<T>) f(integral_constant<int, 4>(), std::true_type());
  else if (pieces <= 4) f(integral_constant<int, 4>(), std::false_type());
  else if (pieces <= 8) f(integral_constant<int, 8>(), std::false_type());
  else if (pieces <= 16) f(integral_constant<int, 16>(), std::false_type());
  else if (pieces <= 32) f(integral_constant<int, 32>(), std::false_type());
  else f(integral_constant<int, 64>(), std::false_type());
}

template <typename T>
spmm_status run_gather(const spmm_embedding_desc* d, const void* weight, const void* ids, void* out, hipStream_t s) {
  if (d->table_rows == 0) {
    const int64_t n = d->count * d->width, blocks = ceil_div(n, kThreads);
    hipLaunchKernelGGL(zero_rows<T>, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(kThreads), 0, s, n,
                       static_cast<T*>(out));
    return check_launch("embedding");
  }
  with_row_lanes<T>(d->width, [&](auto L, auto Narrow) {
    constexpr int kGroups = kThreads / decltype(L)::value;
    const int64_t blocks = ceil_div(d->count, kGroups * kRows);
    hipLaunchKernelGGL((gather_table<T, decltype(L)::value, decltype(Narrow)::value>),
                       dim3(static_cast<unsigned>(blocks < 16384 ? blocks : 16384)), dim3(kThreads), 0, s, table_args(d),
                       static_cast<const T*>(weight), ids, static_cast<T*>(out));
  });
  return check_launch("embedding");
}

// How the ids are sorted, and where in the workspace what lies.
struct SortLayout {
  int passes, bits;
  int64_t range, ranges, pieces;
  size_t counts, keys[2], order[2], runs, slots, bytes;
};

SortLayout sort_layout(const spmm_embedding_desc* d) {
  SortLayout l;
  const int all = bits_of(d->table_rows);
  l.passes = (all + kSortBits - 1) / kSortBits;
  l.bits = (all + l.passes - 1) / l.passes;
  const int64_t piece = 16 / dense_type_bytes(d->value_type);
  l.pieces = ceil_div(d->width, piece);
  l.range = range_of(d->count, l.pieces);
  l.ranges = ceil_div(d->count, l.range);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align_up(bytes, 256);
    return here;
  };
  l.counts = take(static_cast<size_t>(sort_words(d->count, 1 << l.bits)) * 4);
  for (int k = 0; k < 2; ++k) {
    l.keys[k] = take(static_cast<size_t>(d->count) * 4);
    l.order[k] = take(static_cast<size_t>(d->count) * 4);
  }
  l.runs = take(static_cast<size_t>(l.ranges + 1) * 4);
  l.slots = take(static_cast<size_t>(l.ranges) * 2 * l.pieces * piece * 4);
  l.bytes = at;
  return l;
}

template <typename T>
spmm_status run_gradient(const spmm_embedding_desc* d, const void* ids, const void* grad, void* dweight,
                         void* workspace, hipStream_t s) {
  const SortLayout l = sort_layout(d);
  char* ws = static_cast<char*>(workspace);
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + l.counts);
  uint32_t* runs = reinterpret_cast<uint32_t*>(ws + l.runs);
  uint32_t *keys = nullptr, *order = nullptr;
  const IdKeys from_ids = {ids, d->index_type == SPMM_INDEX_I64, d->table_rows};
  const ClearRuns clear = {runs};
  const bool ranked = d->count <= kRankMost;
  for (int pass = 0; pass < (ranked ? 1 : l.passes) && d->count > 0; ++pass) {
    const Digit digit = {pass * l.bits, l.bits, 1 << l.bits};
    const PutPairs put = {order, reinterpret_cast<uint32_t*>(ws + l.keys[pass & 1]),
                          reinterpret_cast<uint32_t*>(ws + l.order[pass & 1])};
    spmm_status st = ranked      ? sort_by_rank(d->count, 1, from_ids, put, clear, s)
                     : pass == 0 ? sort_digit(digit, d->count, from_ids, counts, put, clear, s)
                                 : sort_digit(digit, d->count, SortedKeys{keys}, counts, put, clear, s);
    if (st) return st;
    keys = put.keys;
    order = put.order;
  }
  SumArgs a = {table_args(d), keys, order, reinterpret_cast<float*>(ws + l.slots), runs, l.range, l.ranges, 0, l.pieces};
  a.zero_blocks = ceil_div(d->table_rows, kThreads);
  with_row_lanes<T>(d->width, [&](auto L, auto Narrow) {
    const int64_t sum_blocks = ceil_div(l.ranges, kThreads / decltype(L)::value);
    hipLaunchKernelGGL((sum_runs<T, decltype(L)::value, decltype(Narrow)::value>),
                       dim3(static_cast<unsigned>(a.zero_blocks + sum_blocks),
                            static_cast<unsigned>(ceil_div(l.pieces, decltype(L)::value))),
                       dim3(kThreads), 0, s, a, static_cast<const T*>(grad), static_cast<T*>(dweight));
  });
  if (spmm_status st = check_launch("embedding_grad")) return st;
  if (l.ranges < 2) return SPMM_OK;
  const int64_t groups = ceil_div(l.ranges, kJoinWaves);
  const dim3 grid(static_cast<unsigned>(groups < 512 ? groups : 512), static_cast<unsigned>(ceil_div(l.pieces, 64)));
  if (d->width < kPiece<T>)
    hipLaunchKernelGGL((join_runs<T, true>), grid, dim3(64 * kJoinWaves), 0, s, a, static_cast<T*>(dweight));
  else
    hipLaunchKernelGGL((join_runs<T, false>), grid, dim3(64 * kJoinWaves), 0, s, a, static_cast<T*>(dweight));
  return check_launch("embedding_grad join");
}

}  // namespace
}  // namespace spmm

using namespace spmm;

extern "C" {

spmm_status spmm_embedding_run(const spmm_embedding_desc* d, const void* weight, const void* ids, void* out,
                               spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_embedding_desc(d)) return st;
  if (d->count == 0 || d->width == 0) return SPMM_OK;
  if ((d->table_rows > 0 && weight == nullptr) || ids == nullptr || out == nullptr)
    return fail(SPMM_ERR_INVALID_ARGUMENT, "embedding: null device pointer");
  hipStream_t s = as_stream(stream);
  switch (d->value_type) {
    case SPMM_VALUE_F16: return run_gather<_Float16>(d, weight, ids, out, s);
    case SPMM_VALUE_BF16: return run_gather<__bf16>(d, weight, ids, out, s);
    default: return run_gather<float>(d, weight, ids, out, s);
  }
}

spmm_status spmm_embedding_grad_workspace(const spmm_embedding_desc* d, size_t* bytes) {
  clear_error();
  if (bytes == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null argument");
  if (spmm_status st = check_embedding_desc(d)) return st;
  *bytes = sort_layout(d).bytes;
  return SPMM_OK;
}

spmm_status spmm_embedding_grad_run(const spmm_embedding_desc* d, const void* ids, const void* grad, void* dweight,
                                    void* workspace, size_t workspace_bytes, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_embedding_desc(d)) return st;
  if (d->count > 1 && d->grad_stride < d->width) return fail(SPMM_ERR_CONTRACT, "embedding: rows of grad overlap");
  if (d->table_rows == 0 || d->width == 0) return SPMM_OK;
  if (dweight == nullptr || (d->count > 0 && (ids == nullptr || grad == nullptr)))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "embedding: null device pointer");
  const size_t need = sort_layout(d).bytes;
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SPMM_ERR_CONTRACT, "embedding: workspace too small: need " + std::to_string(need) + " bytes");
  hipStream_t s = as_stream(stream);
  switch (d->value_type) {
    case SPMM_VALUE_F16: return run_gradient<_Float16>(d, ids, grad, dweight, workspace, s);
    case SPMM_VALUE_BF16: return run_gradient<__bf16>(d, ids, grad, dweight, workspace, s);
    default: return run_gradient<float>(d, ids, grad, dweight, workspace, s);
  }
}

}  // extern "C"
