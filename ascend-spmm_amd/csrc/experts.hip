// Rows brought to their experts and back.
//
// Row r has k choices of an expert.  Sorted by expert (stably, those outside of
// the experts behind all), choice (r, j) lies at place[r][j] of the packed rows,
// whose expert e has rows offsets[e] to offsets[e + 1]:
//   pack:     packed[place[r][j]] = x[r],               dx[r] = sum_j dpacked[place[r][j]]
//   restore:  out[r] = sum_j w[r][j] y[place[r][j]],    dy[place[r][j]] = w[r][j] dout[r],
//                                                       dw[r][j] = <dout[r], y[place[r][j]]>
// A choice of no expert is nothing in these sums, and its packed row is zero.
//
// All four are bound by memory.  They go row by row of the unpacked side, so
// that x and dout are read once for all k choices and the sums need no atomics.
#include "lane_reduce.h"
#include "row_pieces.h"
#include "sort_ids.h"

namespace spmm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxCount = 2048;
constexpr int kMaxChoices = 64;

// A choice's expert, or `count` for none.
struct ChoiceKeys {
  const void* ids;
  bool index64;
  int64_t count;
  __device__ inline uint32_t operator()(int64_t i) const {
    const int64_t id = index64 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
    return static_cast<uint32_t>(static_cast<uint64_t>(id) < static_cast<uint64_t>(count) ? id : count);
  }
};
struct PutPlace {
  int32_t* place;
  __device__ inline void operator()(int64_t i, uint32_t, uint32_t at) const { place[i] = static_cast<int32_t>(at); }
};
struct PutOffsets {
  int32_t* offsets;
  __device__ inline void operator()(int b, uint32_t at) const { offsets[b] = static_cast<int32_t>(at); }
};

struct RowsArgs {
  int64_t rows, width, stride, other_stride;  // of x or y; of the incoming gradient
  int32_t k, count;
  int64_t choices;
};

// The packed rows that belong to experts: those from here on are of choices of
// none.  Never more than there are, whatever `offsets` holds.
__device__ inline uint32_t kept_rows(const RowsArgs& a, const int32_t* offsets) {
  const int32_t end = offsets[a.count];
  return end < 0 ? 0u : end < a.choices ? static_cast<uint32_t>(end) : static_cast<uint32_t>(a.choices);
}

// The kernels' common walk: L lanes a row, which take L * I pieces of 16 bytes of
// it at a time, and kTogether choices, whose rows' loads are all under way
// together.  Each group of lanes has consecutive rows.  A whole wave's row is a
// scalar, and so are the loads of its places and weights.
constexpr int kTogether = 8;

template <typename T, int L, int I, bool Narrow>
struct ChoiceTile {
  using Piece = RowPiece<T, Narrow>;
  static constexpr int V = kPiece<T>, kGroups = kThreads / L, kChunk = L * I * V;

  // Rows [first, last) of the group.
  __device__ static inline void rows(int64_t all, int64_t& first, int64_t& last) {
    int64_t group = static_cast<int64_t>(blockIdx.x) * kGroups;
    if constexpr (L == 64) group += __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    else group += threadIdx.x / L;
    const int64_t groups = static_cast<int64_t>(gridDim.x) * kGroups, each = (all + groups - 1) / groups;
    first = group * each;
    last = first + each < all ? first + each : all;
  }
  // The first column of the lane's piece i in the chunk from c0 on.
  __device__ static inline int64_t column(int64_t c0, int i) {
    return c0 + static_cast<int64_t>(i * L + threadIdx.x % L) * V;
  }
  template <bool Once>
  __device__ static inline void load(const T* row, int64_t c0, int64_t width, piece_t<T> (&v)[I]) {
#pragma unroll
    for (int i = 0; i < I; ++i) v[i] = Piece::template load<Once>(row, column(c0, i), width);
  }
  // The packed rows of N choices from j on, ~0 beyond the last.
  template <int N>
  __device__ static inline void places(const RowsArgs& a, const int32_t* place, int64_t r, int j, uint32_t (&p)[N]) {
#pragma unroll
    for (int u = 0; u < N; ++u) p[u] = static_cast<uint32_t>(place[r * a.k + (j + u < a.k ? j + u : a.k - 1)]);
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (j + u >= a.k) p[u] = ~0u;
  }
};

// packed = x's rows, read once and written k times: 32768 x 1024 bf16, k = 8, 104
// us (5.8 TB/s); 16381 x 333 fp32, k = 3, 19 (4.7).  Nontemporal stores: 125 us, which
// the next kernel gains.
template <typename T, int L, int I, bool Narrow>
__global__ __launch_bounds__(kThreads) void pack_choices(RowsArgs a, const T* __restrict__ x,
                                                         const int32_t* __restrict__ place,
                                                         const int32_t* __restrict__ offsets, T* __restrict__ packed) {
  using Tile = ChoiceTile<T, L, I, Narrow>;
  const uint32_t end = kept_rows(a, offsets);
  int64_t r, last;
  for (Tile::rows(a.rows, r, last); r < last; ++r)
    for (int64_t c0 = 0; c0 < a.width; c0 += Tile::kChunk) {
      piece_t<T> raw[I];
      const piece_t<T> none = {};
      Tile::template load<true>(x + r * a.stride, c0, a.width, raw);
      for (int j = 0; j < a.k; j += kTogether) {
        uint32_t p[kTogether];
        Tile::places(a, place, r, j, p);
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
          if (p[u] >= a.choices) continue;
#pragma unroll
          for (int i = 0; i < I; ++i)
            Tile::Piece::store(packed + p[u] * a.width, Tile::column(c0, i), a.width, p[u] < end ? raw[i] : none);
        }
      }
    }
}

// out[r] = sum over its choices of (w or 1) * y[place]: restore, and pack's gradient.
// 32768 x 1024 bf16, k = 8: 105 us (5.8 TB/s); 16381 x 333 fp32, k = 3: 16.6 (5.1).
template <typename T, int L, int I, bool Narrow, bool Weighted>
__global__ __launch_bounds__(kThreads) void add_choices(RowsArgs a, const T* __restrict__ y,
                                                        const float* __restrict__ weights,
                                                        const int32_t* __restrict__ place,
                                                        const int32_t* __restrict__ offsets, T* __restrict__ out) {
  using Tile = ChoiceTile<T, L, I, Narrow>;
  constexpr int V = Tile::V;
  const uint32_t end = kept_rows(a, offsets);
  int64_t r, last;
  for (Tile::rows(a.rows, r, last); r < last; ++r)
    for (int64_t c0 = 0; c0 < a.width; c0 += Tile::kChunk) {
      float sum[I][V] = {};
      for (int j = 0; j < a.k; j += kTogether) {
        piece_t<T> raw[kTogether][I];
        uint32_t p[kTogether];
        float w[kTogether];
        Tile::places(a, place, r, j, p);
#pragma unroll
        for (int u = 0; u < kTogether; ++u) w[u] = Weighted ? weights[r * a.k + (j + u < a.k ? j + u : a.k - 1)] : 1.0f;
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
#pragma unroll
          for (int i = 0; i < I; ++i) raw[u][i] = {};
          if (p[u] < end) Tile::template load<true>(y + p[u] * a.stride, c0, a.width, raw[u]);
          else w[u] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kTogether; ++u)
#pragma unroll
          for (int i = 0; i < I; ++i)
#pragma unroll
            for (int q = 0; q < V; ++q) sum[i][q] = __builtin_fmaf(w[u], static_cast<float>(raw[u][i][q]), sum[i][q]);
      }
#pragma unroll
      for (int i = 0; i < I; ++i)
        Tile::Piece::template store<true>(out + r * a.width, Tile::column(c0, i), a.width, sum[i]);
    }
}

// dy and dw of restore.  The products of grad's row with its choices' rows are
// summed over the row's lanes.  As much is read as written, at the rate of a copy:
// 32768 x 1024 bf16, k = 8, 239 us (4.8 TB/s); 16381 x 333 fp32, k = 3, 31 (5.0).
template <typename T, int L, int I, bool Narrow>
__global__ __launch_bounds__(kThreads) void restore_grad(RowsArgs a, const T* __restrict__ y,
                                                         const float* __restrict__ weights,
                                                         const int32_t* __restrict__ place,
                                                         const int32_t* __restrict__ offsets,
                                                         const T* __restrict__ grad, T* __restrict__ dy,
                                                         float* __restrict__ dw) {
  using Tile = ChoiceTile<T, L, I, Narrow>;
  constexpr int V = Tile::V, kBatch = kTogether / 2;
  const uint32_t end = kept_rows(a, offsets);
  int64_t r, last;
  for (Tile::rows(a.rows, r, last); r < last; ++r)
    for (int j = 0; j < a.k; j += kBatch) {
      uint32_t p[kBatch];
      float w[kBatch], dot[kBatch] = {};
      Tile::places(a, place, r, j, p);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) w[u] = weights[r * a.k + (j + u < a.k ? j + u : a.k - 1)];
      for (int64_t c0 = 0; c0 < a.width; c0 += Tile::kChunk) {
        piece_t<T> g[I], raw[kBatch][I];
        Tile::template load<false>(grad + r * a.other_stride, c0, a.width, g);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
#pragma unroll
          for (int i = 0; i < I; ++i) raw[u][i] = {};
          if (dw != nullptr && p[u] < end) Tile::template load<true>(y + p[u] * a.stride, c0, a.width, raw[u]);
        }
        if (dy != nullptr) {
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            if (p[u] >= a.choices) continue;
#pragma unroll
            for (int i = 0; i < I; ++i) {
              float v[V];
#pragma unroll
              for (int q = 0; q < V; ++q) v[q] = p[u] < end ? w[u] * static_cast<float>(g[i][q]) : 0.0f;
              Tile::Piece::template store<true>(dy + p[u] * a.width, Tile::column(c0, i), a.width, v);
            }
          }
        }
        if (dw == nullptr) continue;
        // A product of a piece that was moved back counts its own elements alone.
#pragma unroll
        for (int i = 0; i < I; ++i) {
          const int shift = Tile::Piece::shift(Tile::column(c0, i), a.width);
#pragma unroll
          for (int q = 0; q < V; ++q)
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
              dot[u] = q >= shift ? __builtin_fmaf(static_cast<float>(g[i][q]), static_cast<float>(raw[u][i][q]), dot[u])
                                  : dot[u];
        }
      }
      if (dw == nullptr) continue;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float sum = lane_sum<L>(p[u] < end ? dot[u] : 0.0f);
        if (threadIdx.x % L == 0 && j + u < a.k) dw[r * a.k + j + u] = sum;
      }
    }
}

spmm_status check_experts_desc(const spmm_experts_desc* d) {
  if (d == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null descriptor");
  if (!dense_type(d->value_type)) return fail(SPMM_ERR_CONTRACT, "ExpertPlan supports only FP16, BF16 and FP32 tensors");
  if (d->rows < 0 || d->width < 0) return fail(SPMM_ERR_CONTRACT, "ExpertPlan: negative extent");
  if (d->top_k < 1 || d->top_k > kMaxChoices)
    return fail(SPMM_ERR_CONTRACT, "ExpertPlan takes 1 to 64 choices a row, but got " + std::to_string(d->top_k));
  if (d->experts < 1 || d->experts > kMaxCount)
    return fail(SPMM_ERR_CONTRACT, "ExpertPlan takes 1 to 2048 experts, but got " + std::to_string(d->experts));
  if (d->rows > INT32_MAX || d->rows * d->top_k > INT32_MAX || d->width >= (1 << 22))
    return fail(SPMM_ERR_CONTRACT, "ExpertPlan: choices must be below 2^31, the width below 2^22");
  if (d->rows * d->top_k > 1 && d->stride < d->width)
    return fail(SPMM_ERR_CONTRACT, "ExpertPlan: rows overlap");
  return SPMM_OK;
}

RowsArgs rows_args(const spmm_experts_desc* d) {
  return {d->rows, d->width, d->stride, d->grad_stride, static_cast<int32_t>(d->top_k),
          static_cast<int32_t>(d->experts), d->rows * d->top_k};
}

// f(L, I, Narrow) for rows of `width`.
template <typename T, typename F>
void with_row(int64_t width, F f) {
  using std::integral_constant;
  const int64_t pieces = ceil_div(width, kPiece<T>);
  if (width < kPiece<T>) f(integral_constant<int, 8>(), integral_constant<int, 1>(), std::true_type());
  else if (pieces <= 8) f(integral_constant<int, 8>(), integral_constant<int, 1>(), std::false_type());
  else if (pieces <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>(), std::false_type());
  else if (pieces <= 32) f(integral_constant<int, 32>(), integral_constant<int, 1>(), std::false_type());
  else if (pieces <= 64) f(integral_constant<int, 64>(), integral_constant<int, 1>(), std::false_type());
  else f(integral_constant<int, 64>(), integral_constant<int, 2>(), std::false_type());
}

template <int L>
dim3 row_grid(int64_t rows) {
  const int64_t blocks = ceil_div(rows, kThreads / L);
  return dim3(static_cast<unsigned>(blocks < 16384 ? blocks : 16384));
}

template <typename F>
spmm_status with_type(int32_t type, F f) {
  switch (type) {
    case SPMM_VALUE_F16: return f(_Float16());
    case SPMM_VALUE_BF16: return f(static_cast<__bf16>(0.0f));
    default: return f(0.0f);
  }
}

template <bool Weighted>
spmm_status run_add(const spmm_experts_desc* d, const void* y, const float* weights, const int32_t* place,
                    const int32_t* offsets, void* out, hipStream_t s) {
  return with_type(d->value_type, [&](auto zero) {
    using T = decltype(zero);
    with_row<T>(d->width, [&](auto L, auto I, auto Narrow) {
      constexpr int Lanes = decltype(L)::value, Each = decltype(I)::value;
      hipLaunchKernelGGL((add_choices<T, Lanes, Each, decltype(Narrow)::value, Weighted>), row_grid<Lanes>(d->rows),
                         dim3(kThreads), 0, s, rows_args(d), static_cast<const T*>(y), weights, place, offsets,
                         static_cast<T*>(out));
    });
    return check_launch(Weighted ? "expert_restore" : "expert_pack_grad");
  });
}

}  // namespace
}  // namespace spmm

using namespace spmm;

extern "C" {

spmm_status spmm_expert_plan_workspace(int64_t choices, int64_t experts, size_t* bytes) {
  clear_error();
  if (bytes == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null argument");
  if (choices < 0 || choices > INT32_MAX)
    return fail(SPMM_ERR_CONTRACT, "ExpertPlan: choices must be at least 0 and below 2^31");
  if (experts < 1 || experts > kMaxCount)
    return fail(SPMM_ERR_CONTRACT, "ExpertPlan takes 1 to 2048 experts, but got " + std::to_string(experts));
  *bytes = static_cast<size_t>(sort_words(choices, static_cast<int>(experts) + 1)) * 4;
  return SPMM_OK;
}

spmm_status spmm_expert_plan_run(int32_t index_type, const void* ids, int64_t choices, int64_t experts,
                                 int32_t* offsets, int32_t* place, void* workspace, size_t workspace_bytes,
                                 spmm_stream stream) {
  size_t need = 0;
  if (spmm_status st = spmm_expert_plan_workspace(choices, experts, &need)) return st;
  if (index_type != SPMM_INDEX_I32 && index_type != SPMM_INDEX_I64)
    return fail(SPMM_ERR_CONTRACT, "ExpertPlan: experts must be int32 or int64");
  if (offsets == nullptr || (choices > 0 && (ids == nullptr || place == nullptr)))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "ExpertPlan: null device pointer");
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(SPMM_ERR_CONTRACT, "ExpertPlan: workspace too small: need " + std::to_string(need) + " bytes");
  const int bins = static_cast<int>(experts) + 1;
  const ChoiceKeys keys = {ids, index_type == SPMM_INDEX_I64, experts};
  if (choices <= kRankMost)
    return sort_by_rank(choices, bins, keys, PutPlace{place}, PutOffsets{offsets}, as_stream(stream));
  return sort_digit(Digit{0, bits_of(experts), bins}, choices, keys, static_cast<uint32_t*>(workspace),
                    PutPlace{place}, PutOffsets{offsets}, as_stream(stream));
}

spmm_status spmm_expert_pack_run(const spmm_experts_desc* d, const void* x, const int32_t* place,
                                 const int32_t* offsets, void* packed, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_experts_desc(d)) return st;
  if (d->rows == 0 || d->width == 0) return SPMM_OK;
  if (x == nullptr || place == nullptr || offsets == nullptr || packed == nullptr)
    return fail(SPMM_ERR_INVALID_ARGUMENT, "ExpertPlan: null device pointer");
  return with_type(d->value_type, [&](auto zero) {
    using T = decltype(zero);
    with_row<T>(d->width, [&](auto L, auto I, auto Narrow) {
      constexpr int Lanes = decltype(L)::value, Each = decltype(I)::value;
      hipLaunchKernelGGL((pack_choices<T, Lanes, Each, decltype(Narrow)::value>), row_grid<Lanes>(d->rows),
                         dim3(kThreads), 0, as_stream(stream), rows_args(d), static_cast<const T*>(x), place, offsets,
                         static_cast<T*>(packed));
    });
    return check_launch("expert_pack");
  });
}

spmm_status spmm_expert_pack_grad_run(const spmm_experts_desc* d, const void* grad, const int32_t* place,
                                      const int32_t* offsets, void* dx, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_experts_desc(d)) return st;
  if (d->rows == 0 || d->width == 0) return SPMM_OK;
  if (grad == nullptr || place == nullptr || offsets == nullptr || dx == nullptr)
    return fail(SPMM_ERR_INVALID_ARGUMENT, "ExpertPlan: null device pointer");
  return run_add<false>(d, grad, nullptr, place, offsets, dx, as_stream(stream));
}

spmm_status spmm_expert_restore_run(const spmm_experts_desc* d, const void* y, const float* weights,
                                    const int32_t* place, const int32_t* offsets, void* out, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_experts_desc(d)) return st;
  if (d->rows == 0 || d->width == 0) return SPMM_OK;
  if (y == nullptr || weights == nullptr || place == nullptr || offsets == nullptr || out == nullptr)
    return fail(SPMM_ERR_INVALID_ARGUMENT, "ExpertPlan: null device pointer");
  return run_add<true>(d, y, weights, place, offsets, out, as_stream(stream));
}

spmm_status spmm_expert_restore_grad_run(const spmm_experts_desc* d, const void* y, const float* weights,
                                         const int32_t* place, const int32_t* offsets, const void* grad, void* dy,
                                         float* dweights, spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_experts_desc(d)) return st;
  if (d->rows > 1 && d->grad_stride < d->width) return fail(SPMM_ERR_CONTRACT, "ExpertPlan: rows of grad overlap");
  if (d->rows == 0 || (dy == nullptr && dweights == nullptr)) return SPMM_OK;
  // The kernel reads the weights of rows of no columns too.
  if (place == nullptr || offsets == nullptr || weights == nullptr ||
      (d->width > 0 && (y == nullptr || grad == nullptr)))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "ExpertPlan: null device pointer");
  return with_type(d->value_type, [&](auto zero) {
    using T = decltype(zero);
    with_row<T>(d->width, [&](auto L, auto I, auto Narrow) {
      constexpr int Lanes = decltype(L)::value, Each = decltype(I)::value;
      hipLaunchKernelGGL((restore_grad<T, Lanes, Each, decltype(Narrow)::value>), row_grid<Lanes>(d->rows),
                         dim3(kThreads), 0, as_stream(stream), rows_args(d), static_cast<const T*>(y), weights, place, offsets,
                         static_cast<const T*>(grad), static_cast<T*>(dy), dweights);
    });
    return check_launch("expert_restore_grad");
  });
}

}  // extern "C"
