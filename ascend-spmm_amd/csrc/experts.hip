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
#include "numeric.h"
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

template <typename T>
__device__ inline void store_raw(T* p, int64_t n, const piece_t<T>& v) {
  if (n >= kPiece<T>) {
    *reinterpret_cast<piece_t<T>*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i)
      if (i < n) p[i] = v[i];
  }
}

// The kernels' common walk: L lanes a row, which take L * I pieces of 16 bytes of
// it at a time, and kTogether choices, whose rows' loads are all under way
// together.  A whole wave's row is a scalar, and so are the loads of its places
// and weights.
constexpr int kTogether = 8;

template <typename T, int L, int I>
struct ChoiceTile {
  static constexpr int V = kPiece<T>, kGroups = kThreads / L, kChunk = L * I * V;

  __device__ static inline int64_t first_row() {
    int64_t group = static_cast<int64_t>(blockIdx.x) * kGroups;
    if constexpr (L == 64) group += __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    else group += threadIdx.x / L;
    return group;
  }
  __device__ static inline int64_t row_step() { return static_cast<int64_t>(gridDim.x) * kGroups; }
  // The first column of the lane's piece i in the chunk from c0 on.
  __device__ static inline int64_t column(int64_t c0, int i) {
    return c0 + static_cast<int64_t>(i * L + threadIdx.x % L) * V;
  }
  __device__ static inline void load(const T* row, int64_t c0, int64_t width, piece_t<T> (&v)[I]) {
#pragma unroll
    for (int i = 0; i < I; ++i) v[i] = load_raw(row + column(c0, i), width - column(c0, i));
  }
};

// packed = x's rows, read once and written k times.
template <typename T, int L, int I>
__global__ __launch_bounds__(kThreads) void pack_choices(RowsArgs a, const T* __restrict__ x,
                                                         const int32_t* __restrict__ place,
                                                         const int32_t* __restrict__ offsets, T* __restrict__ packed) {
  using Tile = ChoiceTile<T, L, I>;
  const uint32_t end = kept_rows(a, offsets);
  for (int64_t r = Tile::first_row(); r < a.rows; r += Tile::row_step())
    for (int64_t c0 = 0; c0 < a.width; c0 += Tile::kChunk) {
      piece_t<T> raw[I];
      const piece_t<T> none = {};
      Tile::load(x + r * a.stride, c0, a.width, raw);
      for (int j = 0; j < a.k; ++j) {
        const uint32_t p = place[r * a.k + j];
        if (p >= a.choices) continue;
#pragma unroll
        for (int i = 0; i < I; ++i) {
          const int64_t c = Tile::column(c0, i);
          store_raw(packed + p * a.width + c, a.width - c, p < end ? raw[i] : none);
        }
      }
    }
}

// out[r] = sum over its choices of (w or 1) * y[place]: restore, and pack's gradient.
template <typename T, int L, int I, bool Weighted>
__global__ __launch_bounds__(kThreads) void add_choices(RowsArgs a, const T* __restrict__ y,
                                                        const float* __restrict__ weights,
                                                        const int32_t* __restrict__ place,
                                                        const int32_t* __restrict__ offsets, T* __restrict__ out) {
  using Tile = ChoiceTile<T, L, I>;
  constexpr int V = Tile::V;
  const uint32_t end = kept_rows(a, offsets);
  for (int64_t r = Tile::first_row(); r < a.rows; r += Tile::row_step())
    for (int64_t c0 = 0; c0 < a.width; c0 += Tile::kChunk) {
      float sum[I][V] = {};
      for (int j = 0; j < a.k; j += kTogether) {
        piece_t<T> raw[kTogether][I];
        float w[kTogether];
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
          const uint32_t p = j + u < a.k ? static_cast<uint32_t>(place[r * a.k + j + u]) : ~0u;
          w[u] = p < end ? (Weighted ? weights[r * a.k + j + u] : 1.0f) : 0.0f;
          if (p < end) {
            Tile::load(y + p * a.stride, c0, a.width, raw[u]);
          } else {
#pragma unroll
            for (int i = 0; i < I; ++i) raw[u][i] = {};
          }
        }
#pragma unroll
        for (int u = 0; u < kTogether; ++u)
#pragma unroll
          for (int i = 0; i < I; ++i)
#pragma unroll
            for (int q = 0; q < V; ++q) sum[i][q] = __builtin_fmaf(w[u], static_cast<float>(raw[u][i][q]), sum[i][q]);
      }
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int64_t c = Tile::column(c0, i);
        store_piece(out + r * a.width + c, a.width - c, sum[i]);
      }
    }
}

// dy and dw of restore.  The products of grad's row with its choices' rows are
// summed over the row's lanes.
template <typename T, int L, int I>
__global__ __launch_bounds__(kThreads) void restore_grad(RowsArgs a, const T* __restrict__ y,
                                                         const float* __restrict__ weights,
                                                         const int32_t* __restrict__ place,
                                                         const int32_t* __restrict__ offsets,
                                                         const T* __restrict__ grad, T* __restrict__ dy,
                                                         float* __restrict__ dw) {
  using Tile = ChoiceTile<T, L, I>;
  constexpr int V = Tile::V, kBatch = kTogether / 2;
  const uint32_t end = kept_rows(a, offsets);
  for (int64_t r = Tile::first_row(); r < a.rows; r += Tile::row_step())
    for (int j = 0; j < a.k; j += kBatch) {
      uint32_t p[kBatch];
      float w[kBatch], dot[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        p[u] = j + u < a.k ? static_cast<uint32_t>(place[r * a.k + j + u]) : ~0u;
        w[u] = p[u] < end ? weights[r * a.k + j + u] : 0.0f;
        dot[u] = 0.0f;
      }
      for (int64_t c0 = 0; c0 < a.width; c0 += Tile::kChunk) {
        piece_t<T> g[I], raw[kBatch][I];
        Tile::load(grad + r * a.other_stride, c0, a.width, g);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (dw != nullptr && p[u] < end) {
            Tile::load(y + p[u] * a.stride, c0, a.width, raw[u]);
          } else {
#pragma unroll
            for (int i = 0; i < I; ++i) raw[u][i] = {};
          }
        }
        if (dy != nullptr) {
#pragma unroll
          for (int u = 0; u < kBatch; ++u)
            if (p[u] < a.choices)
#pragma unroll
              for (int i = 0; i < I; ++i) {
                const int64_t c = Tile::column(c0, i);
                float v[V];
#pragma unroll
                for (int q = 0; q < V; ++q) v[q] = p[u] < end ? w[u] * static_cast<float>(g[i][q]) : 0.0f;
                store_piece(dy + p[u] * a.width + c, a.width - c, v);
              }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
          for (int i = 0; i < I; ++i)
#pragma unroll
            for (int q = 0; q < V; ++q)
              dot[u] = p[u] < end ? __builtin_fmaf(static_cast<float>(g[i][q]), static_cast<float>(raw[u][i][q]), dot[u])
                                  : 0.0f;
      }
      if (dw == nullptr) continue;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float sum = lane_sum<L>(dot[u]);
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
  return {d->rows, d->width, d->stride, d->grad_stride, static_cast<int32_t>(d->top_k), static_cast<int32_t>(d->experts),
          d->rows * d->top_k};
}

template <typename T, typename F>
void with_row(int64_t width, F f) {
  using std::integral_constant;
  const int64_t pieces = ceil_div(width, kPiece<T>);
  if (pieces <= 8) f(integral_constant<int, 8>(), integral_constant<int, 1>());
  else if (pieces <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (pieces <= 32) f(integral_constant<int, 32>(), integral_constant<int, 1>());
  else if (pieces <= 64) f(integral_constant<int, 64>(), integral_constant<int, 1>());
  else f(integral_constant<int, 64>(), integral_constant<int, 2>());
}

template <int L>
dim3 row_grid(int64_t rows) {
  const int64_t blocks = ceil_div(rows, kThreads / L);
  return dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536));
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
    with_row<T>(d->width, [&](auto L, auto I) {
      hipLaunchKernelGGL((add_choices<T, decltype(L)::value, decltype(I)::value, Weighted>), row_grid<decltype(L)::value>(d->rows),
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
    with_row<T>(d->width, [&](auto L, auto I) {
      hipLaunchKernelGGL((pack_choices<T, decltype(L)::value, decltype(I)::value>), row_grid<decltype(L)::value>(d->rows), dim3(kThreads), 0,
                         as_stream(stream), rows_args(d), static_cast<const T*>(x), place, offsets,
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
  if (place == nullptr || offsets == nullptr ||
      (d->width > 0 && (y == nullptr || weights == nullptr || grad == nullptr)))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "ExpertPlan: null device pointer");
  return with_type(d->value_type, [&](auto zero) {
    using T = decltype(zero);
    with_row<T>(d->width, [&](auto L, auto I) {
      hipLaunchKernelGGL((restore_grad<T, decltype(L)::value, decltype(I)::value>), row_grid<decltype(L)::value>(d->rows), dim3(kThreads), 0,
                         as_stream(stream), rows_args(d), static_cast<const T*>(y), weights, place, offsets,
                         static_cast<const T*>(grad), static_cast<T*>(dy), dweights);
    });
    return check_launch("expert_restore_grad");
  });
}

}  // extern "C"
