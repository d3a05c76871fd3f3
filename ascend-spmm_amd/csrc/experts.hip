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

// packed = x's rows: L lanes a row, which read it once and write it k times.
template <typename T, int L>
__global__ __launch_bounds__(kThreads) void pack_choices(RowsArgs a, const T* __restrict__ x,
                                                         const int32_t* __restrict__ place,
                                                         const int32_t* __restrict__ offsets, T* __restrict__ packed) {
  constexpr int V = kPiece<T>, kGroups = kThreads / L;
  const int lane = threadIdx.x % L;
  const uint32_t end = kept_rows(a, offsets);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / L; r < a.rows; r += step)
    for (int64_t c = lane * V; c < a.width; c += L * V) {
      const piece_t<T> raw = load_raw(x + r * a.stride + c, a.width - c), none = {};
      for (int j = 0; j < a.k; ++j) {
        const uint32_t p = place[r * a.k + j];
        if (p < a.choices) store_raw(packed + p * a.width + c, a.width - c, p < end ? raw : none);
      }
    }
}

// out[r] = sum over its choices of (w or 1) * y[place]: restore, and pack's gradient.
constexpr int kTogether = 4;  // rows loaded at a time
template <typename T, int L, bool Weighted>
__global__ __launch_bounds__(kThreads) void add_choices(RowsArgs a, const T* __restrict__ y,
                                                        const float* __restrict__ weights,
                                                        const int32_t* __restrict__ place,
                                                        const int32_t* __restrict__ offsets, T* __restrict__ out) {
  constexpr int V = kPiece<T>, kGroups = kThreads / L;
  const int lane = threadIdx.x % L;
  const uint32_t end = kept_rows(a, offsets);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / L; r < a.rows; r += step)
    for (int64_t c = lane * V; c < a.width; c += L * V) {
      float sum[V] = {};
      for (int j = 0; j < a.k; j += kTogether) {
        piece_t<T> raw[kTogether];
        float w[kTogether];
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
          raw[u] = {};
          w[u] = 0.0f;
          if (j + u >= a.k) continue;
          const uint32_t p = place[r * a.k + j + u];
          if (p >= end) continue;
          raw[u] = load_raw(y + p * a.stride + c, a.width - c);
          w[u] = Weighted ? weights[r * a.k + j + u] : 1.0f;
        }
#pragma unroll
        for (int u = 0; u < kTogether; ++u)
#pragma unroll
          for (int i = 0; i < V; ++i) sum[i] = __builtin_fmaf(w[u], static_cast<float>(raw[u][i]), sum[i]);
      }
      store_piece(out + r * a.width + c, a.width - c, sum);
    }
}

// dy and dw of restore.  L lanes a row; each choice's product of two rows is
// summed over them.
template <typename T, int L>
__global__ __launch_bounds__(kThreads) void restore_grad(RowsArgs a, const T* __restrict__ y,
                                                         const float* __restrict__ weights,
                                                         const int32_t* __restrict__ place,
                                                         const int32_t* __restrict__ offsets,
                                                         const T* __restrict__ grad, T* __restrict__ dy,
                                                         float* __restrict__ dw) {
  constexpr int V = kPiece<T>, kGroups = kThreads / L;
  const int lane = threadIdx.x % L;
  const uint32_t end = kept_rows(a, offsets);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / L; r < a.rows; r += step)
    for (int j = 0; j < a.k; ++j) {
      const int64_t at = r * a.k + j;
      const uint32_t p = place[at];
      const bool kept = p < end;
      const float w = kept ? weights[at] : 0.0f;
      float dot = 0.0f;
      for (int64_t c = lane * V; c < a.width; c += L * V) {
        float g[V], v[V];
        load_piece(grad + r * a.other_stride + c, a.width - c, g);
        if (dw != nullptr && kept) {
          load_piece(y + p * a.stride + c, a.width - c, v);
#pragma unroll
          for (int i = 0; i < V; ++i) dot = __builtin_fmaf(g[i], v[i], dot);
        }
        if (dy != nullptr && p < a.choices) {
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] = kept ? w * g[i] : 0.0f;
          store_piece(dy + p * a.width + c, a.width - c, v);
        }
      }
      if (dw == nullptr) continue;
      dot = lane_sum<L>(dot);
      if (lane == 0) dw[at] = dot;
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
  const int64_t pieces = ceil_div(width, kPiece<T>);
  if (pieces <= 8) f(std::integral_constant<int, 8>());
  else if (pieces <= 16) f(std::integral_constant<int, 16>());
  else if (pieces <= 32) f(std::integral_constant<int, 32>());
  else f(std::integral_constant<int, 64>());
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
    with_row<T>(d->width, [&](auto L) {
      hipLaunchKernelGGL((add_choices<T, decltype(L)::value, Weighted>), row_grid<decltype(L)::value>(d->rows),
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
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SPMM_ERR_CONTRACT, "ExpertPlan: workspace too small: need " + std::to_string(need) + " bytes");
  const int bins = static_cast<int>(experts) + 1;
  return sort_digit(Digit{0, bits_of(experts), bins}, choices, ChoiceKeys{ids, index_type == SPMM_INDEX_I64, experts},
                    static_cast<uint32_t*>(workspace), PutPlace{place}, PutOffsets{offsets}, as_stream(stream));
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
    with_row<T>(d->width, [&](auto L) {
      hipLaunchKernelGGL((pack_choices<T, decltype(L)::value>), row_grid<decltype(L)::value>(d->rows), dim3(kThreads), 0,
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
    with_row<T>(d->width, [&](auto L) {
      hipLaunchKernelGGL((restore_grad<T, decltype(L)::value>), row_grid<decltype(L)::value>(d->rows), dim3(kThreads), 0,
                         as_stream(stream), rows_args(d), static_cast<const T*>(y), weights, place, offsets,
                         static_cast<const T*>(grad), static_cast<T*>(dy), dweights);
    });
    return check_launch("expert_restore_grad");
  });
}

}  // extern "C"
