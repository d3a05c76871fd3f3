// Matrix products grouped by row ranges: out[r] = x[r] W[g] for the rows r of
// group g, with dx[r] = grad[r] W[g]^T and dW[g] = x_g^T grad_g.
#include <climits>
#include <type_traits>
#include <utility>

#include "fma_tile.h"

namespace spmm {
namespace {

struct GroupedArgs {
  int64_t rows, groups;
  int64_t inner, width;  // of the product at hand: depth and output columns
  int64_t in_stride;     // rows of its left operand
  int64_t weight_stride, w_depth, w_col;
};

template <typename I>
__device__ inline int64_t edge(const I* offsets, int64_t g, int64_t rows) {
  const int64_t v = static_cast<int64_t>(offsets[g]);
  return v < 0 ? 0 : v > rows ? rows : v;
}

// The `tile`-th tile of `height` rows, none across a group's end.  Segment 0
// is the rows before the first group, segment groups + 1 those behind the
// last; both are `group` -1.  False past the last tile.  Every lane of a wave
// calls it and gets the same answer.
struct RowRange {
  int64_t first, rows, group;
};
template <typename I>
__device__ inline bool find_rows(const I* offsets, int64_t groups, int64_t rows, int64_t height, int64_t tile,
                                 RowRange& found) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int64_t s0 = 0; s0 < groups + 2; s0 += 64) {
    const int64_t s = s0 + lane;
    int64_t lo = 0, hi = 0;
    if (s < groups + 2) {
      lo = s == 0 ? 0 : edge(offsets, s - 1, rows);
      hi = s == groups + 1 ? rows : edge(offsets, s, rows);
    }
    const int64_t mine = hi > lo ? (hi - lo + height - 1) / height : 0;
    int64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    const unsigned long long past = __ballot(before + upto > tile);
    if (past != 0) {
      const int at = __ffsll(past) - 1;
      const int64_t start = __shfl(lo, at) + (tile - before - __shfl(upto - mine, at)) * height;
      const int64_t end = __shfl(hi, at);
      found.first = start;
      found.rows = end - start < height ? end - start : height;
      found.group = s0 + at == 0 || s0 + at == groups + 1 ? -1 : s0 + at - 1;
      return true;
    }
    before += __shfl(upto, 63);
  }
  return false;
}

// Row tiles times column tiles, the latter fastest.
template <typename T, typename I>
__global__ __launch_bounds__(kThreads) void grouped_rows(GroupedArgs a, const T* __restrict__ in,
                                                         const T* __restrict__ weight,
                                                         const I* __restrict__ offsets, T* __restrict__ out) {
  const int64_t across = (a.width + kTile - 1) / kTile;
  RowRange r;
  if (!find_rows(offsets, a.groups, a.rows, kTile, blockIdx.x / across, r)) return;
  const int64_t c0 = blockIdx.x % across * kTile;
  const int64_t cols = a.width - c0 < kTile ? a.width - c0 : kTile;
  float acc[4][4] = {};
  if (r.group >= 0)
    multiply_tile<T>({in + r.first * a.in_stride, a.in_stride, 1},
                     {weight + r.group * a.weight_stride + c0 * a.w_col, a.w_col, a.w_depth}, r.rows, cols, a.inner, acc);
  store_tile(out + r.first * a.width + c0, a.width, r.rows, cols, acc);
}

// dW[g]: `left` columns by `right` columns, summed over the group's rows.
template <typename T, typename I>
__global__ __launch_bounds__(kThreads) void grouped_weights(GroupedArgs a, const T* __restrict__ left,
                                                            int64_t left_stride, const T* __restrict__ right,
                                                            int64_t right_stride, const I* __restrict__ offsets,
                                                            T* __restrict__ dweight) {
  const int64_t across = (a.width + kTile - 1) / kTile, down = (a.inner + kTile - 1) / kTile;
  const int64_t g = blockIdx.x / (across * down);
  const int64_t i0 = blockIdx.x / across % down * kTile, c0 = blockIdx.x % across * kTile;
  const int64_t rows = a.inner - i0 < kTile ? a.inner - i0 : kTile;
  const int64_t cols = a.width - c0 < kTile ? a.width - c0 : kTile;
  const int64_t lo = edge(offsets, g, a.rows), hi = edge(offsets, g + 1, a.rows);
  float acc[4][4] = {};
  multiply_tile<T>({left + lo * left_stride + i0, 1, left_stride}, {right + lo * right_stride + c0, 1, right_stride},
                   rows, cols, hi > lo ? hi - lo : 0, acc);
  store_tile(dweight + (g * a.inner + i0) * a.width + c0, a.width, rows, cols, acc);
}

spmm_status check_grouped_desc(const spmm_grouped_desc* d, const char* op) {
  if (d == nullptr) return fail(SPMM_ERR_INVALID_ARGUMENT, "null descriptor");
  if (d->index_type != SPMM_INDEX_I32 && d->index_type != SPMM_INDEX_I64)
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": offsets must be int32 or int64");
  if (!dense_type(d->value_type))
    return fail(SPMM_ERR_CONTRACT, std::string(op) + " supports only FP16, BF16 and FP32 tensors");
  if (d->rows < 0 || d->groups < 0 || d->inner < 0 || d->width < 0)
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": negative extent");
  if (d->inner > INT32_MAX || d->width > INT32_MAX)
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": inner and width must be below 2^31");
  if (d->rows > 1 && d->x_stride < d->inner) return fail(SPMM_ERR_CONTRACT, std::string(op) + ": rows of x overlap");
  if (d->groups > 1 && d->weight_stride < d->inner * d->width)
    return fail(SPMM_ERR_CONTRACT, std::string(op) + ": matrices of weight overlap");
  return SPMM_OK;
}

// Work-groups of a launch: a grid's limit is an error, not a wrapped count.
spmm_status check_grid(int64_t blocks, const char* op) {
  if (blocks > INT32_MAX) return fail(SPMM_ERR_OVERFLOW, std::string(op) + ": too many tiles for one launch");
  return SPMM_OK;
}

// The weight's steps along the depth and the columns of the product x W, or
// of grad W^T where `back`.
GroupedArgs rows_args(const spmm_grouped_desc* d, bool back) {
  const int64_t inner_step = d->weight_transposed ? 1 : d->width, width_step = d->weight_transposed ? d->inner : 1;
  if (back)
    return {d->rows, d->groups, d->width, d->inner, d->grad_stride, d->weight_stride, width_step, inner_step};
  return {d->rows, d->groups, d->inner, d->width, d->x_stride, d->weight_stride, inner_step, width_step};
}

template <typename T, typename I>
spmm_status run_rows(const GroupedArgs& a, const void* in, const void* weight, const void* offsets, void* out,
                     hipStream_t s, const char* op) {
  if (a.rows == 0 || a.width == 0) return SPMM_OK;
  const int64_t blocks = (ceil_div(a.rows, kTile) + a.groups + 1) * ceil_div(a.width, kTile);
  if (spmm_status st = check_grid(blocks, op)) return st;
  hipLaunchKernelGGL((grouped_rows<T, I>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s, a,
                     static_cast<const T*>(in), static_cast<const T*>(weight), static_cast<const I*>(offsets),
                     static_cast<T*>(out));
  return check_launch(op);
}

template <typename T, typename I>
spmm_status run_weights(const spmm_grouped_desc* d, const void* x, const void* grad, const void* offsets, void* dweight,
                        hipStream_t s, const char* op) {
  if (d->groups == 0 || d->inner == 0 || d->width == 0) return SPMM_OK;
  const T *tx = static_cast<const T*>(x), *tg = static_cast<const T*>(grad);
  GroupedArgs a{d->rows, d->groups, d->inner, d->width, 0, 0, 0, 0};
  if (d->weight_transposed) std::swap(a.inner, a.width);
  const int64_t blocks = ceil_div(a.inner, kTile) * ceil_div(a.width, kTile) * a.groups;
  if (spmm_status st = check_grid(blocks, op)) return st;
  hipLaunchKernelGGL((grouped_weights<T, I>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s, a,
                     d->weight_transposed ? tg : tx, d->weight_transposed ? d->grad_stride : d->x_stride,
                     d->weight_transposed ? tx : tg, d->weight_transposed ? d->x_stride : d->grad_stride,
                     static_cast<const I*>(offsets), static_cast<T*>(dweight));
  return check_launch(op);
}

// Calls f with null pointers of the value and index types.
template <typename F>
spmm_status with_types(const spmm_grouped_desc* d, F f) {
  auto indexed = [&](auto* t) {
    return d->index_type == SPMM_INDEX_I32 ? f(t, static_cast<int32_t*>(nullptr)) : f(t, static_cast<int64_t*>(nullptr));
  };
  switch (d->value_type) {
    case SPMM_VALUE_F16: return indexed(static_cast<_Float16*>(nullptr));
    case SPMM_VALUE_BF16: return indexed(static_cast<__bf16*>(nullptr));
    default: return indexed(static_cast<float*>(nullptr));
  }
}
template <typename P>
using value_of = std::remove_pointer_t<P>;

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
  return with_types(d, [&](auto* t, auto* i) {
    return run_rows<value_of<decltype(t)>, value_of<decltype(i)>>(rows_args(d, false), x, weight, offsets, out,
                                                                  as_stream(stream), "grouped_matmul");
  });
}

spmm_status spmm_grouped_grad_workspace(const spmm_grouped_desc* d, size_t* bytes) {
  return spmm_grouped_workspace(d, bytes);
}

spmm_status spmm_grouped_grad_run(const spmm_grouped_desc* d, const void* x, const void* weight, const void* offsets,
                                  const void* grad, void* dx, void* dweight, void* workspace, size_t workspace_bytes,
                                  spmm_stream stream) {
  clear_error();
  if (spmm_status st = check_grouped_desc(d, "grouped_matmul")) return st;
  if (d->rows > 1 && d->grad_stride < d->width)
    return fail(SPMM_ERR_CONTRACT, "grouped_matmul: rows of grad overlap");
  if (offsets == nullptr || (d->rows > 0 && d->width > 0 && grad == nullptr) ||
      (dx != nullptr && d->groups > 0 && d->inner > 0 && d->width > 0 && weight == nullptr) ||
      (dweight != nullptr && d->rows > 0 && d->inner > 0 && x == nullptr))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "grouped_matmul: null device pointer");
  (void)workspace;
  (void)workspace_bytes;
  return with_types(d, [&](auto* t, auto* i) {
    using T = value_of<decltype(t)>;
    using I = value_of<decltype(i)>;
    if (dx != nullptr)
      if (spmm_status st = run_rows<T, I>(rows_args(d, true), grad, weight, offsets, dx, as_stream(stream),
                                          "grouped_matmul gradient"))
        return st;
    if (dweight == nullptr) return SPMM_OK;
    return run_weights<T, I>(d, x, grad, offsets, dweight, as_stream(stream), "grouped_matmul gradient");
  });
}

}  // extern "C"
