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
#include "numeric.h"

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

// Order of doubles as whole numbers; NaN above all, so that it is chosen and seen.
__device__ inline uint64_t wide_key(double v) {
  if (v != v) return ~uint64_t(0);
  const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
  return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}
constexpr uint64_t kWideMinusInf = 0x000FFFFFFFFFFFFFull;
__device__ inline uint64_t narrow_key(float v) { return v != v ? 0xFFFFFFFFull : order_key(v); }

template <int L>
__device__ inline double lane_sum64(double v) {
#pragma unroll
  for (int d = 1; d < L; d <<= 1) v += __shfl_xor(v, d, L);
  return v;
}

// Greatest key over L lanes and the lowest index that has it.
template <int L>
__device__ inline void lane_best(uint64_t& key, uint32_t& at) {
  const uint32_t own_high = static_cast<uint32_t>(key >> 32), own_low = static_cast<uint32_t>(key);
  const uint32_t high = lane_max<L>(own_high);
  const uint32_t low = lane_max<L>(own_high == high ? own_low : 0u);
  at = lane_min<L>(own_high == high && own_low == low ? at : 0xFFFFFFFFu);
  key = (static_cast<uint64_t>(high) << 32) | low;
}

// L lanes a row, N logits a lane: expert lane + i * L.  Wide: selection values
// in 64 bits (a bias or groups).
template <typename T, int L, int N, bool Wide>
__global__ __launch_bounds__(kThreads) void route_rows(RouteArgs a, const T* __restrict__ logits,
                                                       const float* __restrict__ bias, float* __restrict__ weights,
                                                       int32_t* __restrict__ chosen, float* stats) {
  constexpr int kGroups = kThreads / L;
  __shared__ double values[Wide ? kGroups * L * N : 1];
  const int lane = threadIdx.x % L;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  // All lanes of the work-group take part in every round (barriers).
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * kGroups; r0 < a.rows; r0 += step) {
    const int64_t r = r0 + threadIdx.x / L;
    const bool live = r < a.rows;
    const T* row = logits + (live ? r : 0) * a.stride;
    float x[N], m = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = lane + i * L < a.experts ? static_cast<float>(row[lane + i * L]) : -INFINITY;
      m = fmaxf(m, x[i]);
    }
    float ls = 0.0f;
    m = lane_max<L>(m);
    if (!a.sigmoid) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) s += expf(x[i] - m);
      ls = logf(lane_sum<L>(s));
    }
    uint64_t key[N];
    if constexpr (Wide) {
      double v[N], total = 0.0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const double d = x[i];
        v[i] = a.sigmoid ? 1.0 / (1.0 + exp(-d)) : exp(d - static_cast<double>(m));
        total += v[i];
      }
      if (!a.sigmoid) {
        total = lane_sum64<L>(total);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] /= total;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float b = bias != nullptr && lane + i * L < a.experts ? bias[lane + i * L] : 0.0f;
        v[i] = x[i] == -INFINITY || b == -INFINITY ? -static_cast<double>(INFINITY) : v[i] + b;
        key[i] = wide_key(v[i]);
      }
      if (a.groups > 1) {
        // A group's value is the sum of its two greatest: lane g looks through group g.
        double* mine = values + (threadIdx.x / L) * L * N;
        const int size = a.experts / a.groups;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (lane + i * L < a.experts) mine[lane + i * L] = v[i];
        __syncthreads();
        uint64_t group_key = 0;
        bool open = false;
        if (lane < a.groups) {
          double first = -static_cast<double>(INFINITY), second = first;
          bool nan = false;
          for (int e = 0; e < size; ++e) {
            const double d = mine[lane * size + e];
            nan |= d != d;
            if (d > first) {
              second = first;
              first = d;
            } else if (d > second) {
              second = d;
            }
          }
          group_key = nan ? ~uint64_t(0) : wide_key(first + (second == -static_cast<double>(INFINITY) ? 0.0 : second));
          if (!nan && first == -static_cast<double>(INFINITY)) group_key = kWideMinusInf;
        }
        int rank = 0;
        for (int g = 0; g < a.groups; ++g) {
          const uint64_t other = __shfl(group_key, g, L);
          rank += other > group_key || (other == group_key && g < lane);
        }
        open = lane < a.groups && rank < a.top_groups;
        const uint64_t opened = __ballot(open) >> (threadIdx.x & 63 & ~(L - 1));
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (lane + i * L < a.experts && !((opened >> ((lane + i * L) / size)) & 1u)) key[i] = kWideMinusInf;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) key[i] = narrow_key(x[i]);
    }
    const uint64_t none = Wide ? kWideMinusInf : static_cast<uint64_t>(kKeyOfMinusInf);
    // Lane j keeps choice j (and j + L, ...): its expert and log score.
    constexpr int K = (kMaxTopK + L - 1) / L;
    int32_t ids[K];
    float score[K], most = -INFINITY;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      ids[c] = -1;
      score[c] = -INFINITY;
    }
    for (int q = 0; q < a.k; ++q) {
      uint64_t best = 0;
      uint32_t at = 0;
      float value = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (key[i] > best) {
          best = key[i];
          at = lane + i * L;
          value = x[i];
        }
      const uint32_t own = at;
      lane_best<L>(best, at);
      if (best <= none) break;  // no expert is left; the same on all lanes of the row
      const bool winner = own == at && own % L == static_cast<uint32_t>(lane);
      // The winner's logit, for all lanes of the row: its order and bits by a maximum.
      const uint32_t bits = lane_max<L>(winner ? as_bits(value) : 0u);
      const float xj = as_float(bits);
      const float l = a.sigmoid ? log_sigmoid(xj) : (xj - m) - ls;
      most = fmaxf(most, l);
#pragma unroll
      for (int c = 0; c < K; ++c)
        if (q == lane + c * L) {
          ids[c] = static_cast<int32_t>(at);
          score[c] = l;
        }
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (lane + i * L == static_cast<int>(at)) key[i] = 0;
    }
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      score[c] = ids[c] < 0 ? 0.0f : expf(a.renormalize ? score[c] - most : score[c]);
      sum += score[c];
    }
    const float over = a.renormalize ? lane_sum<L>(sum) : 1.0f;
    if (!live) continue;
#pragma unroll
    for (int c = 0; c < K; ++c)
      if (lane + c * L < a.k) {
        weights[r * a.k + lane + c * L] = ids[c] < 0 ? 0.0f : a.scale * (score[c] / over);
        chosen[r * a.k + lane + c * L] = ids[c];
      }
    if (stats != nullptr && lane == 0) {
      stats[2 * r] = m;
      stats[2 * r + 1] = ls;
    }
  }
}

// dlogits of kRowsLds / experts rows a work-group, put together in LDS: what
// every expert has of it (softmax that is not renormalised), then the chosen.
constexpr int kRowsLds = 4096;
template <typename T>
__global__ __launch_bounds__(kThreads) void route_grad(RouteArgs a, const T* __restrict__ logits,
                                                       const int32_t* __restrict__ chosen,
                                                       const float* __restrict__ weights,
                                                       const float* __restrict__ stats, const float* __restrict__ grad,
                                                       T* __restrict__ dlogits) {
  __shared__ float out[kRowsLds];
  __shared__ float sums[kRowsLds];  // by row
  const int tile = kRowsLds / a.experts;
  const bool dense = !a.sigmoid && !a.renormalize;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * tile; r0 < a.rows; r0 += static_cast<int64_t>(gridDim.x) * tile) {
    const int rows = static_cast<int>(a.rows - r0 < tile ? a.rows - r0 : tile);
    for (int q = threadIdx.x; q < rows; q += kThreads) {
      float sum = 0.0f;
      for (int j = 0; j < a.k; ++j) {
        const int64_t at = (r0 + q) * a.k + j;
        if (static_cast<uint32_t>(chosen[at]) < static_cast<uint32_t>(a.experts))
          sum += (a.renormalize ? weights[at] / a.scale : weights[at]) * grad[at];
      }
      sums[q] = sum;
    }
    __syncthreads();
    for (int q = threadIdx.x; q < rows * a.experts; q += kThreads) {
      float v = 0.0f;
      if (dense) {
        const int row = q / a.experts;
        const float x = static_cast<float>(logits[(r0 + row) * a.stride + (q - row * a.experts)]);
        const float p = expf((x - stats[2 * (r0 + row)]) - stats[2 * (r0 + row) + 1]);
        v = x == -INFINITY ? 0.0f : -p * sums[row];
      }
      out[q] = v;
    }
    __syncthreads();
    for (int q = threadIdx.x; q < rows * a.k; q += kThreads) {
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
    for (int q = threadIdx.x; q < rows * a.experts; q += kThreads) dlogits[r0 * a.experts + q] = static_cast<T>(out[q]);
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
  if (!(d->scale > 0.0) || !(d->scale <= FLT_MAX))
    return fail(SPMM_ERR_INVALID_ARGUMENT, "route: scale must be finite and positive");
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
  auto launch = [&](auto L, auto N) {
    constexpr int kGroups = kThreads / decltype(L)::value;
    const int64_t blocks = ceil_div(d->rows, kGroups);
    const dim3 grid(static_cast<unsigned>(blocks < 16384 ? blocks : 16384));
    if (bias != nullptr || d->groups > 1)
      hipLaunchKernelGGL((route_rows<T, decltype(L)::value, decltype(N)::value, true>), grid, dim3(kThreads), 0, s, a,
                         static_cast<const T*>(logits), bias, weights, chosen, stats);
    else
      hipLaunchKernelGGL((route_rows<T, decltype(L)::value, decltype(N)::value, false>), grid, dim3(kThreads), 0, s, a,
                         static_cast<const T*>(logits), bias, weights, chosen, stats);
  };
  using std::integral_constant;
  // Groups are looked through by a lane each, 64 at most.
  if (d->experts <= 16 && d->groups <= 16) launch(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (d->experts <= 64 && d->groups <= 16) launch(integral_constant<int, 16>(), integral_constant<int, 4>());
  else if (d->experts <= 64) launch(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (d->experts <= 256) launch(integral_constant<int, 64>(), integral_constant<int, 4>());
  else launch(integral_constant<int, 64>(), integral_constant<int, 16>());
  return check_launch("route");
}

template <typename T>
spmm_status run_route_grad(const spmm_route_desc* d, const void* logits, const int32_t* chosen, const float* weights,
                           const float* stats, const float* grad, void* dlogits, hipStream_t s) {
  const RouteArgs a = route_args(d);
  const int64_t blocks = ceil_div(d->rows, kRowsLds / d->experts);
  hipLaunchKernelGGL(route_grad<T>, dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536)), dim3(kThreads), 0, s,
                     a, static_cast<const T*>(logits), chosen, weights, stats, grad, static_cast<T*>(dlogits));
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
