// Reductions over the lanes that share a row: aligned groups of L lanes of a
// wave (L a power of two up to 64), or a whole work-group.
//
// Steps over 1 to 8 lanes are DPP moves, those over 16 and 32 lane swaps, all
// at the rate of ordinary vector instructions; an exchange through LDS hardware
// (__shfl_xor) waits about ten times as long.  The moves over 4 and 8 lanes
// mirror, which brings the other half's result as all lanes of a half hold the
// same one by then.
#pragma once

#include "common.h"

namespace spmm {

// f(v of a lane, v of its partner D lanes away), the same on both.
template <int D, typename F>
__device__ inline uint32_t reduce_step(uint32_t v, F f) {
  if constexpr (D == 1) {
    return f(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true)));
  } else if constexpr (D == 2) {
    return f(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true)));
  } else if constexpr (D == 4) {
    return f(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 0xF, 0xF, true)));
  } else if constexpr (D == 8) {
    return f(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 0xF, 0xF, true)));
  } else if constexpr (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return f(r[0], r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(r[0], r[1]);
  }
}

template <int L, typename F>
__device__ inline uint32_t lane_reduce(uint32_t v, F f) {
  if constexpr (L >= 2) v = reduce_step<1>(v, f);
  if constexpr (L >= 4) v = reduce_step<2>(v, f);
  if constexpr (L >= 8) v = reduce_step<4>(v, f);
  if constexpr (L >= 16) v = reduce_step<8>(v, f);
  if constexpr (L >= 32) v = reduce_step<16>(v, f);
  if constexpr (L >= 64) v = reduce_step<32>(v, f);
  return v;
}

__device__ inline float as_float(uint32_t v) { return __builtin_bit_cast(float, v); }
__device__ inline uint32_t as_bits(float v) { return __builtin_bit_cast(uint32_t, v); }

template <int L>
__device__ inline float lane_sum(float v) {
  return as_float(lane_reduce<L>(as_bits(v), [](uint32_t a, uint32_t b) { return as_bits(as_float(a) + as_float(b)); }));
}
template <int L>
__device__ inline float lane_max(float v) {
  return as_float(
      lane_reduce<L>(as_bits(v), [](uint32_t a, uint32_t b) { return as_bits(fmaxf(as_float(a), as_float(b))); }));
}
template <int L>
__device__ inline float lane_min_value(float v) {
  return as_float(
      lane_reduce<L>(as_bits(v), [](uint32_t a, uint32_t b) { return as_bits(fminf(as_float(a), as_float(b))); }));
}
template <int L>
__device__ inline uint32_t lane_max(uint32_t v) {
  return lane_reduce<L>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int L>
__device__ inline uint32_t lane_min(uint32_t v) {
  return lane_reduce<L>(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}

// The same over a work-group of 64 * W threads, with W floats of LDS.  Callers
// keep a barrier between two uses of one buffer.
template <int W>
__device__ inline float block_max(float v, float* lds) {
  v = lane_max<64>(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < W; ++w) v = fmaxf(v, lds[w]);
  return v;
}

// Values in the order of whole numbers: greater floats have greater keys, -0
// has the key of 0.
__device__ inline uint32_t order_key(float v) {
  const uint32_t u = as_bits(v + 0.0f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ inline float key_value(uint32_t key) {
  return as_float(key ^ ((key & 0x80000000u) != 0 ? 0x80000000u : 0xFFFFFFFFu));
}
constexpr uint32_t kKeyOfMinusInf = 0x007FFFFFu;

}  // namespace spmm
