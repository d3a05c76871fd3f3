// Operands and matrix instructions of the product tiles (mma_256.h, mma_ring.h,
// mma_staged.h).
#pragma once

#include "numeric.h"

namespace spmm {
namespace mma {

// threadIdx.x, computed anew: in a loop over tiles, addresses made from it are
// not kept in registers across the other tiles' sums.
__device__ inline int thread_here() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// An operand of the product: element (i, k) of the tile.  Where C is false k
// is the contiguous one, at p[i * ld + k]; where true i is, at p[k * ld + i].
// p and ld are multiples of 16 bytes, and so is `depth` where C is false.
// Rows i >= valid and k >= depth are not read and count as zeros, but where C
// is true: memory up to the 16-byte piece of the last valid element is read
// there, and sums with i >= valid hold anything.  `lo` is the second plane of
// an operand held as the sum of two, else null.
template <typename T>
struct Operand {
  const T* p;
  const T* lo;
  int64_t ld;
  int64_t valid;
  int64_t depth;
};

typedef __attribute__((address_space(3))) void* lds_ptr;

__device__ inline unsigned lds_address(const void* p) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((lds_ptr)p));
}

// A value that is the same on all lanes, in scalar registers.
__device__ inline int64_t uniform(int64_t v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v));
  const unsigned hi = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// Work-groups run on the XCDs in turn; each XCD gets one run of the tiles, so
// that neighbours share its L2.  (32-bit: a division of 64 bits takes longer
// than a step of the sum.)
__device__ inline unsigned run_of_xcd(unsigned block, unsigned blocks) {
  const unsigned each = blocks / kXcds, rest = blocks % kXcds, x = block % kXcds;
  return x * each + (x < rest ? x : rest) + block / kXcds;
}

// Tile `n` of down x across: blocks of four tile rows, down them first, so
// that the tiles at work together share rows of both operands.
__device__ inline void place_tile(unsigned n, unsigned down, unsigned across, unsigned& i, unsigned& j) {
  const unsigned block = n / (4 * across), first = 4 * block, high = down - first < 4 ? down - first : 4;
  const unsigned m = n - block * 4 * across;
  i = high == 4 ? first + (m & 3) : first + m % high;
  j = high == 4 ? m >> 2 : m / high;
}

// Two fours of neighbouring columns, of fragments 16 columns apart: lane group q
// = lane / 16 % 4 holds columns 4 q .. 4 q + 3 of either.  Exchanged with the
// next group, each lane holds eight neighbouring columns, from eight_column().
__device__ inline void exchange_fours(f32x4& a, f32x4& b) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, static_cast<float>(a[e])),
                                                     __builtin_bit_cast(unsigned, static_cast<float>(b[e])), false, false);
    a[e] = __builtin_bit_cast(float, static_cast<unsigned>(r[0]));
    b[e] = __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
  }
}
__device__ inline int eight_column(int lane) { return (lane >> 4 & 1) * 16 + (lane >> 5) * 8; }

// The 16 x 16 x 32 matrix instruction: lane (i = lane % 16, q = lane / 16) holds
// k = 8 q .. 8 q + 7 of row i of either operand, and gets the sums of b's row i
// with a's rows 4 q .. 4 q + 3.
template <typename T>
__device__ inline f32x4 multiply(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same_v<T, _Float16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

}  // namespace mma
}  // namespace spmm
