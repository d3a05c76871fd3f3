// Value types of the dense operators (layer norm, grouped products,
// orthogonalised updates): fp16, bf16 and fp32, with all arithmetic in fp32.
#pragma once

#include <type_traits>

#include "common.h"

namespace spmm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// Elements of one 16-byte piece.
template <typename T>
constexpr int kPiece = 16 / static_cast<int>(sizeof(T));

// A 16-byte piece that may start at any element: the hardware takes vector
// accesses of any alignment, so rows of odd widths keep wide loads.
template <typename T>
struct PieceOf {
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};
template <typename T>
using piece_t = typename PieceOf<T>::type;

// Loads up to one piece of `n` remaining elements at p as fp32, zeros past n.
template <typename T>
__device__ inline void load_piece(const T* p, int64_t n, float (&v)[kPiece<T>]) {
  if (n >= kPiece<T>) {
    const piece_t<T> x = *reinterpret_cast<const piece_t<T>*>(p);
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) v[i] = static_cast<float>(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) v[i] = i < n ? static_cast<float>(p[i]) : 0.0f;
  }
}

// The same as they lie, to be converted later: a load that is converted at once
// is waited for at once.
template <typename T>
__device__ inline piece_t<T> load_raw(const T* p, int64_t n) {
  if (n >= kPiece<T>) return *reinterpret_cast<const piece_t<T>*>(p);
  piece_t<T> x;
#pragma unroll
  for (int i = 0; i < kPiece<T>; ++i) x[i] = i < n ? p[i] : static_cast<T>(0.0f);
  return x;
}

// Stores up to one piece, each value rounded once to nearest even.
template <typename T>
__device__ inline void store_piece(T* p, int64_t n, const float (&v)[kPiece<T>]) {
  if (n >= kPiece<T>) {
    piece_t<T> x;
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) x[i] = static_cast<T>(v[i]);
    *reinterpret_cast<piece_t<T>*>(p) = x;
  } else {
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i)
      if (i < n) p[i] = static_cast<T>(v[i]);
  }
}

inline bool dense_type(int32_t t) { return t == SPMM_VALUE_F16 || t == SPMM_VALUE_BF16 || t == SPMM_VALUE_F32; }
inline int64_t dense_type_bytes(int32_t t) { return t == SPMM_VALUE_F32 ? 4 : 2; }

}  // namespace spmm
