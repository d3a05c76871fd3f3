// Rows in pieces of 16 bytes, whatever their width.
//
// The last piece of a row that no whole number of pieces fills is moved back to
// end with the row, so that every load and store is a whole piece: elements that
// two pieces hold are loaded twice and stored twice, the same.  Sums over a row
// leave out the first `shift` elements of a piece, which the piece before has.
// Rows narrower than one piece (Narrow) are taken element by element.
//
// Nontemporal: what is read or written once and not soon again.  On MI355X such
// loads of whole rows run at 6.8 TB/s where ordinary ones reach 6.0, copies at
// 5.6 against 5.35.
#pragma once

#include "numeric.h"

namespace spmm {

template <typename T, bool Narrow>
struct RowPiece {
  static constexpr int V = kPiece<T>;

  // Where the piece at `column` begins; past the row's end it is the last one.
  __device__ static inline int64_t begin(int64_t column, int64_t width) {
    if constexpr (Narrow) return column;
    return column < width - V ? column : width - V;
  }
  // Elements of the piece that belong to the piece before it; V past the row's end.
  __device__ static inline int shift(int64_t column, int64_t width) {
    const int64_t s = column - begin(column, width);
    return s < V ? static_cast<int>(s) : V;
  }

  template <bool Once = false>
  __device__ static inline piece_t<T> load(const T* row, int64_t column, int64_t width) {
    if constexpr (Narrow) {
      return load_raw(row + column, width - column);
    } else {
      const piece_t<T>* p = reinterpret_cast<const piece_t<T>*>(row + begin(column, width));
      if constexpr (Once) return __builtin_nontemporal_load(p);
      return *p;
    }
  }

  template <bool Once = false>
  __device__ static inline void store(T* row, int64_t column, int64_t width, const piece_t<T>& v) {
    if (column >= width) return;
    if constexpr (Narrow) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (column + i < width) row[column + i] = v[i];
    } else {
      piece_t<T>* p = reinterpret_cast<piece_t<T>*>(row + begin(column, width));
      if constexpr (Once) __builtin_nontemporal_store(v, p);
      else *p = v;
    }
  }

  template <bool Once = false>
  __device__ static inline void store(T* row, int64_t column, int64_t width, const float (&v)[V]) {
    piece_t<T> x;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = static_cast<T>(v[i]);
    store<Once>(row, column, width, x);
  }
};

}  // namespace spmm
