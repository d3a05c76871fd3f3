// Tiles of matrix products, four waves, for operands of any alignment and for
// fp32: 64 x 64, or 32 x 128 for groups of few rows.
//
// Operands pass through registers into LDS, one step of the sum at a time; the
// next step's loads are under way during the matrix instructions, and four or
// more work-groups of a CU hide each other's barriers.
//
// fp32 operands are split into three bf16 parts on the way, each the leading
// eight digits of what the ones before leave over, so their sum is the fp32
// value; all their products but that of the last two, which is below 2^-28 of
// the whole, are added in fp32.  That is the precision of fp32 products at 8 of
// the 16 matrix cycles that fp32 instructions take.  4096^3 runs at 137 TFLOP/s,
// 1.1 PFLOP/s of bf16 products, and at 167 on zeros: a fifth is the card's power,
// the rest LDS reads and barriers between the steps.  Parts of an infinity's
// counterpart may be zero, and their product with it a NaN where fp32 has an
// infinity: a tile that meets an infinity is summed once more with each finite
// value's sign in its place (kSigns).  That sum is infinite or NaN exactly where
// fp32's is for its factors' sake, and takes the first one's place there.
#pragma once

#include "mma.h"

namespace spmm {
namespace mma {

constexpr int kThreads128 = 256;

template <typename T>
struct Step {
  static constexpr int kParts = std::is_same_v<T, float> ? 3 : 1;
  static constexpr int kDepth = std::is_same_v<T, float> ? 32 : 64;
};

// Three bf16 parts of an fp32 value, by truncation: all parts of a value have
// its sign, and what the last one leaves is below 2^-24 of it.
__device__ inline void split(float x, unsigned& hi, unsigned& mid, unsigned& lo) {
  hi = __builtin_bit_cast(unsigned, x) & 0xffff0000u;
  const float rest = x - __builtin_bit_cast(float, hi);
  mid = __builtin_bit_cast(unsigned, rest) & 0xffff0000u;
  lo = __builtin_bit_cast(unsigned, rest - __builtin_bit_cast(float, mid));
}
// In the upper half: an infinity, a NaN or a zero as it is, else 1 with x's
// sign.
__device__ inline unsigned sign_part(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x), size = u & 0x7fffffffu;
  return size > 0x7f800000u ? 0x7fc00000u : size == 0x7f800000u || size == 0u ? u : (u & 0x80000000u) | 0x3f800000u;
}
// The upper halves of a and b as two neighbouring bf16 values.
__device__ inline unsigned upper_halves(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// One operand's kRows x depth of a step in LDS and its way there.  Layouts as
// the 256 tile's halves: where k is contiguous, lines of kDepth elements whose
// 16-byte pieces are exchanged by the line; else lines of kRows elements whose
// 32-byte units are exchanged by k.  A thread's pieces lie whole rounds of
// lines apart, which leaves the exchange alike: one offset serves them all.
template <typename T, bool C, int kRows, bool kAligned>
struct Stage {
  typedef Step<T> S;
  static constexpr int kPieces = kRows * S::kDepth / 8;  // of eight elements
  static constexpr int kEach = (kPieces + kThreads128 - 1) / kThreads128;
  static constexpr bool kWhole = kPieces % kThreads128 == 0;  // else the last threads have none
  static constexpr int kBytes = kRows * S::kDepth * 2;        // of one part
  static constexpr int kAcross = (C ? kRows : S::kDepth) / 8;
  static constexpr int kLines = kThreads128 / kAcross;        // of a round
  static constexpr int kLineBytes = kAcross * 16;
  static constexpr int kVectors = sizeof(T) / 2;
  static_assert(!C || kRows == 128 || kRows == 64, "low tiles are of contiguous k");
  static_assert(kLines % 16 == 0, "the exchange repeats every 16 lines");

  u32x4 held[kEach][kVectors];
  int line, piece;   // of the thread's first piece
  unsigned from;     // its offset in the operand, in elements
  unsigned round;    // offset between rounds
  int to;            // its place in LDS

  // The exchange: place of a 16-byte piece of a line.
  __device__ static inline int place(int line, int piece) {
    if constexpr (C && kRows == 128)
      return line * kLineBytes + (piece ^ (((line & 3) | ((line >> 3 & 1) << 2)) << 1)) * 16;
    else if constexpr (C)
      return line * kLineBytes + (piece ^ (((line >> 1 & 1) | ((line >> 3 & 1) << 1)) << 1)) * 16;
    else if constexpr (S::kDepth == 64)
      return line * kLineBytes + (piece ^ (line & 7)) * 16;
    else
      return line * kLineBytes + (piece ^ (line >> 1 & 3)) * 16;
  }

  __device__ inline void start(int64_t ld, int thread) {
    line = thread / kAcross;
    piece = thread % kAcross;
    from = static_cast<unsigned>(line * ld) + piece * 8;
    round = static_cast<unsigned>(kLines * ld);
    to = place(line, piece);
    if (!kWhole && line >= (C ? S::kDepth : kRows)) line = 1 << 28;  // none
  }

  // Loads the step at p, with `left` of the sum's depth, into registers.  With
  // aligned pieces nothing is done with the results here, so that they stay
  // under way during the matrix instructions: outside the operand p's first
  // piece is read instead, sums of rows that there are not hold anything, and
  // store() clears what is past the depth.
  __device__ inline void load(const T* p, int valid, int left) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int l = line + e * kLines, c = piece * 8;
      const bool in = l < (C ? left : valid) && c < (C ? valid : left);
      const T* at = p + (in ? from + e * round : 0u);
      if constexpr (kAligned) {
#pragma unroll
        for (int h = 0; h < kVectors; ++h) held[e][h] = reinterpret_cast<const u32x4*>(at)[h];
      } else {
        const int count = in ? (C ? valid : left) - c : 0;
        if (count >= 8) {
#pragma unroll
          for (int h = 0; h < kVectors; ++h)
            held[e][h] = __builtin_bit_cast(u32x4, *reinterpret_cast<const piece_t<T>*>(at + kPiece<T> * h));
        } else {
          T some[8];
#pragma unroll
          for (int m = 0; m < 8; ++m) some[m] = m < count ? at[m] : static_cast<T>(0.0f);
          __builtin_memcpy(&held[e], some, sizeof(some));
        }
      }
    }
  }

  // Stores the step, which has `left` of the depth, to LDS.  `most`: raised to
  // the largest magnitude that passes (fp32).  kSigns: the first part alone.
  template <bool kSigns>
  __device__ inline void store(char* lds, int left, float& most) {
    if (kAligned && left < S::kDepth) {  // (load() has done so for others)
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int inside = C ? (line + e * kLines < left ? 8 : 0) : left - piece * 8;
        T some[8];
        __builtin_memcpy(some, &held[e], sizeof(some));
#pragma unroll
        for (int m = 0; m < 8; ++m) some[m] = m < inside ? some[m] : static_cast<T>(0.0f);
        __builtin_memcpy(&held[e], some, sizeof(some));
      }
    }
    if (!kWhole && line == 1 << 28) return;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      char* at = lds + to + e * kLines * kLineBytes;
      if constexpr (S::kParts == 1) {
        *reinterpret_cast<u32x4*>(at) = held[e][0];
      } else {
        u32x4 parts[3];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const float x = __builtin_bit_cast(float, static_cast<unsigned>(held[e][m / 2][m % 2 * 2]));
          const float y = __builtin_bit_cast(float, static_cast<unsigned>(held[e][m / 2][m % 2 * 2 + 1]));
          if constexpr (kSigns) {
            parts[0][m] = upper_halves(sign_part(x), sign_part(y));
          } else {
            most = fmaxf(fmaxf(most, fabsf(x)), fabsf(y));
            unsigned a[3], b[3];
            split(x, a[0], a[1], a[2]);
            split(y, b[0], b[1], b[2]);
#pragma unroll
            for (int q = 0; q < 3; ++q) parts[q][m] = upper_halves(a[q], b[q]);
          }
        }
#pragma unroll
        for (int q = 0; q < (kSigns ? 1 : 3); ++q) *reinterpret_cast<u32x4*>(at + q * kBytes) = parts[q];
      }
    }
  }
};

// Reads kCount fragments of 16 rows, from row `first`: one address for each
// that the exchange tells apart, the rest by constant offsets.
template <typename T, bool C, int kRows, int kCount>
struct StageReader {
  typedef Stage<T, C, kRows, true> G;
  static constexpr int kDepth = G::S::kDepth;
  static constexpr int kAddresses = C ? kCount : kDepth / 32;
  int at[kAddresses];

  __device__ inline StageReader(int first, int thread) {
    const int lane = thread & 63, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < kAddresses; ++i) {
      if constexpr (C)
        at[i] = G::place(8 * q + ((lane & 15) >> 2), first / 8 + 2 * i + ((lane & 3) >> 1)) + (lane & 1) * 8;
      else
        at[i] = G::place(first + (lane & 15), 4 * i + q);
    }
  }

  // Fragment r for 32 k from 32 * kk, of a part.
  __device__ inline u32x4 read(const char* lds, int r, int kk, int part) const {
    if constexpr (!C) {
      return *reinterpret_cast<const u32x4*>(lds + at[kk] + r * 16 * G::kLineBytes + part * G::kBytes);
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
      u32x2 h[2];
#pragma unroll
      for (int m = 0; m < 2; ++m)
        h[m] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                             (lds_s16x4)(lds + at[r] + (kk * 32 + m * 4) * G::kLineBytes + part * G::kBytes)));
      return __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3);
    }
  }
};

// A tile's sums: wave (w / kAlong, w % kAlong) holds kA x kB fragments.
template <int kRowFragments, int kColFragments, int kWavesAlong>
struct SumsOf {
  static constexpr int kA = kRowFragments, kB = kColFragments, kAlong = kWavesAlong;
  f32x4 c[kA][kB];

  __device__ inline void clear() {
#pragma unroll
    for (int i = 0; i < kA; ++i)
#pragma unroll
      for (int j = 0; j < kB; ++j) c[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // The lane's sums as eights of neighbouring columns; place() comes first.
  static constexpr int kEights = kA * kB / 2;
  int row0, col0;
  __device__ inline void place() {
    const int thread = thread_here(), lane = thread & 63, wave = thread >> 6;
    row0 = wave / kAlong * kA * 16 + (lane & 15);
    col0 = wave % kAlong * kB * 16 + eight_column(lane);
#pragma unroll
    for (int i = 0; i < kA; ++i)
#pragma unroll
      for (int j = 0; j < kB; j += 2) exchange_fours(c[i][j], c[i][j + 1]);
  }
  // Columns that eights share: group(k) of kGroups, from group_col().
  static constexpr int kGroups = kB / 2;
  __device__ static inline constexpr int group(int k) { return k % kGroups; }
  __device__ inline int group_col(int g) const { return g * 32 + col0; }
  __device__ inline int row(int k) const { return k / (kB / 2) * 16 + row0; }
  __device__ inline int col(int k) const { return k % (kB / 2) * 32 + col0; }
  __device__ inline f32x4 four(int k, int half) const { return c[k / (kB / 2)][k % (kB / 2) * 2 + half]; }
};

template <typename T, bool kAC, bool kBC, int kRows, int kCols, bool kAligned>
struct Staged {
  typedef Step<T> S;
  typedef Stage<T, kAC, kRows, kAligned> StageA;
  typedef Stage<T, kBC, kCols, kAligned> StageB;
  // A low tile has its waves along the columns.
  static constexpr int kAlong = kRows == 32 ? 4 : 2;
  typedef SumsOf<kRows * kAlong / 64, kCols / kAlong / 16, kAlong> Sums;
  static constexpr int kLdsBytes = S::kParts * (StageA::kBytes + StageB::kBytes);

  // The sum over k of A(i, k) B(j, k).
  __device__ static inline void sum(const Operand<T>& a, const Operand<T>& b, char* lds, Sums& s) {
    float most = 0.0f;
    s.clear();
    add<false>(a, b, lds, s, most);
    if constexpr (S::kParts == 3) {
      if (__syncthreads_or(most == __builtin_inff())) {
        Sums t;
        t.clear();
        add<true>(a, b, lds, t, most);
#pragma unroll
        for (int i = 0; i < Sums::kA; ++i)
#pragma unroll
          for (int j = 0; j < Sums::kB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!__builtin_isfinite(t.c[i][j][e])) s.c[i][j][e] = t.c[i][j][e];
      }
    }
  }

  template <bool kSigns>
  __device__ static inline void add(const Operand<T>& a, const Operand<T>& b, char* lds, Sums& s, float& most) {
    const int thread = thread_here(), wave = thread >> 6;
    char* lb = lds + S::kParts * StageA::kBytes;
    const StageReader<T, kAC, kRows, Sums::kA> ra(wave / kAlong * Sums::kA * 16, thread);
    const StageReader<T, kBC, kCols, Sums::kB> rb(wave % kAlong * Sums::kB * 16, thread);
    const int va = static_cast<int>(a.valid), vb = static_cast<int>(b.valid);
    StageA sa;
    StageB sb;
    sa.start(a.ld, thread);
    sb.start(b.ld, thread);
    const T *pa = a.p, *pb = b.p;
    const int64_t step_a = S::kDepth * (kAC ? a.ld : 1), step_b = S::kDepth * (kBC ? b.ld : 1);
    int left = static_cast<int>(a.depth);
    if (left <= 0) return;
    auto load = [&]() {
      const int most_k = left < S::kDepth ? left : S::kDepth;
      sa.load(left > 0 ? pa : a.p, va, most_k);
      sb.load(left > 0 ? pb : b.p, vb, most_k);
      pa += step_a;
      pb += step_b;
    };
    load();
    do {
      __syncthreads();  // the last step's fragments have been read
      sa.template store<kSigns>(lds, left, most);
      sb.template store<kSigns>(lb, left, most);
      left -= S::kDepth;
      if (kAligned || left > 0) load();  // (a last, unused one costs less than the branch)
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < S::kDepth / 32; ++kk) {
        constexpr int kParts = kSigns ? 1 : S::kParts;
        u32x4 fa[Sums::kA][kParts];
#pragma unroll
        for (int i = 0; i < Sums::kA; ++i)
#pragma unroll
          for (int q = 0; q < kParts; ++q) fa[i][q] = ra.read(lds, i, kk, q);
        u32x4 fb[Sums::kB][kParts];
#pragma unroll
        for (int j = 0; j < Sums::kB; ++j)
#pragma unroll
          for (int q = 0; q < kParts; ++q) fb[j][q] = rb.read(lb, j, kk, q);
        // products of parts, the smallest first
        constexpr int kProducts = kParts == 1 ? 1 : 8;
        constexpr int kOrder[8][2] = {{0, 0}, {0, 1}, {1, 0}, {1, 1}, {0, 2}, {2, 0}, {1, 2}, {2, 1}};
        typedef std::conditional_t<S::kParts == 3, __bf16, T> Part;
        if constexpr (kProducts == 1) {
#pragma unroll
          for (int j = 0; j < Sums::kB; ++j)
#pragma unroll
            for (int i = 0; i < Sums::kA; ++i) s.c[i][j] = multiply<Part>(fb[j][0], fa[i][0], s.c[i][j]);
        } else {
          // Matrix instructions cut their sums to fp32, always to the same side:
          // the parts' products of 32 k are summed apart, from zero, and their
          // sum is added with fp32's rounding.
          f32x4 c[Sums::kA][Sums::kB] = {};
#pragma unroll
          for (int o = kProducts - 1; o >= 0; --o)
#pragma unroll
            for (int j = 0; j < Sums::kB; ++j)
#pragma unroll
              for (int i = 0; i < Sums::kA; ++i)
                c[i][j] = multiply<Part>(fb[j][kOrder[o][1]], fa[i][kOrder[o][0]], c[i][j]);
#pragma unroll
          for (int j = 0; j < Sums::kB; ++j)
#pragma unroll
            for (int i = 0; i < Sums::kA; ++i) s.c[i][j] += c[i][j];
        }
      }
    } while (left > 0);
    __syncthreads();
  }
};

}  // namespace mma
}  // namespace spmm
