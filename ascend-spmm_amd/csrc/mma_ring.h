// Tiles of matrix products of fp16 or bf16 operands, four waves: 128 or 64 rows
// and columns.
//
// A step of the sum is 32 deep.  Its operands are copied from memory straight
// to LDS, into a ring of four steps.  A wave reads the next step's fragments and
// starts a copy beside the matrix instructions of the step at hand, so that the
// matrix cores and LDS work at once also where a CU has one tile.  One barrier a
// step: it says that the next step has arrived, and that the one before has been
// read, whose place the copies started next take.
#pragma once

#include "mma_staged.h"
#include "mma_256.h"

namespace spmm {
namespace mma {

// Each wave holds a quarter of the tile.  kPair: fp16 operands held as sums of
// two planes; see multiply_tile.
template <typename T, bool kAC, bool kBC, bool kPair, int kRows, int kCols>
struct Ring {
  static constexpr int kDepth = 32;
  static constexpr int kStages = 4;
  static constexpr int kPlanes = kPair ? 2 : 1;
  static constexpr int kBytesA = kRows * kDepth * 2, kBytesB = kCols * kDepth * 2;  // of a step of one plane
  static constexpr int kStage = kPlanes * (kBytesA + kBytesB);
  static constexpr int kLdsBytes = kStages * kStage;
  static constexpr int kCopies = kPlanes * (kBytesA + kBytesB) / 4096;  // instructions of a wave and step
  static constexpr int kA = kRows / 32, kB = kCols / 32;                // fragments of a wave
  typedef SumsOf<kA, kB, 2> Sums;

  // Layout of a step of one operand of kSize lines or columns: lines of 64
  // bytes (k contiguous; 16-byte piece c of line i at c ^ (i / 2 % 4)), or of
  // 2 kSize bytes (C; 32-byte unit u of line k at u ^ swizzle).
  template <bool C, int kSize>
  struct Copier {
    static constexpr int kRounds = kSize / 64;
    const char *p, *lo;
    int64_t step_bytes;
    int left, step_pieces;  // 16-byte pieces to the operand's last
    int at, to, last, tail, bytes;
    unsigned offset[kRounds];
    int k;

    __device__ static inline int swizzle(int line) {
      return kSize == 128 ? Half<true>::swizzle(line) : (line >> 1 & 1) | (line >> 3 & 1) << 1;
    }

    __device__ inline Copier(const Operand<T>& o, int from, int end, int wave, int lane) {
      const int64_t ld = uniform(o.ld), depth = uniform(o.depth), valid = uniform(o.valid);
      step_bytes = C ? 2 * kDepth * ld : 2 * kDepth;
      step_pieces = static_cast<int>(step_bytes / 16);
      const int64_t elements = C ? (depth - 1) * ld + (valid + 7) / 8 * 8 : (valid - 1) * ld + depth;
      at = __builtin_amdgcn_readfirstlane(from);
      to = __builtin_amdgcn_readfirstlane(end);
      left = valid > 0 && depth > 0 ? static_cast<int>(elements / 8) - at * step_pieces : 0;
      p = reinterpret_cast<const char*>(uniform(reinterpret_cast<int64_t>(o.p)) + at * step_bytes);
      lo = kPair ? reinterpret_cast<const char*>(uniform(reinterpret_cast<int64_t>(o.lo)) + at * step_bytes) : nullptr;
      last = static_cast<int>((depth + kDepth - 1) / kDepth) - 1;
      tail = static_cast<int>(depth - static_cast<int64_t>(last) * kDepth);
      k = 0;
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        if constexpr (C) {
          constexpr int kAcross = kSize / 8;  // pieces of a line
          const int line = (r * 256 + wave * 64 + lane) / kAcross;
          offset[r] = static_cast<unsigned>(2 * (line * o.ld + ((lane % kAcross) ^ (swizzle(line) << 1)) * 8));
        } else {
          const int line = r * 64 + wave * 16 + lane / 4;
          k = ((lane & 3) ^ (line >> 1 & 3)) * 8;
          offset[r] = static_cast<unsigned>(2 * (line * o.ld + k));
        }
      }
    }

    // What is left of the operand from the step at hand on; past the end nothing
    // is read and zeros arrive.
    __device__ inline void begin() {
      const int n = at >= to || left < 0 ? 0 : left > 0x7ffffff ? 0x7ffffff : left;
      bytes = n * 16;
      if constexpr (!C)
        if (at == last && tail < kDepth && k >= tail)
#pragma unroll
          for (int r = 0; r < kRounds; ++r) offset[r] = 0x80000000u;  // past any buffer
    }

    // Instruction n of the step's copies, to `lds` (the wave's part).  Written
    // as assembly, which keeps the compiler from waiting for it before every
    // read of LDS: the barriers order them.  m0, which holds the place in LDS, is
    // the compiler's own, and is left as it was.
    static constexpr int kInstructions = kPlanes * kRounds;
    template <int n>
    __device__ inline void copy(unsigned lds) const {
      const uint64_t from = reinterpret_cast<uint64_t>(n / kRounds == 0 ? p : lo);
      const u32x4 b = {static_cast<unsigned>(from), static_cast<unsigned>(from >> 32) & 0xffffu,
                       static_cast<unsigned>(bytes), 0x00020000u};
      unsigned m0;
      asm volatile(
          "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
          "s_mov_b32 m0, %0"
          : "=&s"(m0)
          : "s"(lds + n / kRounds * kSize * kDepth * 2 + n % kRounds * 4096), "v"(offset[n % kRounds]), "s"(b)
          : "memory");
    }

    __device__ inline void advance() {
      ++at;
      p += step_bytes;
      if constexpr (kPair) lo += step_bytes;
      left -= step_pieces;
    }
  };

  // Addresses of a wave's fragments of one operand.
  template <bool C, int kSize>
  struct Reader {
    static constexpr int kAddresses = C ? kSize / 32 : 1;
    unsigned at[kAddresses];
    __device__ inline Reader(int first, int lane) {
      const int q = lane >> 4, i = lane & 15;
      if constexpr (C) {
        const int k = 8 * q + (i >> 2);
#pragma unroll
        for (int r = 0; r < kAddresses; ++r)
          at[r] = k * kSize * 2 + ((first / 16 + r) ^ Copier<C, kSize>::swizzle(k)) * 32 + (lane & 3) * 8;
      } else {
        at[0] = (first + i) * 64 + (q ^ (i >> 1 & 3)) * 16;
      }
    }
  };

  // Fragment r of a wave, from the operand's step of one plane in LDS.
  template <bool C, int kSize>
  __device__ static inline u32x4 read(const Reader<C, kSize>& reader, const char* lds, int r) {
    if constexpr (!C) {
      return *reinterpret_cast<const u32x4*>(lds + reader.at[0] + r * 1024);
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
      u32x2 h[2];
#pragma unroll
      for (int m = 0; m < 2; ++m)
        h[m] = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(lds + reader.at[r] + m * 8 * kSize)));
      return __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3);
    }
  }

  struct Fragments {
    u32x4 a[kPlanes][kA], b[kPlanes][kB];
  };

  // Instructions [n, end) of both operands' copies of a step.
  template <int n, int end>
  __device__ static inline void copy_some(const Copier<kAC, kRows>& a, const Copier<kBC, kCols>& b, unsigned lds) {
    if constexpr (n < end) {
      constexpr int kFirst = Copier<kAC, kRows>::kInstructions;
      if constexpr (n < kFirst) a.template copy<n>(lds);
      else b.template copy<n - kFirst>(lds + kPlanes * kBytesA);
      copy_some<n + 1, end>(a, b, lds);
    }
  }

  // The matrix instructions of a step in rows of the wave's sums, and between
  // them the step's copies.
  template <int i>
  __device__ static inline void multiply_some(const Fragments& f, Sums& s, Sums& low, const Copier<kAC, kRows>& a,
                                              const Copier<kBC, kCols>& b, unsigned lds) {
    if constexpr (i < kA) {
#pragma unroll
      for (int q = 2 * kPlanes - 2; q >= 0; --q)  // planes (0, 1), (1, 0), then (0, 0)
#pragma unroll
        for (int j = 0; j < kB; ++j) {
          f32x4& c = q == 0 ? s.c[i][j] : low.c[i][j];
          c = multiply<T>(f.b[q == 2 ? 1 : 0][j], f.a[q == 1 ? 1 : 0][i], c);
        }
      __builtin_amdgcn_sched_barrier(0);
      copy_some<i * kCopies / kA, (i + 1) * kCopies / kA>(a, b, lds);
      multiply_some<i + 1>(f, s, low, a, b, lds);
    }
  }

  // Adds the steps [from, to) of the sum over k of A(i, k) B(j, k); operands
  // as mma_256.h takes them.
  __device__ static inline void add(const Operand<T>& a, const Operand<T>& b, char* lds, int from, int to,
                                    Sums& s) {
    const int thread = thread_here(), lane = thread & 63;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    Copier<kAC, kRows> ca(a, from, to, wave, lane);
    Copier<kBC, kCols> cb(b, from, to, wave, lane);
    const Reader<kAC, kRows> ra((wave >> 1) * (kRows / 2), lane);
    const Reader<kBC, kCols> rb((wave & 1) * (kCols / 2), lane);
    const unsigned base = lds_address(lds) + wave * 1024;
    int fill = 0;  // where the next copies go
    auto next = [](int stage) { return stage + kStage < kLdsBytes ? stage + kStage : 0; };
    auto begin_copies = [&]() {
      ca.begin();
      cb.begin();
    };
    auto end_copies = [&]() {
      ca.advance();
      cb.advance();
      fill = next(fill);
    };
    auto copy_all = [&]() {
      begin_copies();
      copy_some<0, kCopies>(ca, cb, base + fill);
      end_copies();
    };
    auto read_all = [&](Fragments& f, int stage) {
#pragma unroll
      for (int q = 0; q < kPlanes; ++q) {
        const char *la = lds + stage + q * kBytesA, *lb = lds + stage + kPlanes * kBytesA + q * kBytesB;
#pragma unroll
        for (int j = 0; j < kB; ++j) f.b[q][j] = read<kBC, kCols>(rb, lb, j);
#pragma unroll
        for (int i = 0; i < kA; ++i) f.a[q][i] = read<kAC, kRows>(ra, la, i);
      }
    };
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t) copy_all();
    int stage = 0;  // of the step at hand
    Fragments f0, f1;
    // Products with a low plane, apart: an instruction's sum is cut to fp32, not
    // rounded, and the large sums are cut by a third as many.
    Sums low;
    if constexpr (kPair) low.clear();
    wait_copies<(kStages - 2) * kCopies>();
    barrier();
    read_all(f0, stage);
    // Step t with fragments `f`; those of the next go to `g`.
    auto step = [&](Fragments& f, Fragments& g) {
      wait_copies<(kStages - 3) * kCopies>();
      barrier();
      begin_copies();
      stage = next(stage);
      read_all(g, stage);
      multiply_some<0>(f, s, low, ca, cb, base + fill);
      end_copies();
    };
    for (int t = from; t < to; t += 2) {
      step(f0, f1);
      if (t + 1 < to) step(f1, f0);
    }
    // No copy outlives the loop: LDS is free again.
    wait_copies<0>();
    barrier();
    if constexpr (kPair) {
#pragma unroll
      for (int i = 0; i < kA; ++i)
#pragma unroll
        for (int j = 0; j < kB; ++j) s.c[i][j] += low.c[i][j];
    }
  }
};

}  // namespace mma
}  // namespace spmm
