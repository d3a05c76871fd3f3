// 256 x 256 tile of a matrix product of fp16 or bf16 operands in fp32.
//
// Eight waves (two groups of four, one wave of each group per SIMD) share the
// tile.  A step of the sum is 64 deep: its operands are four half tiles
// A0 A1 B0 B1 of 128 x 64, copied from memory straight to LDS, in two buffers.
// A wave multiplies a 64 x 32 piece of each quadrant Ai Bj in turn, so a step
// has four phases; a phase reads one half tile's fragments (which serve two
// phases) and starts the copy of one half tile of the next step, then does 16
// matrix instructions.  The second group runs half a phase behind the first:
// on every SIMD one wave's reads and copies go on beside the other wave's
// matrix instructions.  The matrix cores bound it: a step takes 2048 cycles of
// them, against 192 KB of LDS reads.  One tile a CU, 4096^3 in bf16, takes 102 us
// (1340 TFLOP/s); 8192^3 runs at 1250, where the card's power bounds it (1670
// on zeros).  Without the offset between the groups 8192^3 ran at 1130 (1320
// with it, measured one after the other).
#pragma once

#include "mma.h"

namespace spmm {
namespace mma {

constexpr int kTile = 256;
constexpr int kDepth = 64;
constexpr int kThreads = 512;
constexpr int kLdsBytes = 128 * 1024;

// Barrier of the work-group that the compiler moves nothing across.
__device__ inline void barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
template <int N>
__device__ inline void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%c0)" ::"i"(N) : "memory");
}

// Fragments of R x 16 rows (i) and 64 columns (k) of a half tile in LDS, for
// matrix instructions 32 deep: lane (i = lane % 16, q = lane / 16) of fragment
// [r][k] holds elements 32 k + 8 q .. + 7 of row 16 r + i.
template <int R>
struct Fragments {
  u32x4 f[R][2];
};

// Half tiles in LDS.  C false: 128 rows of 64 k (128 bytes); the 16-byte piece
// c of row i lies at c ^ (i % 8), so that eight rows' same pieces lie in
// different banks.  C true: 64 rows k of 128 i (256 bytes); the 32-byte unit u
// of row k lies at u ^ swizzle(k), so that the rows that one transposing read
// takes (four k of each 16 lanes) do.  The copies apply the same on their
// source side.
template <bool C>
struct Half;

template <>
struct Half<false> {
  // Copy: element offset of the lane's 16 bytes of round r, and its first k.
  __device__ static inline int64_t source(int wave, int lane, int r, int64_t ld) {
    const int row = r * 64 + wave * 8 + lane / 8;
    return row * ld + source_k(wave, lane);
  }
  __device__ static inline int source_k(int wave, int lane) { return ((lane & 7) ^ (lane / 8)) * 8; }

  // Addresses of a wave's fragments, rows from `first`.
  template <int R>
  struct Reader {
    unsigned at[2];
    __device__ inline Reader(unsigned lds, int first, int lane) {
#pragma unroll
      for (int k = 0; k < 2; ++k) at[k] = lds + (first + (lane & 15)) * 128 + (((lane >> 4) + 4 * k) ^ (lane & 7)) * 16;
    }
    template <int kOffset>
    __device__ inline void read(Fragments<R>& d) const {
      if constexpr (R == 4)
        asm volatile(
            "ds_read_b128 %0, %8 offset:%c10\n\tds_read_b128 %1, %9 offset:%c10\n\t"
            "ds_read_b128 %2, %8 offset:%c10+2048\n\tds_read_b128 %3, %9 offset:%c10+2048\n\t"
            "ds_read_b128 %4, %8 offset:%c10+4096\n\tds_read_b128 %5, %9 offset:%c10+4096\n\t"
            "ds_read_b128 %6, %8 offset:%c10+6144\n\tds_read_b128 %7, %9 offset:%c10+6144\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(d.f[0][0]), "=&v"(d.f[0][1]), "=&v"(d.f[1][0]), "=&v"(d.f[1][1]), "=&v"(d.f[2][0]),
              "=&v"(d.f[2][1]), "=&v"(d.f[3][0]), "=&v"(d.f[3][1])
            : "v"(at[0]), "v"(at[1]), "i"(kOffset)
            : "memory");
      else
        asm volatile(
            "ds_read_b128 %0, %4 offset:%c6\n\tds_read_b128 %1, %5 offset:%c6\n\t"
            "ds_read_b128 %2, %4 offset:%c6+2048\n\tds_read_b128 %3, %5 offset:%c6+2048\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(d.f[0][0]), "=&v"(d.f[0][1]), "=&v"(d.f[1][0]), "=&v"(d.f[1][1])
            : "v"(at[0]), "v"(at[1]), "i"(kOffset)
            : "memory");
    }
  };
};

template <>
struct Half<true> {
  __device__ static inline int swizzle(int k) { return (k & 3) | ((k >> 3 & 1) << 2); }
  __device__ static inline int64_t source(int wave, int lane, int r, int64_t ld) {
    const int k = r * 32 + wave * 4 + lane / 16;
    return k * ld + ((lane & 15) ^ (swizzle(k) << 1)) * 8;
  }

  // ds_read_b64_tr_b16: within 16 lanes, lane 4 e + c reads four i of row k + e,
  // and lane i gets rows k .. k + 3 of its column.
  template <int R>
  struct Reader {
    unsigned at[R];
    __device__ inline Reader(unsigned lds, int first, int lane) {
      const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
      for (int r = 0; r < R; ++r) at[r] = lds + k * 256 + ((first / 16 + r) ^ swizzle(k)) * 32 + (lane & 3) * 8;
    }
    template <int kOffset>
    __device__ inline void read(Fragments<R>& d) const {
      u32x2 h[R][2][2];
      if constexpr (R == 4)
        asm volatile(
            "ds_read_b64_tr_b16 %0, %16 offset:%c20\n\tds_read_b64_tr_b16 %1, %16 offset:%c20+1024\n\t"
            "ds_read_b64_tr_b16 %2, %16 offset:%c20+8192\n\tds_read_b64_tr_b16 %3, %16 offset:%c20+9216\n\t"
            "ds_read_b64_tr_b16 %4, %17 offset:%c20\n\tds_read_b64_tr_b16 %5, %17 offset:%c20+1024\n\t"
            "ds_read_b64_tr_b16 %6, %17 offset:%c20+8192\n\tds_read_b64_tr_b16 %7, %17 offset:%c20+9216\n\t"
            "ds_read_b64_tr_b16 %8, %18 offset:%c20\n\tds_read_b64_tr_b16 %9, %18 offset:%c20+1024\n\t"
            "ds_read_b64_tr_b16 %10, %18 offset:%c20+8192\n\tds_read_b64_tr_b16 %11, %18 offset:%c20+9216\n\t"
            "ds_read_b64_tr_b16 %12, %19 offset:%c20\n\tds_read_b64_tr_b16 %13, %19 offset:%c20+1024\n\t"
            "ds_read_b64_tr_b16 %14, %19 offset:%c20+8192\n\tds_read_b64_tr_b16 %15, %19 offset:%c20+9216\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(h[0][0][0]), "=&v"(h[0][0][1]), "=&v"(h[0][1][0]), "=&v"(h[0][1][1]), "=&v"(h[1][0][0]),
              "=&v"(h[1][0][1]), "=&v"(h[1][1][0]), "=&v"(h[1][1][1]), "=&v"(h[2][0][0]), "=&v"(h[2][0][1]),
              "=&v"(h[2][1][0]), "=&v"(h[2][1][1]), "=&v"(h[3][0][0]), "=&v"(h[3][0][1]), "=&v"(h[3][1][0]),
              "=&v"(h[3][1][1])
            : "v"(at[0]), "v"(at[1]), "v"(at[R - 2]), "v"(at[R - 1]), "i"(kOffset)
            : "memory");
      else
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8 offset:%c10\n\tds_read_b64_tr_b16 %1, %8 offset:%c10+1024\n\t"
            "ds_read_b64_tr_b16 %2, %8 offset:%c10+8192\n\tds_read_b64_tr_b16 %3, %8 offset:%c10+9216\n\t"
            "ds_read_b64_tr_b16 %4, %9 offset:%c10\n\tds_read_b64_tr_b16 %5, %9 offset:%c10+1024\n\t"
            "ds_read_b64_tr_b16 %6, %9 offset:%c10+8192\n\tds_read_b64_tr_b16 %7, %9 offset:%c10+9216\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(h[0][0][0]), "=&v"(h[0][0][1]), "=&v"(h[0][1][0]), "=&v"(h[0][1][1]), "=&v"(h[1][0][0]),
              "=&v"(h[1][0][1]), "=&v"(h[1][1][0]), "=&v"(h[1][1][1])
            : "v"(at[0]), "v"(at[1]), "i"(kOffset)
            : "memory");
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          d.f[r][k] = __builtin_shufflevector(h[r][k][0], h[r][k][1], 0, 1, 2, 3);
    }
  };
};

// A wave's 64 x 32 piece of a quadrant.  The operands are passed in turned
// order, so a lane's four sums are four neighbouring columns of one row.
typedef f32x4 Quadrant[4][2];
template <typename T>
__device__ inline void multiply(Quadrant& c, const Fragments<4>& a, const Fragments<2>& b) {
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) c[i][j] = multiply<T>(b.f[j][k], a.f[i][k], c[i][j]);
  __builtin_amdgcn_s_setprio(0);
}

// The copies of one operand's half tiles, step after step.  The buffer's
// descriptor starts at the step's origin and ends where the operand does; the
// scalar work of a step is done beside the matrix instructions (advance), so
// that a copy is one instruction.
template <typename T, bool C, int kPlanes>
struct Copier {
  const char *p, *second;   // of the step at hand; of the other plane
  int64_t step_bytes;
  int left, total;          // 16-byte pieces from p to the operand's last
  int step_pieces;
  int at, steps;            // step at hand, steps of one plane
  int tail;                 // C false: valid k of the last step
  unsigned offset[2][2];    // of the lane's 16 bytes: half tile, round
  int k;                    // C false: the lane's first k
  unsigned lds;             // the wave's part of the first buffer's first half tile
  __amdgpu_buffer_rsrc_t b;

  // `low_first`: the first of the three rounds is the low plane's.
  __device__ inline Copier(const Operand<T>& o, bool low_first, const char* base, int wave, int lane) {
    p = reinterpret_cast<const char*>(kPlanes > 1 && low_first ? o.lo : o.p);
    second = reinterpret_cast<const char*>(kPlanes > 1 && low_first ? o.p : o.lo);
    step_bytes = C ? 2 * kDepth * o.ld : 2 * kDepth;
    step_pieces = static_cast<int>(step_bytes / 16);
    const int64_t elements = C ? (o.depth - 1) * o.ld + (o.valid + 7) / 8 * 8 : (o.valid - 1) * o.ld + o.depth;
    total = o.valid > 0 && o.depth > 0 ? static_cast<int>(elements / 8) : 0;
    left = total;
    at = 0;
    steps = static_cast<int>((o.depth + kDepth - 1) / kDepth);
    tail = static_cast<int>(o.depth - static_cast<int64_t>(steps - 1) * kDepth);
    k = 0;
    if constexpr (!C) k = Half<false>::source_k(wave, lane);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        offset[h][r] = static_cast<unsigned>(2 * (Half<C>::source(wave, lane, r, o.ld) + h * 128 * (C ? 1 : o.ld)));
    lds = lds_address(base) + wave * 1024;
    describe();
  }

  __device__ inline void describe() {
    const int n = left < 0 ? 0 : left > 0x7ffffff ? 0x7ffffff : left;
    b = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), static_cast<short>(0), n * 16, 0x00020000);
    if constexpr (!C)
      if (at == steps - 1 && tail < kDepth && k >= tail)  // past any buffer; the last step of a single plane
#pragma unroll
        for (int h = 0; h < 2; ++h) offset[h][0] = offset[h][1] = 0x80000000u;
  }

  // To the next step.  Of three rounds over the depth, the plane changes before
  // round `first` and, where they differ, round `then`.  Past all of them, zeros.
  __device__ inline void advance(int first, int then) {
    ++at;
    p += step_bytes;
    left -= step_pieces;
    if constexpr (kPlanes == 1) {
      if (at >= steps) left = 0;
    } else if (at == steps || at == 2 * steps || at == 3 * steps) {
      // back to the origin, of the other plane where it is its turn
      const int64_t back = static_cast<int64_t>(steps) * step_bytes;
      p -= back;
      left = at < 3 * steps ? total : 0;
      if (at == first * steps || at == then * steps) {
        const char* other = p;
        p = second;
        second = other;
      }
    }
    describe();
  }

  __device__ inline void copy(int buf, int half) const {
    const unsigned to = lds + buf * 32768 + half * 16384;
#pragma unroll
    for (int r = 0; r < 2; ++r)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (lds_ptr)(uintptr_t)(to + r * 8192), 16,
                                               static_cast<int>(offset[half][r]), 0, 0, 0);
  }
};

// The sums of a tile: quadrant [h][g] of the wave.
struct Sums {
  Quadrant c[2][2];

  // The lane's sums as eights of neighbouring columns; place() comes first.
  static constexpr int kEights = 16;
  int row0, col0;
  __device__ inline void place() {
    const int thread = thread_here(), lane = thread & 63, wave = thread >> 6;
    row0 = (wave >> 2) * 64 + (lane & 15);
    col0 = (wave & 3) * 32 + eight_column(lane);
#pragma unroll
    for (int k = 0; k < kEights; ++k) exchange_fours(quadrant(k)[k >> 1 & 3][0], quadrant(k)[k >> 1 & 3][1]);
  }
  // Columns that eights share: group(k) of kGroups, from group_col().
  static constexpr int kGroups = 2;
  __device__ static inline constexpr int group(int k) { return k & 1; }
  __device__ inline int group_col(int g) const { return g * 128 + col0; }
  // k: row half, row, column half
  __device__ inline Quadrant& quadrant(int k) { return c[k >> 3][k & 1]; }
  __device__ inline int row(int k) const { return (k >> 3) * 128 + (k >> 1 & 3) * 16 + row0; }
  __device__ inline int col(int k) const { return (k & 1) * 128 + col0; }
  __device__ inline f32x4 four(int k, int half) const { return c[k >> 3][k & 1][k >> 1 & 3][half]; }
};

// One tile: sum over k of A(i, k) B(j, k).  kPlanes 3: operands held as sums of
// two planes, high and low; the products low high, high low and high high are
// added, in this order (low low is below fp32's rounding): matrix instructions
// cut their sums to fp32, always to the same side, and the large sums of high
// high are cut by their own steps alone.  `lds`: kLdsBytes.
template <typename T, bool kAC, bool kBC, int kPlanes>
struct Tile256 {
  Copier<T, kAC, kPlanes> ca;
  Copier<T, kBC, kPlanes> cb;

  __device__ inline Tile256(const Operand<T>& a, const Operand<T>& b, const char* lds, int thread)
      : ca(a, true, lds, __builtin_amdgcn_readfirstlane(thread >> 6), thread & 63),
        cb(b, false, lds + 65536, __builtin_amdgcn_readfirstlane(thread >> 6), thread & 63) {}
  // Planes: A low, high, high; B high, low, high.
  __device__ inline void advance_a() { ca.advance(1, 1); }
  __device__ inline void advance_b() { cb.advance(1, 2); }

  // Starts the copies of the first step: B0 A0 B1 A1, two instructions each.
  // LDS is free.
  __device__ inline void start() {
    cb.copy(0, 0);
    ca.copy(0, 0);
    cb.copy(0, 1);
    ca.copy(0, 1);
    advance_b();
    advance_a();
  }

  // Sums the tile.  kStores: memory instructions of the wave, no more and no
  // fewer, that may be under way since start(): another tile's stores, which
  // the first step does not wait for.
  template <int kStores>
  __device__ inline void run(char* lds, Sums& s) {
    const int thread = thread_here(), lane = thread & 63;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int wr = wave >> 2, wc = wave & 3;
    const typename Half<kAC>::template Reader<4> ra(lds_address(lds), wr * 64, lane);
    const typename Half<kBC>::template Reader<2> rb(lds_address(lds + 65536), wc * 32, lane);
    const int all = kPlanes * ca.steps;

#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) s.c[h][g][i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    Fragments<4> fa;
    Fragments<2> b0, b1, b2;
    // A phase that is about to read a half tile waits until at most the two
    // started after it are still under way, and the barrier makes the other
    // waves' parts certain.
    wait_copies<6 + kStores>();
    barrier();
    rb.template read<0>(b0);
    wait_copies<4 + kStores>();
    barrier();
    if (wr == 1) barrier();  // half a phase behind

// `bx`: B0 of this step, read in the last phase of the step before; `by`: of
// the next.  `extra`: stores under way behind the half tiles that the first
// two phases wait for.
#define SPMM_MMA_STEP(buf, bx, by, extra)                      \
  {                                                            \
    ra.template read<(buf) * 32768>(fa);                       \
    cb.copy((buf) ^ 1, 0);                                     \
    wait_copies<4 + (extra)>();                                \
    barrier();                                                 \
    multiply<T>(s.c[0][0], fa, bx);                            \
    barrier();                                                 \
    rb.template read<(buf) * 32768 + 16384>(b1);               \
    ca.copy((buf) ^ 1, 0);                                     \
    wait_copies<4 + (extra)>();                                \
    barrier();                                                 \
    multiply<T>(s.c[0][1], fa, b1);                            \
    barrier();                                                 \
    ra.template read<(buf) * 32768 + 16384>(fa);               \
    cb.copy((buf) ^ 1, 1);                                     \
    wait_copies<4>();                                          \
    barrier();                                                 \
    multiply<T>(s.c[1][1], fa, b1);                            \
    advance_b();                                               \
    barrier();                                                 \
    rb.template read<((buf) ^ 1) * 32768>(by);                 \
    ca.copy((buf) ^ 1, 1);                                     \
    wait_copies<4>();                                          \
    barrier();                                                 \
    multiply<T>(s.c[1][0], fa, bx);                            \
    advance_a();                                               \
    barrier();                                                 \
  }
    int t = 0;
    if constexpr (kStores > 0)
      if (all > 0) {
        SPMM_MMA_STEP(0, b0, b2, kStores)
        SPMM_MMA_STEP(1, b2, b0, 0)
        t = 2;
      }
    for (; t < all; t += 2) {
      SPMM_MMA_STEP(0, b0, b2, 0)
      SPMM_MMA_STEP(1, b2, b0, 0)
    }
#undef SPMM_MMA_STEP
    if (wr == 0) barrier();
    // No copy outlives the loop: LDS is free again.
    wait_copies<0>();
    barrier();
  }
};

template <typename T, bool kAC, bool kBC, int kPlanes>
__device__ inline void multiply_tile(const Operand<T>& a, const Operand<T>& b, char* lds, Sums& s) {
  Tile256<T, kAC, kBC, kPlanes> t(a, b, lds, thread_here());
  t.start();
  t.template run<0>(lds, s);
}

}  // namespace mma
}  // namespace spmm
