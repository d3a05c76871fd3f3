// 128 x 128 tiles of matrix products of fp16 or bf16 operands, four waves.
//
// A step of the sum is 32 deep.  Its operands are copied from memory straight
// to LDS, into a ring of four steps, so that three steps' copies are under way
// beside the one that is multiplied: where a CU has one or two tiles, what
// bounds them is the memory's latency.  One barrier a step: it says that the
// step has arrived and that the step before has been read, whose place the
// copies started next may take.
#pragma once

#include "mma_128.h"
#include "mma_256.h"

namespace spmm {
namespace mma {

// fp16 pairs: operands held as sums of two planes; see multiply_tile.
template <typename T, bool kAC, bool kBC, bool kPair>
struct Ring {
  static constexpr int kDepth = 32;
  static constexpr int kStages = 4;
  static constexpr int kPlanes = kPair ? 2 : 1;
  static constexpr int kOperand = 128 * kDepth * 2;  // bytes of a step of one plane
  static constexpr int kStage = 2 * kPlanes * kOperand;
  static constexpr int kLdsBytes = kStages * kStage;
  static constexpr int kCopies = 4 * kPlanes;  // instructions of a wave and step

  // Layout of a step of one operand: lines of 64 bytes (k contiguous; 16-byte
  // piece c of line i at c ^ (i / 2 % 4)), or of 256 bytes (C; as Half<true>).
  template <bool C>
  struct Copier {
    const char *p, *lo;
    int64_t step_bytes;
    int left, step_pieces;  // 16-byte pieces to the operand's last
    int at, to, last, tail;
    unsigned offset[2];
    int k;

    __device__ inline Copier(const Operand<T>& o, int from, int end, int wave, int lane) {
      step_bytes = C ? 2 * kDepth * o.ld : 2 * kDepth;
      step_pieces = static_cast<int>(step_bytes / 16);
      const int64_t elements = C ? (o.depth - 1) * o.ld + (o.valid + 7) / 8 * 8 : (o.valid - 1) * o.ld + o.depth;
      left = o.valid > 0 && o.depth > 0 ? static_cast<int>(elements / 8) - from * step_pieces : 0;
      p = reinterpret_cast<const char*>(o.p) + from * step_bytes;
      lo = kPair ? reinterpret_cast<const char*>(o.lo) + from * step_bytes : nullptr;
      at = from;
      to = end;
      last = static_cast<int>((o.depth + kDepth - 1) / kDepth) - 1;
      tail = static_cast<int>(o.depth - static_cast<int64_t>(last) * kDepth);
      k = 0;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if constexpr (C) {
          const int line = r * 16 + wave * 4 + lane / 16;
          offset[r] = static_cast<unsigned>(2 * (line * o.ld + ((lane & 15) ^ (Half<true>::swizzle(line) << 1)) * 8));
        } else {
          const int line = r * 64 + wave * 16 + lane / 4;
          k = ((lane & 3) ^ (line >> 1 & 3)) * 8;
          offset[r] = static_cast<unsigned>(2 * (line * o.ld + k));
        }
      }
    }

    // Copies the step at hand to `lds` (the wave's part) and goes on to the
    // next; past the end nothing is read.
    __device__ inline void copy(unsigned lds) {
      const int n = at >= to || left < 0 ? 0 : left > 0x7ffffff ? 0x7ffffff : left;
      if constexpr (!C)
        if (at == last && tail < kDepth && k >= tail) offset[0] = offset[1] = 0x80000000u;  // past any buffer
#pragma unroll
      for (int q = 0; q < kPlanes; ++q) {
        const __amdgpu_buffer_rsrc_t b = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(q == 0 ? p : lo), static_cast<short>(0), n * 16, 0x00020000);
#pragma unroll
        for (int r = 0; r < 2; ++r)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (lds_ptr)(uintptr_t)(lds + q * kOperand + r * 4096), 16,
                                                   static_cast<int>(offset[r]), 0, 0, 0);
      }
      ++at;
      p += step_bytes;
      if constexpr (kPair) lo += step_bytes;
      left -= step_pieces;
    }
  };

  // Addresses of a wave's four fragments of one operand.
  template <bool C>
  struct Reader {
    unsigned at[C ? 4 : 1];
    __device__ inline Reader(int first, int lane) {
      const int q = lane >> 4, i = lane & 15;
      if constexpr (C) {
        const int k = 8 * q + (i >> 2);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          at[r] = k * 256 + ((first / 16 + r) ^ Half<true>::swizzle(k)) * 32 + (lane & 3) * 8;
      } else {
        at[0] = (first + i) * 64 + (q ^ (i >> 1 & 3)) * 16;
      }
    }
  };

#define SPMM_RING_ROWS(n, base)                                                              \
  "ds_read_b128 %[" n "0], %[" base "]\n\tds_read_b128 %[" n "1], %[" base "] offset:1024\n\t" \
  "ds_read_b128 %[" n "2], %[" base "] offset:2048\n\tds_read_b128 %[" n "3], %[" base "] offset:3072\n\t"
#define SPMM_RING_ACROSS(n, base)                                                                 \
  "ds_read_b64_tr_b16 %[" n "00], %[" base "0]\n\tds_read_b64_tr_b16 %[" n "01], %[" base "0] offset:1024\n\t" \
  "ds_read_b64_tr_b16 %[" n "10], %[" base "1]\n\tds_read_b64_tr_b16 %[" n "11], %[" base "1] offset:1024\n\t" \
  "ds_read_b64_tr_b16 %[" n "20], %[" base "2]\n\tds_read_b64_tr_b16 %[" n "21], %[" base "2] offset:1024\n\t" \
  "ds_read_b64_tr_b16 %[" n "30], %[" base "3]\n\tds_read_b64_tr_b16 %[" n "31], %[" base "3] offset:1024\n\t"
#define SPMM_RING_OUT_ROWS(n, f) [n##0] "=&v"(f[0]), [n##1] "=&v"(f[1]), [n##2] "=&v"(f[2]), [n##3] "=&v"(f[3])
#define SPMM_RING_OUT_ACROSS(n, h)                                                              \
  [n##00] "=&v"(h[0][0]), [n##01] "=&v"(h[0][1]), [n##10] "=&v"(h[1][0]), [n##11] "=&v"(h[1][1]), \
      [n##20] "=&v"(h[2][0]), [n##21] "=&v"(h[2][1]), [n##30] "=&v"(h[3][0]), [n##31] "=&v"(h[3][1])
#define SPMM_RING_IN_ACROSS(n, a) [n##0] "v"(a[0]), [n##1] "v"(a[1]), [n##2] "v"(a[2]), [n##3] "v"(a[3])

  // Both operands' fragments of a step of one plane, from LDS at `a` and `b`.
  __device__ static inline void read(const Reader<kAC>& ra, const Reader<kBC>& rb, unsigned a, unsigned b,
                                     u32x4 (&fa)[4], u32x4 (&fb)[4]) {
    unsigned aa[kAC ? 4 : 1], ab[kBC ? 4 : 1];
#pragma unroll
    for (int r = 0; r < (kAC ? 4 : 1); ++r) aa[r] = ra.at[r] + a;
#pragma unroll
    for (int r = 0; r < (kBC ? 4 : 1); ++r) ab[r] = rb.at[r] + b;
    u32x2 ha[4][2], hb[4][2];
    if constexpr (!kAC && !kBC)
      asm volatile(SPMM_RING_ROWS("a", "x") SPMM_RING_ROWS("b", "y") "s_waitcnt lgkmcnt(0)"
                   : SPMM_RING_OUT_ROWS(a, fa), SPMM_RING_OUT_ROWS(b, fb)
                   : [x] "v"(aa[0]), [y] "v"(ab[0])
                   : "memory");
    else if constexpr (!kAC)
      asm volatile(SPMM_RING_ROWS("a", "x") SPMM_RING_ACROSS("b", "y") "s_waitcnt lgkmcnt(0)"
                   : SPMM_RING_OUT_ROWS(a, fa), SPMM_RING_OUT_ACROSS(b, hb)
                   : [x] "v"(aa[0]), SPMM_RING_IN_ACROSS(y, ab)
                   : "memory");
    else
      asm volatile(SPMM_RING_ACROSS("a", "x") SPMM_RING_ACROSS("b", "y") "s_waitcnt lgkmcnt(0)"
                   : SPMM_RING_OUT_ACROSS(a, ha), SPMM_RING_OUT_ACROSS(b, hb)
                   : SPMM_RING_IN_ACROSS(x, aa), SPMM_RING_IN_ACROSS(y, ab)
                   : "memory");
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr (kAC) fa[r] = __builtin_shufflevector(ha[r][0], ha[r][1], 0, 1, 2, 3);
      if constexpr (kBC) fb[r] = __builtin_shufflevector(hb[r][0], hb[r][1], 0, 1, 2, 3);
    }
  }
#undef SPMM_RING_ROWS
#undef SPMM_RING_ACROSS
#undef SPMM_RING_OUT_ROWS
#undef SPMM_RING_OUT_ACROSS
#undef SPMM_RING_IN_ACROSS

  // Adds the steps [from, to) of the sum over k of A(i, k) B(j, k); operands
  // as mma_256.h takes them.
  __device__ static inline void add(const Operand<T>& a, const Operand<T>& b, char* lds, int from, int to,
                                    Sums128<128>& s) {
    const int thread = thread_here(), lane = thread & 63;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    Copier<kAC> ca(a, from, to, wave, lane);
    Copier<kBC> cb(b, from, to, wave, lane);
    const Reader<kAC> ra((wave >> 1) * 64, lane);
    const Reader<kBC> rb((wave & 1) * 64, lane);
    const unsigned base = lds_address(lds);
    unsigned fill = base + wave * 1024;  // where the wave's next copies go
    auto copy = [&]() {
      ca.copy(fill);
      cb.copy(fill + kPlanes * kOperand);
      fill = fill + kStage < base + kLdsBytes ? fill + kStage : base + wave * 1024;
    };
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t) copy();
    unsigned from_lds = base;
    for (int t = from; t < to; ++t) {
      wait_copies<(kStages - 2) * kCopies>();
      barrier();
      copy();
      u32x4 fa[kPlanes][4], fb[kPlanes][4];
#pragma unroll
      for (int q = 0; q < kPlanes; ++q)
        read(ra, rb, from_lds + q * kOperand, from_lds + (kPlanes + q) * kOperand, fa[q], fb[q]);
      from_lds = from_lds + kStage < base + kLdsBytes ? from_lds + kStage : base;
#pragma unroll
      for (int q = 2 * kPlanes - 2; q >= 0; --q)  // (0, 1), (1, 0), then (0, 0)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s.c[i][j] = multiply<T>(fb[q == 2 ? 1 : 0][j], fa[q == 1 ? 1 : 0][i], s.c[i][j]);
    }
    // No copy outlives the loop: LDS is free again.
    wait_copies<0>();
    barrier();
  }
};

}  // namespace mma
}  // namespace spmm
