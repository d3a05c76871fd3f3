// A stable sort by ids: what brings equal ids together in the order of their
// positions, so that sums over them repeat exactly.
//
// Up to kRankMost keys take one launch, in which each key's place is counted:
// the keys below it, and the equal ones before it.  More keys are counted and
// placed digit by digit: count_digits counts the digits of each tile of keys,
// add_digits adds each digit's counts up over the tiles (of few tiles
// place_digits does that by itself, two launches for three), and place_digits
// finds each key's place.  Within a tile a wave takes 64 consecutive keys at a
// time, in order, and ranks each among the equal ones by ballots over the
// digit's bits: no atomic decides an order.
#pragma once

#include "lane_reduce.h"

namespace spmm {

constexpr int kRankThreads = 256;
constexpr int kManyWaves = 4, kFewWaves = 16;    // of a tile's work-group
constexpr int kSortBits = 11;                    // most bits of one digit of several
constexpr int kSortBins = (1 << kSortBits) + 1;  // most values of a single digit
constexpr int64_t kRankMost = 4096;

// Few tiles of many waves, so that place_digits adds up the counts of the tiles
// before by itself: as many as leave it 32768 counts to read, and each wave at
// most 4 rounds of 64 keys, 2 where it has many counts to read.  Beyond, that
// costs more than the launch of add_digits.  A plan for 64 experts: 16384
// choices 7.5 us against 9.0, 524288 11.3 against 14.4, 1048576 (8 rounds) 15.8
// against 18.3; for 511: 100000 choices 10.6 against 12.4, 524288 (8 rounds) 18.3
// against 16.0; for 2048: 16384 choices 13.9 against 17.0, 49143 (4 rounds) 19.0
// against 18.4.
inline int64_t few_most(int bins) { return bins > 256 ? 32768 / bins : 128; }
inline bool few_tiles(int64_t n, int bins) { return n <= few_most(bins) * kFewWaves * 64 * (bins > 256 ? 2 : 4); }

// Keys of a wave in one tile, in rounds of 64: as few as leave 512 tiles at
// most (few_most of the few), as a round waits for the one before it.
inline int sort_rounds(int64_t n, int bins) {
  if (few_tiles(n, bins)) return static_cast<int>(ceil_div(n > 0 ? n : 1, few_most(bins) * kFewWaves * 64));
  int rounds = 1;
  while (rounds < 16 && n > int64_t(512) * kManyWaves * 64 * rounds) rounds *= 2;
  return rounds;
}
inline int64_t sort_tiles(int64_t n, int bins) {
  return ceil_div(n > 0 ? n : 1, (few_tiles(n, bins) ? kFewWaves : kManyWaves) * 64 * sort_rounds(n, bins));
}

// Bits of the values 0 to `most`.
inline int bits_of(int64_t most) {
  int bits = 1;
  while ((most >> bits) != 0) ++bits;
  return bits;
}

// One digit of the keys: (key >> shift) & mask, below `bins`.
struct Digit {
  int shift, bits, bins;
  __device__ inline uint32_t of(uint32_t key) const { return (key >> shift) & ((1u << bits) - 1); }
};

// Counts by wave of the tile's digits in LDS: hist[wave][bins].
template <int W, typename Keys>
__device__ inline void count_tile(uint32_t* hist, Digit d, int64_t n, int rounds, Keys keys) {
  for (int k = threadIdx.x; k < W * d.bins; k += W * 64) hist[k] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * W + wave) * rounds * 64 + lane;
  for (int q = 0; q < rounds; ++q)
    if (first + q * 64 < n) atomicAdd(&hist[wave * d.bins + d.of(keys(first + q * 64))], 1u);
  __syncthreads();
}

// counts: [tiles][bins].  keys(i) gives key i.  (Counting the next digit in
// place_digits, by atomics, costs more than this launch: 10.4 and 22.9 us for
// 6.6 + 2.7 and 9.2 + 4.8.)
template <int W, typename Keys>
__global__ __launch_bounds__(W * 64) void count_digits(Digit d, int64_t n, int rounds, Keys keys, uint32_t* counts) {
  __shared__ uint32_t hist[W * kSortBins];
  count_tile<W>(hist, d, n, rounds, keys);
  for (int b = threadIdx.x; b < d.bins; b += W * 64) {
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += hist[w * d.bins + b];
    counts[static_cast<int64_t>(blockIdx.x) * d.bins + b] = sum;
  }
}

// Exclusive sums of values[0..bins) in LDS over the work-group, in place.
template <int W>
__device__ inline void scan_bins(uint32_t* values, int bins, uint32_t* sums) {
  const int per = (bins + W * 64 - 1) / (W * 64), tid = threadIdx.x;
  uint32_t own = 0;
  for (int k = 0; k < per; ++k)
    if (tid * per + k < bins) own += values[tid * per + k];
  uint32_t run = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = __shfl_up(run, d);
    if ((tid & 63) >= d) run += up;
  }
  if ((tid & 63) == 63) sums[tid >> 6] = run;
  __syncthreads();
  uint32_t at = run - own;
  for (int w = 0; w < (tid >> 6); ++w) at += sums[w];
  for (int k = 0; k < per; ++k) {
    const int b = tid * per + k;
    if (b < bins) {
      const uint32_t v = values[b];
      values[b] = at;
      at += v;
    }
  }
  __syncthreads();
}

// Lanes of the wave with this lane's digit, among those with `valid`.
__device__ inline uint64_t same_digit(uint32_t digit, int bits, bool valid) {
  uint64_t peers = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const bool set = (digit >> b) & 1u;
    const uint64_t has = __ballot(set);
    peers &= set ? has : ~has;
  }
  return peers;
}

// put(i, key, place) for each key; base_of(bin, start) for each digit, with the
// place of its first key, by the first work-group.
template <int W, typename Keys, typename Put, typename Bases>
__global__ __launch_bounds__(W * 64) void place_digits(Digit d, int64_t n, int rounds, Keys keys,
                                                       const uint32_t* counts, const uint32_t* totals, Put put,
                                                       Bases base_of) {
  constexpr int kThreads = W * 64;
  constexpr bool kFew = W == kFewWaves;
  __shared__ uint32_t hist[W * kSortBins], base[kSortBins], before[kFew ? kSortBins : 1], sums[W];
  if constexpr (kFew) {
    for (int b = threadIdx.x; b < d.bins; b += kThreads) base[b] = before[b] = 0;
    __syncthreads();
    const int tiles = static_cast<int>(gridDim.x), own = static_cast<int>(blockIdx.x);
    const int shares = d.bins < kThreads ? kThreads / d.bins : 1;
    for (int k = threadIdx.x; k < shares * d.bins; k += kThreads) {
      const int share = k / d.bins, b = k - share * d.bins;
      uint32_t all = 0, lower = 0;
#pragma unroll 8
      for (int t = share; t < tiles; t += shares) {
        const uint32_t c = counts[static_cast<int64_t>(t) * d.bins + b];
        all += c;
        lower += t < own ? c : 0;
      }
      atomicAdd(&base[b], all);
      atomicAdd(&before[b], lower);
    }
  } else {
    for (int b = threadIdx.x; b < d.bins; b += kThreads) base[b] = totals[b];
  }
  count_tile<W>(hist, d, n, rounds, keys);  // with barriers
  scan_bins<W>(base, d.bins, sums);
  for (int b = threadIdx.x; b < d.bins; b += kThreads) {
    uint32_t at = base[b];
    if (blockIdx.x == 0) base_of(b, at);
    if constexpr (kFew) at += before[b];
    else at += counts[static_cast<int64_t>(blockIdx.x) * d.bins + b];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t c = hist[w * d.bins + b];
      hist[w * d.bins + b] = at;
      at += c;
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  volatile uint32_t* next = hist + wave * d.bins;  // the place of the wave's next key of each digit
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * W + wave) * rounds * 64 + lane;
  for (int q = 0; q < rounds; ++q) {
    const int64_t i = first + q * 64;
    const bool valid = i < n;
    const uint32_t key = valid ? keys(i) : 0, digit = d.of(key);
    const uint64_t peers = same_digit(digit, d.bits, valid);
    if (valid) {
      // A wave's LDS accesses are performed in order: all peers read before the first of them writes.
      const uint64_t before = peers & ((uint64_t(1) << lane) - 1);
      const uint32_t start = next[digit];
      if (before == 0) next[digit] = start + static_cast<uint32_t>(__popcll(peers));
      put(i, key, start + static_cast<uint32_t>(__popcll(before)));
    }
  }
}

// The places of up to kRankMost keys, by counting: a work-group of kRankKeys
// keys holds all keys in LDS, and 16 threads share the comparisons of one key.
// Beyond the keys, `bins` bounds are ranked alike: base_of(b, keys below b).
// 4096 keys: 5 us, against 27 for two digits.
constexpr int kRankKeys = 16;
template <typename Keys, typename Put, typename Bases>
__global__ __launch_bounds__(kRankThreads) void rank_keys(int n, int bins, Keys keys, Put put, Bases base_of) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  __shared__ u32x4 all[kRankMost / 4 + 64];
  __shared__ uint32_t part[kRankThreads / 64][kRankKeys];
  uint32_t* words = reinterpret_cast<uint32_t*>(all);
  // Filled up with keys above all others, which no key counts.
  const int padded = (n + 63) / 64 * 64;
  for (int k = threadIdx.x; k < padded; k += kRankThreads) words[k] = k < n ? keys(k) : ~0u;
  __syncthreads();
  const int own = threadIdx.x % kRankKeys, share = threadIdx.x / kRankKeys, wave = threadIdx.x >> 6;
  const int q = blockIdx.x * kRankKeys + own;
  // A bound counts the keys below it; a key those equal before it too.
  const uint32_t key = q < n ? words[q] : static_cast<uint32_t>(q - n);
  const int index = q < n ? q : 0;
  uint32_t rank = 0;
  for (int k = share; k < padded / 4; k += kRankThreads / kRankKeys) {
    const u32x4 v = all[k];
#pragma unroll
    for (int j = 0; j < 4; ++j) rank += v[j] < key + (4 * k + j < index ? 1u : 0u);
  }
  rank += __shfl_xor(rank, 16);
  rank += __shfl_xor(rank, 32);
  if ((threadIdx.x & 63) < kRankKeys) part[wave][own] = rank;
  __syncthreads();
  if (threadIdx.x >= kRankKeys || q >= n + bins) return;
  rank = 0;
#pragma unroll
  for (int w = 0; w < kRankThreads / 64; ++w) rank += part[w][own];
  if (q < n) put(q, key, rank);
  else base_of(q - n, rank);
}

// Words of the counts and totals of n keys.
inline int64_t sort_words(int64_t n, int bins) { return n <= kRankMost ? 0 : (sort_tiles(n, bins) + 1) * bins; }

// Turns each digit's counts into those of the tiles before, and totals[bins]
// into the counts of all.
spmm_status launch_add_digits(int bins, int64_t tiles, uint32_t* counts, uint32_t* totals, hipStream_t s);

template <typename Keys, typename Put, typename Bases>
spmm_status sort_by_rank(int64_t n, int bins, Keys keys, Put put, Bases base_of, hipStream_t s) {
  hipLaunchKernelGGL((rank_keys<Keys, Put, Bases>), dim3(static_cast<unsigned>(ceil_div(n + bins, kRankKeys))),
                     dim3(kRankThreads), 0, s, static_cast<int>(n), bins, keys, put, base_of);
  return check_launch("rank_keys");
}

// One digit's launches.  `counts` holds sort_words(n, d.bins) words.
template <typename Keys, typename Put, typename Bases>
spmm_status sort_digit(Digit d, int64_t n, Keys keys, uint32_t* counts, Put put, Bases base_of, hipStream_t s) {
  const int64_t tiles = sort_tiles(n, d.bins);
  const int rounds = sort_rounds(n, d.bins);
  uint32_t* totals = counts + tiles * d.bins;
  const dim3 grid(static_cast<unsigned>(tiles));
  auto launch = [&](auto waves) {
    constexpr int W = decltype(waves)::value;
    hipLaunchKernelGGL((count_digits<W, Keys>), grid, dim3(W * 64), 0, s, d, n, rounds, keys, counts);
    if (spmm_status st = check_launch("count_digits")) return st;
    if (W == kManyWaves)
      if (spmm_status st = launch_add_digits(d.bins, tiles, counts, totals, s)) return st;
    hipLaunchKernelGGL((place_digits<W, Keys, Put, Bases>), grid, dim3(W * 64), 0, s, d, n, rounds, keys, counts,
                       totals, put, base_of);
    return check_launch("place_digits");
  };
  if (few_tiles(n, d.bins)) return launch(std::integral_constant<int, kFewWaves>());
  return launch(std::integral_constant<int, kManyWaves>());
}

}  // namespace spmm
