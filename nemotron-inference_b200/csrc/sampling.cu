// Tokens from logits: temperature, top-k, top-p, min-p, and the token on which a given random number falls.
//
// For a row x with largest value m the weights are w_i = e^((x_i - m) / T).  In falling order of x, ties by rising i:
// the first k tokens; of these as many as reach p of their sum (a token stays if those before it sum up to less);
// of these those with w_i >= min_p.  The token is the first in rising order of i at which the sum of what stays
// exceeds u times the whole.
//
// Which token that is changes with the last bits of a sum when a row has many likely tokens: of n equal ones an error
// of e in the sum moves n e of the random numbers to a neighbour, and FP32 sums of 131072 weights would give another
// token than the formula in one of a hundred such rows.  So weights are within 2^-36 of themselves, a thread's sums are
// FP64 and all others whole numbers of 2^-44 of the largest weight.
//
// What bounds it is reading the logits once, and FP64 where all weights are summed up: 16 of a scheduler's cycles for 32
// tokens, 9 us for a row of 131072 on an SM.  Below that the steps of a row wait for one another: a barrier of a cluster
// and the sums behind it take 1.5 us each, and a row with top-p has a dozen.  One block or a cluster goes over a row as
// often as its parameters ask, the first time for the largest and the sum of all weights (by a reference that the first
// tokens give).  No sort: the border of what stays is found by histograms over the values, whose bin at the border is
// listed and ranked one by one (or split again while it holds too many; equal values go by their place).
//   top-k   the k-th largest of the threads' own largest values is no larger than the k-th largest of all: one entry a
//           thread finds a bound that few more than k tokens reach, and these are ranked
//   top-p   some thousand of the tokens tell about where the border lies: the pass that sums up the weights above notes
//           the tokens near it, and the rest goes over these.  (If it lies elsewhere, in one of some hundred rows where
//           few weights are most of the sum: once more with a wider guess, and then all.)  Counts of many tokens do the same.
// The sums in order of i come last, of what stays.
//
// Measured (B200, FP32): 256 rows of 131072 as they are 67 us, 40 of them for the first pass (half of what copying
// reaches); 64 rows of as many settings 80 to 89 us; one row 30 to 33 us; 37 rows of 50001 in BF16, top-k and top-p, 22 us.  Rows that
// lay in the shared memory of clusters of eight blocks took 145, 102, 33 and 22 us: such clusters left a third of the
// SMs' room empty, and SMs idle while a row's steps waited.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "attention.h"
#include "attention_mma.cuh"
#include "common.cuh"
#include "kernels.h"
#include "serving.h"

namespace nmoe {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 1024;
constexpr int kListed = 256;  // tokens ranked one by one
constexpr int kSamples = 16;  // tokens to a thread that guess() goes by, over the blocks of a row
// top_k that the bound from the threads' largest values is for (64 rows, k 50: 39 us, by a guess 49; k 150: 41, 47)
constexpr int kFewK = 160;
constexpr int kVector = 16;   // bytes
constexpr int kMostSlice = 1 << 17;  // tokens to a block (the histogram's words)
constexpr int kMostRowBytes = 1536 * 1024;
constexpr int kTable = 1024;          // powers 2^(i / 1024)
constexpr double kTenth = 6597069766656.0;  // 1.5 * 2^42: a sum with it is a whole number of 2^-10, its lower word in 32 bits
constexpr int kMostUnit = 44;         // weights are counted in 2^-44 of the largest at the finest
constexpr float kAbove = 500.0f;      // binary orders that a weight may lie above the reference's (FP64 has 1023)
constexpr float kBelow = 64.0f;       // and below, before it is 0
constexpr float kWhole = 8388608.0f;    // 2^23: a sum with it is a whole number
constexpr int kWholeBits = 0x4b000000;

enum SearchState { kFound, kTooMany };

// What the blocks of a cluster tell each other; written for all, read behind the next barrier of the cluster.
struct Box {
  float top[kMaxCluster];
  int bad[kMaxCluster];
  double sum[kMaxCluster];           // of e^(x - m)
  u64 part[kMaxCluster];             // of a sum in order of i
  u64 higher[kMaxCluster];           // of weights above those noted
  float low[kMaxCluster], high[kMaxCluster];  // values in a bin
  int first;
  float border_value;
  int border_index;
  int state;  // of a search
};

template <int kBlocks>
struct Shared {
  static constexpr int kSpots = kBlocks == 1 ? 2048 : 1024;  // noted places of a warp
  static constexpr int kAside = kBlocks == 1 ? 160 : 96;     // vectors that wait for each_from()
  Box box;
  double table[kTable];
  uint4 edges[2];
  alignas(16) unsigned bins[3][kBins];  // the histogram: weights in three words of 15 bits and some, or counts
  union {
    u64 sums[kBins];              // of all blocks' histograms
    ulonglong2 own_list[kListed];  // (once a bin is chosen)
  };
  unsigned listed, noted;     // of the cluster's list (in the first block), of this block's
  ulonglong2 list[kListed];   // of the first block: order and weight
  uint4 aside[kWarps][kAside];
  uint16_t aside_at[kWarps][kAside];  // vectors from the warp's first on
  uint16_t spots[kWarps][kSpots];  // from the warp's first token on
  unsigned warp_noted[kWarps];
  u64 warp_part[kWarps];
  double warp_double[kWarps];
  float warp_top[kWarps], warp_low[kWarps];
  int bad;
  int bin;
  u64 before, list_kept;
};

// The last token that stays.
struct Border {
  float value;
  int index;
  __device__ bool keeps(float x, int i) const { return (x > value) | ((x == value) & (i <= index)); }
};

// A token's place in falling order, as a whole number that falls; both zeros are one.
__device__ __forceinline__ u64 order_of(float x, int i) {
  const unsigned bits = __float_as_uint(x + 0.0f);
  const unsigned key = bits ^ ((bits >> 31) != 0 ? 0xffffffffu : 0x80000000u);
  return (static_cast<u64>(key) << 32) | ~static_cast<unsigned>(i);
}
__device__ __forceinline__ Border border_of(u64 order) {
  const unsigned key = static_cast<unsigned>(order >> 32);
  return {__uint_as_float(key ^ ((key >> 31) != 0 ? 0x80000000u : 0xffffffffu)), static_cast<int>(~static_cast<unsigned>(order))};
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ u64 warp_total(u64 x) {
#pragma unroll 1
  for (int step = 16; step > 0; step /= 2) x += __shfl_xor_sync(0xffffffffu, x, step);
  return x;
}
__device__ __forceinline__ u64 warp_upto(u64 x, int lane) {
#pragma unroll 1
  for (int step = 1; step < 32; step *= 2) {
    const u64 other = __shfl_up_sync(0xffffffffu, x, step);
    if (lane >= step) x += other;
  }
  return x;
}
__device__ __forceinline__ double warp_total(double x) {
#pragma unroll 1
  for (int step = 16; step > 0; step /= 2) x += __shfl_xor_sync(0xffffffffu, x, step);
  return x;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll 1
  for (int step = 16; step > 0; step /= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, step));
  return x;
}

// Bins of equal width over the values [low, high], the largest first.  Where it matters is only that they rise with x,
// and that low and high are in two of them if they differ.
struct Bins {
  float low, high, factor, from, scale;

  __device__ void set(float lower, float upper) {
    low = lower;
    high = upper;
    const float range = high - low;
    // (differences beyond FP32's range, or next to its end)
    factor = range > 1e38f ? 0.5f : range < 1e-30f ? 0x1p100f : 1.0f;
    from = factor * high;
    scale = range > 0.0f ? (kBins - 1) / (from - factor * low) : 0.0f;
  }
  __device__ __forceinline__ bool has(float x) const { return x >= low && x <= high; }
  __device__ __forceinline__ int of(float x) const {  // of one that it has
    return min(__float_as_int(fmaf(fmaf(-factor, x, from), scale, kWhole)) - kWholeBits, kBins - 1);
  }
  __device__ float edge(int b) const { return scale > 0.0f ? (from - static_cast<float>(b) / scale) / factor : low; }
};

extern __shared__ __align__(16) uint8_t dynamic_shared[];
#define s (*reinterpret_cast<Shared<kBlocks>*>(dynamic_shared))  // (by name: a pointer in a register has no address space)

template <typename T, int kBlocks>
struct Row {
  static constexpr int kMany = kBlocks == 1 ? 8 : 4;   // values at once: their steps wait for one another
  static constexpr int kAhead = kBlocks == 1 ? 4 : 2;  // vectors on their way
  static constexpr int kSpots = Shared<kBlocks>::kSpots;
  static_assert(32 * (kAhead + 1) <= Shared<kBlocks>::kAside);
  static constexpr int kElements = kVector / sizeof(T);
  // This block's slice, in sixteen bytes each: `vectors` of them from an aligned address on, at which `lead` elements
  // of something else come first; `tokens` of its own, the first of them token `first` + `lead`.
  const uint4* from;
  int vectors, lead, tokens, first;
  int rank, size;        // of the cluster
  int warp, lane, begin, end;  // this warp's vectors
  int each_warp;
  float top, lowest;     // the largest logit, the last that has a weight
  double scale;          // log2(e) / T
  float ratio;           // of all tokens to those that guess() goes by
  int unit;              // weights are counted in 2^-unit

  __device__ __forceinline__ bool whole(int c) const { return c * kElements >= lead && (c + 1) * kElements <= lead + tokens; }
  // Token first + at; -infinity beside the slice.
  __device__ __forceinline__ float value(int at) const {
    return at >= lead && at < lead + tokens ? static_cast<float>(reinterpret_cast<const T*>(from)[at]) : -INFINITY;
  }
  // visit(x, index) of this warp's tokens, a lane each; all lanes together, with -infinity behind the end.
  template <typename Visit>
  __device__ __forceinline__ void each(Visit visit) const {
#pragma unroll 1
    for (int at = begin * kElements + lane; at < end * kElements + lane; at += 32) {
      visit(at < end * kElements ? value(at) : -INFINITY, first + at);
    }
  }
  // Sixteen bytes of the slice, -infinity beside it.
  __device__ __forceinline__ uint4 vector(int c) const {
    constexpr unsigned kNone = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
    uint4 v = make_uint4(kNone, kNone, kNone, kNone);
    if (c < end) {
      if (whole(c)) {
        v = __ldg(from + c);
      } else {
        v = s.edges[c != 0];
      }
    }
    return v;
  }
  // The first and the last sixteen bytes, of which some lie beside the slice.
  __device__ __forceinline__ void set_edges() const {
    constexpr int kWords = kVector / 4;
    if (threadIdx.x < 2 * kWords) {
      const int at = (threadIdx.x / kWords * (vectors - 1)) * kElements + threadIdx.x % kWords * (4 / static_cast<int>(sizeof(T)));
      unsigned bits;
      if constexpr (sizeof(T) == 4) {
        bits = __float_as_uint(value(at));
      } else {
        bits = (__float_as_uint(value(at)) >> 16) | (__float_as_uint(value(at + 1)) & 0xffff0000u);
      }
      reinterpret_cast<unsigned*>(s.edges)[threadIdx.x] = bits;
    }
  }
  // visit(x, index of x[0]), kMany at a time; all lanes together, with -infinity beside the slice.  The index of x[m] is that
  // of x[0] + place(m).  `behind`: a function called after each few vectors.  (The next ones are on their way meanwhile.)
  static __device__ __forceinline__ constexpr int place(int m) { return m + m / kElements * (31 * kElements); }
  template <typename Visit, typename Behind>
  __device__ __forceinline__ void each_many(Visit visit, Behind behind) const {
    constexpr int kTogether = kMany < kElements ? 1 : kMany / kElements;  // vectors
    uint4 next[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) next[k] = vector(begin + lane + 32 * k);
#pragma unroll 1
    for (int c = begin + lane; c < end + lane; c += 32 * kAhead) {
#pragma unroll
      for (int k = 0; k < kAhead; k += kTogether) {
        const int at = first + (c + 32 * k) * kElements;
        unsigned words[kTogether][4];
#pragma unroll
        for (int j = 0; j < kTogether; ++j) {
          words[j][0] = next[k + j].x;
          words[j][1] = next[k + j].y;
          words[j][2] = next[k + j].z;
          words[j][3] = next[k + j].w;
          next[k + j] = vector(c + 32 * (k + j + kAhead));
        }
        float x[kMany];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int m = 0; m < kMany; ++m) x[m] = __uint_as_float(words[m / 4][m % 4]);
          visit(x, at);
        } else {
#pragma unroll 1
          for (int part = 0; part < kElements * kTogether / kMany; ++part) {  // (halves of a vector)
#pragma unroll
            for (int m = 0; m < kMany; m += 2) {
              const int in = m % kElements / 2;
              const unsigned word = kMany < kElements && part != 0 ? words[0][in + 2] : words[m / kElements][in];
              x[m] = __uint_as_float(word << 16);
              x[m + 1] = __uint_as_float(word & 0xffff0000u);
            }
            visit(x, at + kMany * part);
          }
        }
      }
      behind();
    }
  }
  template <typename Visit>
  __device__ __forceinline__ void each_many(Visit visit) const {
    each_many(visit, [] {});
  }
  static __device__ __forceinline__ float largest_of(const float (&x)[kMany]) {
    float largest = x[0];
#pragma unroll
    for (int m = 1; m < kMany; ++m) largest = fmaxf(largest, x[m]);
    return largest;
  }
  static __device__ __forceinline__ double sum_of(const double (&w)[kMany]) {
    double sum = (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
    for (int m = 4; m < kMany; m += 4) sum += (w[m] + w[m + 1]) + (w[m + 2] + w[m + 3]);
    return sum;
  }

  // visit(x[4], index of x[0]) of the fours among whose neighbours in sixteen bytes one is `least` or more: few, mostly, so
  // that these are put aside until each lane has one.  (Visited where they were met, a lane or two of a warp at a time,
  // they took 18 us of 64 rows' time where they take 7 now.)
  template <typename Visit>
  __device__ __forceinline__ void each_from(float least, Visit visit) const {
    uint4* aside = s.aside[warp];
    uint16_t* places = s.aside_at[warp];
    int waiting = 0;
    uint4 next[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) next[k] = vector(begin + lane + 32 * k);
#pragma unroll 1
    for (int c = begin + lane; c < end + lane; c += 32 * kAhead) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const uint4 v = next[k];
        next[k] = vector(c + 32 * (k + kAhead));
        float largest;
        if constexpr (sizeof(T) == 4) {
          largest = fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
        } else {
          auto pair = [](unsigned word) { return *reinterpret_cast<const __nv_bfloat162*>(&word); };
          const float2 two = __bfloat1622float2(__hmax2(__hmax2(pair(v.x), pair(v.y)), __hmax2(pair(v.z), pair(v.w))));
          largest = fmaxf(two.x, two.y);
        }
        const unsigned here = __ballot_sync(0xffffffffu, largest >= least);
        if (largest >= least) {
          const int at = waiting + __popc(here & ((1u << lane) - 1));
          aside[at] = v;
          places[at] = static_cast<uint16_t>(c + 32 * k - begin);
        }
        waiting += __popc(here);
      }
      const bool last = c - lane + 32 * kAhead >= end;
#pragma unroll 1
      while (waiting >= 32 || (last && waiting > 0)) {
        __syncwarp();
        constexpr unsigned kNone = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
        uint4 v = make_uint4(kNone, kNone, kNone, kNone);
        const int at = waiting - 1 - lane;
        int i = 0;
        if (at >= 0) {
          v = aside[at];
          i = first + (begin + places[at]) * kElements;
        }
        if constexpr (sizeof(T) == 4) {
          const float x[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
          visit(x, i);
        } else {
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            const unsigned w0 = half ? v.z : v.x, w1 = half ? v.w : v.y;
            const float x[4] = {__uint_as_float(w0 << 16), __uint_as_float(w0 & 0xffff0000u), __uint_as_float(w1 << 16),
                                __uint_as_float(w1 & 0xffff0000u)};
            visit(x, i + 4 * half);
          }
        }
        __syncwarp();
        waiting -= 32;
      }
      waiting = max(waiting, 0);
    }
  }

  // 2^y with y = (x - reference) scale: the nearest whole number of 2^-10 to y is a power of two times one from the table,
  // the rest r, at most 2^-11, makes a factor of which the first three terms are taken (the fourth is 2^-37).
  __device__ __forceinline__ double power(float x, float reference) const { return power(x, reference, scale); }
  __device__ __forceinline__ double power(float x, float reference, double scale) const {
    constexpr double c1 = 0.6931471805599453, c2 = 0.2402265069591007;  // ln 2, its square / 2
    const double d = static_cast<double>(x) - static_cast<double>(reference);
    const double z = fma(d, scale, kTenth);
    const double r = fma(d, scale, -(z - kTenth));
    const int tenths = __double2loint(z);
    const double w = s.table[tenths & (kTable - 1)];
    const double of_two = __hiloint2double(__double2hiint(w) + ((tenths >> 10) << 20), __double2loint(w));
    return of_two * fma(fma(c2, r, c1), r, 1.0);
  }
  __device__ __forceinline__ double weight_of(float x) const { return x >= lowest ? power(fmaxf(x, lowest), top) : 0.0; }
  __device__ u64 whole_of(double w) const { return __double2ull_rn(w * static_cast<double>(1ull << unit)); }
  __device__ __forceinline__ u64 weight(float x) const { return whole_of(weight_of(x)); }

  // visit(x, index) of the noted tokens, or of all from `least` on for which `in` holds where they were too many to be
  // noted.
  template <typename In, typename Visit>
  __device__ __forceinline__ void each_noted(int count, float least, In in, Visit visit) const {
    if (count > kSpots) {  // (the same for a warp)
      each_from(least, [&](const float (&x)[4], int i) {
#pragma unroll 1
        for (int m = 0; m < 4; ++m) {
          const float one = m == 0 ? x[0] : m == 1 ? x[1] : m == 2 ? x[2] : x[3];
          if (in(one, i + m)) visit(one, i + m);
        }
      });
      return;
    }
#pragma unroll 1
    for (int j = lane; j < count; j += 32) {
      const int at = begin * kElements + s.spots[warp][j];
      visit(value(at), first + at);
    }
  }

  // All threads of the cluster.
  __device__ void sync() const {
    cluster_arrive();
    cluster_wait();
  }
  // Each block's value to all of them; a warp calls it.
  template <typename V>
  __device__ void tell(V* box, V value) const {
    cg::cluster_group cluster = cg::this_cluster();
    if (lane < size) *cluster.map_shared_rank(box, lane) = value;
  }
  // A sum over the block to all blocks' boxes; warp_part keeps those of the warps.
  __device__ __forceinline__ u64 tell_total(u64* box, u64 mine) const {
    mine = warp_total(mine);
    if (lane == 0) s.warp_part[warp] = mine;
    __syncthreads();
    if (warp == 0) tell(box, warp_total(lane < kWarps ? s.warp_part[lane] : 0));
    return mine;
  }
  __device__ u64 total(const u64* box) const {
    u64 all = 0;
    for (int r = 0; r < size; ++r) all += box[r];
    return all;
  }

  __device__ void clear_histogram() {
    for (int i = threadIdx.x; i < 3 * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(s.bins)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) s.listed = s.noted = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void count_weight(int bin, u64 w) {
    atomicAdd(&s.bins[0][bin], static_cast<unsigned>(w) & 0x7fffu);
    atomicAdd(&s.bins[1][bin], static_cast<unsigned>(w >> 15) & 0x7fffu);
    atomicAdd(&s.bins[2][bin], static_cast<unsigned>(w >> 30));
  }

  // All blocks' histograms are there (behind a barrier): each block sums up its share of the bins and tells all.
  __device__ __forceinline__ void merge_bins() {
    cg::cluster_group cluster = cg::this_cluster();
    // as many lanes to a bin as there are blocks
    const int r = threadIdx.x & (size - 1);
    const unsigned* bins = cluster.map_shared_rank(&s.bins[0][0], r);
    u64* sums = cluster.map_shared_rank(s.sums, r);
#pragma unroll 2
    for (int b = rank * (kBins / size) + threadIdx.x / size; b < (rank + 1) * (kBins / size); b += kThreads / size) {
      u64 x = bins[b] + (static_cast<u64>(bins[kBins + b]) << 15) + (static_cast<u64>(bins[2 * kBins + b]) << 30);
#pragma unroll 1
      for (int step = 1; step < size; step *= 2) x += __shfl_xor_sync(0xffffffffu, x, step);
      sums[b] = x;
    }
    sync();
  }
  // The bin at which their sum reaches `target`: s.bin, and the sum before it, s.before.  False where the whole is less.
  __device__ __forceinline__ bool choose_bin(u64 target) {
    static_assert(kBins == 2 * kThreads);
    const u64 one = s.sums[2 * threadIdx.x], own = one + s.sums[2 * threadIdx.x + 1];
    u64 before = warp_upto(own, lane);
    if (lane == 31) s.warp_part[warp] = before;
    if (threadIdx.x == 0) s.bin = -1;
    __syncthreads();
    before += warp_total(lane < warp ? s.warp_part[lane & (kWarps - 1)] : 0) - own;
    if (before < target && target <= before + own) {
      const bool second = target > before + one;
      s.bin = 2 * threadIdx.x + second;
      s.before = second ? before + one : before;
    }
    __syncthreads();
    return s.bin >= 0;
  }

  // A token into this block's list, ...
  __device__ __forceinline__ void list(float x, int i) {
    const unsigned at = atomicAdd(&s.noted, 1u);
    if (at < kListed) s.own_list[at] = make_ulonglong2(order_of(x, i), weight(x));
  }
  // ... which go into the first block's, and are ranked there.  Before them tokens of the sum `before` lie.  The last
  // token before which fewer than `target` lie, or weights that sum up to less; with by_count and top_p < 1 then the
  // last before which less than that part of the sum up to there lies.  kTooMany: the list does not hold all.
  __device__ __forceinline__ SearchState rank_listed(bool by_count, u64 target, u64 before, float top_p, Border& border) {
    cg::cluster_group cluster = cg::this_cluster();
    __syncthreads();
    if (warp == 0) {
      const int n = static_cast<int>(s.noted);
      unsigned base = 0;
      if (n > 0) {
        if (lane == 0) base = atomicAdd(cluster.map_shared_rank(&s.listed, 0), static_cast<unsigned>(n));
        base = __shfl_sync(0xffffffffu, base, 0);
        ulonglong2* list = cluster.map_shared_rank(s.list, 0);
        for (int j = lane; j < n && base + j < kListed; j += 32) list[base + j] = s.own_list[j];
      }
    }
    sync();
    if (rank == 0) {
      const int n = static_cast<int>(s.listed);
      if (n <= kListed) {
        const int lanes = n <= 32 ? 16 : n <= 64 ? 8 : n <= 128 ? 4 : 2;  // to a token
        const int mine = threadIdx.x / lanes, sub = threadIdx.x & (lanes - 1);
        const ulonglong2 own = mine < n ? s.list[mine] : make_ulonglong2(0, 0);
        unsigned count = 0;
        u64 weights = 0;
#pragma unroll 2
        for (int j = sub; j < n; j += lanes) {
          const ulonglong2 other = s.list[j];
          const bool ahead = other.x > own.x;
          count += ahead;
          weights += ahead ? other.y : 0;
        }
#pragma unroll 1
        for (int step = lanes / 2; step > 0; step /= 2) {
          count += __shfl_xor_sync(0xffffffffu, count, step);
          weights += __shfl_xor_sync(0xffffffffu, weights, step);
        }
        if (by_count && top_p < 1.0f) {
          if (mine < n && sub == 0 && count + 1 == target) s.list_kept = weights + own.y;
          __syncthreads();
          target = part_of(top_p, s.list_kept);
          before = 0;
          by_count = false;
        }
        const u64 ahead = before + (by_count ? count : weights), upto = ahead + (by_count ? 1 : own.y);
        if (mine < n && ahead < target && target <= upto) {
          const Border found = border_of(own.x);
          for (int r = sub; r < size; r += lanes) {
            Box* box = cluster.map_shared_rank(&s.box, r);
            box->border_value = found.value;
            box->border_index = found.index;
            box->state = kFound;
          }
        }
      } else if (warp == 0) {
        tell(&s.box.state, static_cast<int>(kTooMany));
      }
    }
    sync();
    const SearchState state = static_cast<SearchState>(s.box.state);
    if (state == kFound) border = {s.box.border_value, s.box.border_index};
    return state;
  }
  // The sum before which tokens stay: p of `sum`, rounded up.
  static __device__ u64 part_of(float top_p, u64 sum) {
    const double part = ceil(static_cast<double>(top_p) * static_cast<double>(sum));
    return part >= 1.0 ? static_cast<u64>(part) : 1;
  }

  // Which tokens a sum in order of i counts: those of a value that `stay` keeps, one each, or those that `border` keeps,
  // their weights.
  struct Counted {
    bool equal;
    Border border, stay;
  };
  __device__ __forceinline__ u64 measure(const Counted& what, float x, int i) const {
    if (what.equal) return x == what.border.value && what.stay.keeps(x, i);
    return what.border.keeps(x, i) ? weight(x) : 0;
  }
  // The first token in order of i at which the sum exceeds u of the whole (equal: `target`).  `mine`: this thread's part of
  // the sum.
  __device__ __forceinline__ int locate(const Counted& what, u64 mine, float u, u64 target) {
    cg::cluster_group cluster = cg::this_cluster();
    tell_total(&s.box.part[rank], mine);
    sync();
    u64 before = 0;
    for (int r = 0; r < rank; ++r) before += s.box.part[r];
    const u64 whole = total(s.box.part);
    if (!what.equal) {
      const double at = u > 0.0f ? static_cast<double>(u) * static_cast<double>(whole) : 0.0;
      target = at < static_cast<double>(whole) ? min(static_cast<u64>(at), whole - 1) : whole - 1;
    }
    if (target >= before && target < before + s.box.part[rank]) {  // this block, ...
      const u64 of_warp = lane < kWarps ? s.warp_part[lane] : 0, upto = warp_upto(of_warp, lane);
      const int owner = __ffs(__ballot_sync(0xffffffffu, target < before + upto)) - 1;
      before += __shfl_sync(0xffffffffu, upto - of_warp, owner);  // ... and this warp's tokens
      const int from = min(owner * each_warp, vectors) * kElements, to = min((owner + 1) * each_warp, vectors) * kElements;
      if (threadIdx.x == 0) s.bin = -1;
      // as many tokens to each thread, and then one by one those of the thread at which it is exceeded
      const int each_thread = (to - from + kThreads - 1) / kThreads;
      const int my_from = min(from + static_cast<int>(threadIdx.x) * each_thread, to), my_to = min(my_from + each_thread, to);
      u64 own = 0;
#pragma unroll 2
      for (int at = my_from; at < my_to; ++at) own += measure(what, value(at), first + at);
      u64 sum = warp_upto(own, lane);
      __syncthreads();  // (what was there has been read)
      if (lane == 31) s.warp_part[warp] = sum;
      __syncthreads();
      sum += before + warp_total(lane < warp ? s.warp_part[lane & (kWarps - 1)] : 0);
      // (single tokens' weights, rounded one by one, may sum up to a little less than their sum did: the last one then)
      const bool mine = own != 0 && sum - own <= target;
      if (mine) atomicMax(&s.bin, static_cast<int>(threadIdx.x));
      __syncthreads();
      const bool none = s.bin < 0, chosen = mine && s.bin == static_cast<int>(threadIdx.x);
      __syncthreads();
      if (none) {
        // Each weighs less than half a unit, together they have one: their first, or their last for u of 1 and more.  (Half as
        // many orders again as `lowest` lies below: the sum of all weights counts those down to kBelow orders.)
        const float light = fmaxf(fmaf(1.5f, lowest - top, top), -FLT_MAX);
#pragma unroll 1
        for (int at = my_from; at < my_to; ++at) {
          const float x = value(at);
          if (!(x >= light && what.border.keeps(x, first + at))) continue;
          if (u >= 1.0f) {
            atomicMax(&s.bin, first + at);
          } else {
            atomicMin(reinterpret_cast<unsigned*>(&s.bin), static_cast<unsigned>(first + at));  // (of -1, the highest)
          }
        }
      } else if (chosen) {
        u64 upto = sum - own;
#pragma unroll 1
        for (int at = my_from; at < my_to && upto <= target; ++at) {
          const u64 one = measure(what, value(at), first + at);
          if (one != 0) s.bin = first + at;
          upto += one;
        }
      }
      __syncthreads();
      if (threadIdx.x < size) *cluster.map_shared_rank(&s.box.first, threadIdx.x) = s.bin;
    }
    sync();
    return s.box.first;
  }

  // What a search by weights leaves for the sums of what stays: this warp's sum above the noted tokens, and these.
  struct Known {
    bool is;
    u64 above;
    int noted;
  };

  // About where `target` tokens lie, or weights that reach top_p of `sum`, by one in `ratio` of the tokens: the bins of
  // `bins` before which tokens surely stay and behind which none does, most likely; false where these say nothing.
  __device__ __forceinline__ bool guess(bool weights, const Bins& bins, u64 target, float top_p, u64 sum, int reach, int& from, int& to) {
    clear_histogram();
    for (int k = 0; k < kSamples / size; k += 2) {
      const int at = begin * kElements + lane + 32 * k;
      const float x[2] = {at < end * kElements ? value(at) : -INFINITY, at + 32 < end * kElements ? value(at + 32) : -INFINITY};
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (!bins.has(x[m])) continue;
        if (weights) {
          count_weight(bins.of(x[m]), weight(x[m]));
        } else {
          atomicAdd(&s.bins[0][bins.of(x[m])], 1u);
        }
      }
    }
    sync();
    merge_bins();
    double middle, above, below;  // how much there may lie between the border and the ends
    if (weights) {
      u64 some = 0;
#pragma unroll 4
      for (int b = lane; b < kBins; b += 32) some += s.sums[b];
      some = warp_total(some);
      // what lies behind the border has this part of the sum (off by about the root of the sum of the weights' squares)
      const double behind = (1.0 - fmax(static_cast<double>(top_p), 0.0)) * (static_cast<double>(sum) / ratio);
      middle = static_cast<double>(some) - behind;
      if (!choose_bin(middle >= 1.0 ? static_cast<u64>(middle) : 1)) return false;
      const double off = sqrt(static_cast<double>(weight(bins.edge(s.bin))) * behind);
      above = 6.0 * reach * off;  // (weights there are larger)
      below = fmin(5.0 * reach * off, (reach == 1 ? 0.9 : 1.0) * behind);
      __syncthreads();
    } else {
      middle = static_cast<double>(target) / ratio;
      above = below = reach * (5.0 * sqrt(middle) + 4.0);
    }
    from = 0;
    if (middle - above >= 1.0) {
      if (!choose_bin(static_cast<u64>(middle - above))) return false;
      from = s.bin;
      __syncthreads();
    }
    to = choose_bin(middle + below >= 1.0 ? static_cast<u64>(middle + below) : 1) ? s.bin : kBins - 1;
    return true;
  }

  // Of the tokens that `stay` keeps, the last before which fewer than `target` of them lie, or (weights) before which
  // weights of less than top_p of their sum lie.  Its value is in [low, top].
  __device__ __forceinline__ Border search(bool weights, const Border stay, u64 target, float top_p, float low, u64 sum, Known& known) {
    Bins bins;
    u64 before = 0;
    int noted = 0;  // of this warp
    float lower = low, upper = top;  // the values that are noted
    auto in_range = [&](float x, int i) { return x >= lower && x <= upper && stay.keeps(x, i); };
    known.is = false;
    const bool all = stay.value < low;  // (what does not stay is not among them)
    float least_of = low, most_of = top;  // the border lies between these
    int reach = 1;
    bool whole = true;
#pragma unroll 1
    for (;;) {
      if (whole) {
        bins.set(low, top);
        int from, to;
        const bool guessed = all && reach > 0 && guess(weights, bins, target, top_p, sum, reach, from, to);
        lower = guessed ? fmaxf(least_of, bins.edge(to + 1)) : least_of;
        upper = guessed && from > 0 ? fminf(most_of, bins.edge(from - 1)) : most_of;
        if (!(lower <= upper)) {
          lower = least_of;
          upper = most_of;
        }
        bins.set(lower, upper);
        double sums = 0.0;  // of those above what is noted, or of all that stay
        unsigned counted = 0;  // above what is noted
        if (lane == 0) s.warp_noted[warp] = 0;
        __syncwarp();
        const float least = all ? lower : fmaxf(fminf(lower, lowest), stay.value);
        each_from(least, [&](const float (&x)[4], int i) {
          if (weights) {
            double w[4];  // (all at once, whether they count or not: their steps wait for one another)
#pragma unroll
            for (int m = 0; m < 4; ++m) w[m] = power(fmaxf(x[m], lowest), top);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const bool counts = all ? x[m] > upper : (x[m] >= lowest) & stay.keeps(x[m], i + m);
              w[m] = counts ? w[m] : 0.0;
            }
            sums += (w[0] + w[1]) + (w[2] + w[3]);
          }
          unsigned mine = 0;
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            counted += x[m] > upper;
            mine |= ((x[m] >= lower) & (x[m] <= upper) & (all | stay.keeps(x[m], i + m))) << m;
          }
          if (mine != 0) {
            unsigned at = atomicAdd(&s.warp_noted[warp], static_cast<unsigned>(__popc(mine)));
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              if (((mine >> m) & 1) == 0) continue;
              if (at < kSpots) s.spots[warp][at] = static_cast<uint16_t>(i + m - first - begin * kElements);
              ++at;
            }
          }
        });
        __syncwarp();
        noted = static_cast<int>(s.warp_noted[warp]);
        const u64 total_of = tell_total(&s.box.higher[rank], weights ? whole_of(sums) : counted);
        known.above = all ? total_of : 0;
        known.noted = noted;
      }
      clear_histogram();
      each_noted(noted, lower, in_range, [&](float x, int) {
        if (!bins.has(x)) return;
        if (weights) {
          count_weight(bins.of(x), weight(x));
        } else {
          atomicAdd(&s.bins[0][bins.of(x)], 1u);
        }
      });
      sync();
      if (whole) {
        const u64 summed = total(s.box.higher);
        if (weights) target = part_of(top_p, all ? sum : summed);
        before = all ? summed : 0;
      }
      merge_bins();
      if ((all && target <= before) || !choose_bin(target - before)) {
        if (!all || (reach == 0 && !weights)) return stay;  // (all of them)
        // Known on both sides by now, and the border in neither: the sum of what lies above, rounded once for a thread, and that
        // of single weights, rounded one by one, have it on different sides of one value.
        if (reach == 0) return {target <= before ? most_of : least_of, INT_MAX};
        // the guess was wrong: a wider one, and then all, on the side where the border is
        if (target <= before) {
          least_of = upper;
        } else {
          most_of = lower;
        }
        reach = reach == 1 ? 4 : 0;
        whole = true;
        before = 0;
        continue;
      }
      whole = false;
      const int chosen = s.bin;
      before += s.before;
      auto in_bin = [&](float x) { return bins.has(x) && bins.of(x) == chosen; };
      each_noted(noted, lower, in_range, [&](float x, int i) {
        if (in_bin(x)) list(x, i);
      });
      Border border;
      known.is = weights && noted <= kSpots;
      if (rank_listed(!weights, target, before, 1.0f, border) == kFound) return border;
      // too many in the bin: their range
      float lowest_of = INFINITY, highest_of = -INFINITY;
      each_noted(noted, lower, in_range, [&](float x, int) {
        if (in_bin(x)) {
          lowest_of = fminf(lowest_of, x);
          highest_of = fmaxf(highest_of, x);
        }
      });
      lowest_of = -warp_max(-lowest_of);
      highest_of = warp_max(highest_of);
      if (lane == 0) {
        s.warp_low[warp] = lowest_of;
        s.warp_top[warp] = highest_of;
      }
      __syncthreads();
      if (warp == 0) {
        tell(&s.box.low[rank], -warp_max(-s.warp_low[lane & (kWarps - 1)]));
        tell(&s.box.high[rank], warp_max(s.warp_top[lane & (kWarps - 1)]));
      }
      sync();
      lowest_of = s.box.low[0];
      highest_of = s.box.high[0];
      for (int r = 1; r < size; ++r) {
        lowest_of = fminf(lowest_of, s.box.low[r]);
        highest_of = fmaxf(highest_of, s.box.high[r]);
      }
      if (lowest_of == highest_of) {  // equal values: by their places
        const u64 w = weight(lowest_of);
        const u64 some = weights ? (target - before + w - 1) / w : target - before;
        const Counted what{true, {lowest_of, INT_MAX}, stay};
        u64 mine = 0;
        each([&](float x, int i) { mine += measure(what, x, i); });
        return {lowest_of, locate(what, mine, 0.0f, some - 1)};
      }
      bins.set(lowest_of, highest_of);
    }
  }

  // The first `k` tokens, few, and of these as many as reach top_p.  False where the list is too short for it.
  __device__ __forceinline__ bool search_few(float largest_of_thread, int k, float top_p, Border& border) {
    Bins bins;
    bins.set(lowest, top);
    clear_histogram();
    if (largest_of_thread >= bins.low) atomicAdd(&s.bins[0][bins.of(largest_of_thread)], 1u);
    sync();
    merge_bins();
    if (!choose_bin(k)) return false;
    const int chosen = s.bin;
    const float least = bins.edge(chosen + 1);  // (surely below)
    if (__any_sync(0xffffffffu, largest_of_thread >= least)) {
      each_from(least, [&](const float (&x)[4], int i) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if (x[m] >= bins.low && bins.of(x[m]) <= chosen) list(x[m], i + m);
        }
      });
    }
    return rank_listed(true, k, 0, top_p, border) == kFound;
  }
};

// `slice`: elements to a block, a multiple of those in sixteen bytes.
template <typename T, int kBlocks>
__global__ void __launch_bounds__(kThreads, kBlocks) sample_kernel(const SampleArgs args, int slice, int unit) {
  constexpr int kElements = kVector / sizeof(T), kMany = Row<T, kBlocks>::kMany;
  cg::cluster_group cluster = cg::this_cluster();
  Row<T, kBlocks> row;
  row.rank = static_cast<int>(cluster.block_rank());
  row.size = static_cast<int>(cluster.num_blocks());
  row.warp = threadIdx.x >> 5;
  row.lane = threadIdx.x & 31;
  const int number = blockIdx.x / row.size, lane = row.lane, warp = row.warp;
  if (threadIdx.x == 0) {
    s.bad = 0;
    s.box.first = -1;
  }
  cluster_arrive();  // (the blocks' shared memory is there)
  wait_for_predecessor();
  release_successor();
  const T* logits = static_cast<const T*>(args.logits) + args.stride * number + static_cast<int64_t>(row.rank) * slice;
  // sixteen bytes at a time from the boundary below; what lies beside the slice is not read
  row.tokens = min(max(args.vocab - row.rank * slice, 0), slice);
  row.lead = static_cast<int>((reinterpret_cast<uintptr_t>(logits) & (kVector - 1)) / sizeof(T));
  row.from = reinterpret_cast<const uint4*>(logits - row.lead);
  row.vectors = row.tokens > 0 ? (row.lead + row.tokens + kElements - 1) / kElements : 0;
  row.each_warp = (row.vectors + kWarps - 1) / kWarps;
  row.first = row.rank * slice - row.lead;
  row.begin = min(warp * row.each_warp, row.vectors);
  row.end = min(row.begin + row.each_warp, row.vectors);
  row.unit = unit;
  // (the same in all blocks)
  row.ratio = fmaxf(1.0f, static_cast<float>((slice / kElements + kWarps) / kWarps * kElements) / (32.0f * (kSamples / row.size)));
  const float temperature = args.temperature.of(number), top_p = args.top_p.of(number);
  const float least = args.min_p.of(number), u = args.uniform[number];
  const int top_k = args.top_k.of(number);
  const bool logprobs = args.logprobs != nullptr, some_k = top_k >= 1 && top_k < args.vocab;
  row.scale = 1.4426950408889634 / static_cast<double>(temperature);
  // the reference: the largest of the first vectors
  float reference = -INFINITY;
  {
    constexpr unsigned kNone = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
    uint4 v = make_uint4(kNone, kNone, kNone, kNone);
    const int c = row.begin + lane;
    if (c < row.end && row.whole(c)) v = __ldg(row.from + c);
    if (row.vectors > 0) row.set_edges();
#pragma unroll 1
    for (int i = threadIdx.x; i < kTable; i += kThreads) s.table[i] = exp2(i * (1.0 / kTable));
    const unsigned words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        reference = fmaxf(reference, __uint_as_float(words[i]));
      } else {
        reference = fmaxf(reference, fmaxf(__uint_as_float(words[i] << 16), __uint_as_float(words[i] & 0xffff0000u)));
      }
    }
  }
  reference = warp_max(reference);
  if (lane == 0) s.warp_low[warp] = reference;
  __syncthreads();
  reference = warp_max(s.warp_low[lane & (kWarps - 1)]);
  if (!(fabsf(reference) < INFINITY)) reference = 0.0f;
  // the first time over the row: the largest, sums of weights and of e^(x - reference)
  float mine = -INFINITY;
  bool bad = false;
  double weights = 0.0, sum = 0.0;
  const bool weighed = temperature > 0.0f && (top_p < 1.0f || !some_k), same = temperature == 1.0f;
  constexpr double kLog2eOf = 1.4426950408889634;
  {
    const float lowest = fmaxf(__double2float_ru(static_cast<double>(reference) - kBelow / row.scale), -FLT_MAX);
    const float least_of = fmaxf(reference - kBelow * 0.693147f, -FLT_MAX);
    const bool summed = logprobs && !(weighed && same);
    const float least_used = fminf(weighed ? lowest : INFINITY, summed ? least_of : INFINITY);
    __syncthreads();  // (the table, the edges)
    row.each_many([&](const float (&x)[kMany], int) {
#pragma unroll
      for (int m = 0; m < kMany; ++m) bad |= x[m] != x[m];
      const float largest = row.largest_of(x);
      mine = fmaxf(mine, largest);
      if (!__any_sync(0xffffffffu, largest >= least_used)) return;
      double w[kMany];
      if (weighed) {
#pragma unroll
        for (int m = 0; m < kMany; ++m) w[m] = row.power(fmaxf(x[m], lowest), reference);
#pragma unroll
        for (int m = 0; m < kMany; ++m) w[m] = x[m] >= lowest ? w[m] : 0.0;
        weights += row.sum_of(w);
      }
      if (summed) {
#pragma unroll
        for (int m = 0; m < kMany; ++m) w[m] = row.power(fmaxf(x[m], least_of), reference, kLog2eOf);
#pragma unroll
        for (int m = 0; m < kMany; ++m) w[m] = x[m] >= least_of ? w[m] : 0.0;
        sum += row.sum_of(w);
      }
    });
    if (weighed && same) sum = weights;
  }
  float top = warp_max(mine);
  if (__any_sync(0xffffffffu, bad) && lane == 0) s.bad = 1;
  if (lane == 0) s.warp_top[warp] = top;
  cluster_wait();  // (and the table and the words above are written)
  __syncthreads();
  if (warp == 0) {
    row.tell(&s.box.top[row.rank], warp_max(s.warp_top[lane & (kWarps - 1)]));
    row.tell(&s.box.bad[row.rank], s.bad);
  }
  row.sync();
  top = s.box.top[0];
  int any_bad = s.box.bad[0];
  for (int r = 1; r < row.size; ++r) {
    top = fmaxf(top, s.box.top[r]);
    any_bad |= s.box.bad[r];
  }
  row.top = top;
  if (any_bad || !(fabsf(top) < INFINITY)) {  // no distribution
    if (row.rank == 0 && threadIdx.x == 0) {
      args.tokens[number] = -1;
      if (logprobs) args.logprobs[number] = NAN;
    }
    return;  // (behind a barrier that all blocks have passed; nobody reads a neighbour any more)
  }
  // by the largest now; a block whose own largest lies far above its reference goes over its slice once more
  const float own = warp_max(s.warp_top[lane & (kWarps - 1)]);
  row.lowest = top;
  if (temperature > 0.0f) {
    // 2^-1.5 of a unit and less is 0
    const double reach = (unit + 1.5) / row.scale;
    row.lowest = fmaxf(__double2float_ru(static_cast<double>(top) - reach), -FLT_MAX);
  }
  u64 all_weights = 0;  // of the row
  if (weighed) {
    if (own >= reference && static_cast<double>(own) - static_cast<double>(reference) <= kAbove / row.scale) {
      weights *= exp2((static_cast<double>(reference) - static_cast<double>(top)) * row.scale);
    } else {
      weights = 0.0;
      if (own >= row.lowest) row.each([&](float x, int) { weights += row.weight_of(x); });
    }
    row.tell_total(&s.box.part[row.rank], row.whole_of(weights));
    row.sync();
    all_weights = row.total(s.box.part);
  }
  if (logprobs) {
    if (own >= reference && static_cast<double>(own) - static_cast<double>(reference) <= kAbove / kLog2eOf) {
      sum *= exp2((static_cast<double>(reference) - static_cast<double>(top)) * kLog2eOf);
    } else {
      sum = 0.0;
      const float least_of = fmaxf(top - kBelow * 0.693147f, -FLT_MAX);
      if (own >= least_of) row.each([&](float x, int) { sum += x >= least_of ? row.power(fmaxf(x, least_of), top, kLog2eOf) : 0.0; });
    }
    sum = warp_total(sum);
    if (lane == 0) s.warp_double[warp] = sum;
    __syncthreads();
    if (warp == 0) row.tell(&s.box.sum[row.rank], warp_total(lane < kWarps ? s.warp_double[lane] : 0.0));  // (read behind a barrier that is still to come)
  }
  typename Row<T, kBlocks>::Counted what{true, {top, INT_MAX}, {-INFINITY, INT_MAX}};  // the first of the largest
  typename Row<T, kBlocks>::Known known;
  known.is = false;
  if (temperature > 0.0f) {
    Border border{-INFINITY, INT_MAX};
    bool done = false;
    if (some_k && top_k <= kFewK) done = row.search_few(mine, top_k, top_p, border);
#pragma unroll 1
    for (int by_weight = 0; by_weight < 2 && !done; ++by_weight) {
      if (by_weight ? !(top_p < 1.0f) : !some_k) continue;
      float low = border.value;
      if (by_weight && !some_k) {
        // what lies lower never stays (a hundredth less than that, and nothing for the rounding of weights)
        const double cut = 0.99 * (1.0 - fmax(static_cast<double>(top_p), 0.0)) / args.vocab;
        low = __double2float_rd(static_cast<double>(top) + static_cast<double>(temperature) * log(cut));
      }
      border = row.search(by_weight != 0, border, top_k, top_p, fmaxf(low, row.lowest), all_weights, known);
    }
    if (least > 0.0f && temperature < INFINITY) {  // w >= p where x - m >= T ln p
      const double below = least < 1.0f ? static_cast<double>(temperature) * log(static_cast<double>(least)) : 0.0;
      const float value = __double2float_ru(static_cast<double>(top) + below);
      if (value > border.value) {
        border = {fminf(value, top), INT_MAX};
        known.is = false;
      }
    }
    what = {false, border, border};
  }
  u64 stays = 0;
  if (!what.equal && weighed && !(what.border.value > -INFINITY)) {
    stays = row.whole_of(weights);
  } else if (known.is) {
    stays = lane == 0 ? known.above : 0;
    row.each_noted(known.noted, 0.0f, [](float, int) { return false; }, [&](float x, int i) { stays += row.measure(what, x, i); });
  } else {
    row.each_from(what.border.value, [&](const float (&x)[4], int i) {
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const u64 w = what.equal ? x[m] == top : row.whole_of(row.power(fmaxf(x[m], row.lowest), top));
        stays += (x[m] >= row.lowest) & what.border.keeps(x[m], i + m) ? w : 0;
      }
    });
  }
  int token = row.locate(what, stays, u, 0);
  if (static_cast<unsigned>(token) >= static_cast<unsigned>(args.vocab)) token = -1;  // (there is always one)
  if (row.rank == 0 && threadIdx.x == 0) {
    args.tokens[number] = token;
    if (logprobs && token >= 0) {
      double all = 0.0;
      for (int r = 0; r < row.size; ++r) all += s.box.sum[r];
      const float x = static_cast<float>(static_cast<const T*>(args.logits)[args.stride * number + token]);
      args.logprobs[number] = static_cast<float>(static_cast<double>(x) - static_cast<double>(top) - log(all));
    }
  }
}

#undef s

template <typename T, int kBlocks>
cudaError_t launch(const SampleArgs& args, cudaStream_t stream) {
  // One block to a row where there are enough; else as many as find room beside each other, but for what clusters leave
  // empty, those of eight a quarter (16 rows, top-k: in clusters of eight, some behind the others, 41 us, of four 27).
  const int room = device_sms() * kBlocks * 9 / 10;
  constexpr int kElements = kVector / sizeof(T);
  int size = 1;
  while (size < kMaxCluster &&
         ((args.vocab + size - 1) / size > kMostSlice ||
          (static_cast<int64_t>(args.rows) * size * 2 <= (size * 2 == 8 ? room * 4 / 5 : room) && args.vocab > 2048 * size))) {
    size *= 2;
  }
  const int slice = ((args.vocab + size - 1) / size + kElements - 1) / kElements * kElements;
  int bits = 0;
  while ((1ll << bits) < args.vocab) ++bits;
  const int unit = std::min(kMostUnit, 63 - bits);  // so that the sum of all weights has 64 bits
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t err = allow_shared_memory_once(sample_kernel<T, kBlocks>, allowed);
  if (err != cudaSuccess) return err;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim = {static_cast<unsigned>(size), 1, 1};
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(args.rows) * size);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = sizeof(Shared<kBlocks>);
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, sample_kernel<T, kBlocks>, args, slice, unit);
}

}  // namespace

bool sample_supported(int vocab, bool bf16) {
  return static_cast<int64_t>(vocab) * (bf16 ? 2 : 4) <= kMostRowBytes;
}

cudaError_t launch_sample(const SampleArgs& args, bool bf16, cudaStream_t stream) {
  // Few rows: one block to an SM, whose threads then have registers enough (64 rows of 131072: 80 us; two blocks, which
  // spill, 96).  Many, of which an SM has more than one block's: two, which hide each other's waits (128 rows, top-p 106 us,
  // 96 rows, top-k 55; with one block to an SM 133 and 57; 256 rows as they are 67, 95).
  if (static_cast<int64_t>(args.rows) * 20 > device_sms() * 9) {
    return bf16 ? launch<__nv_bfloat16, 2>(args, stream) : launch<float, 2>(args, stream);
  }
  return bf16 ? launch<__nv_bfloat16, 1>(args, stream) : launch<float, 1>(args, stream);
}

}  // namespace nmoe
