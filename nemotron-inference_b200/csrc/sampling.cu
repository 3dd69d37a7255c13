// Tokens from logits: temperature, top-k, top-p, min-p, and the token on which a given random number falls.
//
// For a row x with largest value m the weights are w_i = e^((x_i - m) / T).  In falling order of x, ties by rising i:
// the first k tokens; of these as many as reach p of their sum (a token stays if those before it sum up to less);
// of these those with w_i >= min_p.  The token is the first in rising order of i at which the sum of what stays
// exceeds u times the whole.
//
// Which token that is changes with the last bits of a sum when a row has many likely tokens: of n equal ones an error
// of e in the sum moves n e of the random numbers to a neighbour, and FP32 sums of 131072 weights would give another
// token than the formula in one of a hundred such rows.  So weights are whole numbers of 2^-44 of the largest, or
// smaller units where the vocabulary leaves room, each within 2^-31 of itself and without a bias, and sums are 64-bit
// integers: they do not depend on an order, and rows come out the same whatever the split.
//
// What bounds it is reading the logits once.  A cluster of blocks holds a row in its shared memory and goes over it as
// often as the parameters ask.  No sort: the border of what stays is found by histograms over the values, whose bin at
// the border is listed and ranked one by one (or split again while it holds too many; equal values go by their place).
//   top-k   the k-th largest of the threads' own largest values is no larger than the k-th largest of all: one entry a
//           thread finds a bound that few more than k tokens reach, and these are ranked
//   top-p   a sixteenth of the tokens tells about where the border lies: the pass that takes the exact sums of all weights
//           and of those above notes the tokens near it, and the rest goes over these.  (If it lies elsewhere: over
//           all with weights of (1 - p) / n of the largest's, below which no token of n stays.)
// The sums in order of i come last, of what stays; where all do, they are taken in FP32 first, whose error has a bound
// (kSumError): only where the random number lies within it of another token the row is gone over with exact weights.
//
// Most of the code runs once for a row, so instructions that are not in the cache yet cost more than the work of a
// pass: loops take a token to a lane, without unrolling, where the arithmetic is long.
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
constexpr int kSpots = 64;    // noted places of a warp
constexpr int kSamples = 2;   // tokens to a thread that guess() goes by
constexpr int kFewK = 160;    // top_k that the bound from the threads' largest values is for
constexpr int kVector = 16;   // bytes
constexpr int kSliceBytes = 64 * 1024;  // of a row to a block where clusters suffice: two blocks to an SM
constexpr int kMostSliceBytes = 192 * 1024;
// Logarithms of the weights to base 2: 42 bits behind the point, of which ten choose a power in the table.
constexpr int kTable = 1024;
constexpr double kPoint = 1536.0;       // 1.5 * 2^10: a sum with it has 2^-42 as its last bit
constexpr int kPointHigh = 0x40980000;  // its upper word
constexpr int kMostUnit = 46;           // weights are counted in 2^-46 of the largest at the finest
// Relative error of a sum of weights 2^y in FP32 at most: y = (x - m) c is off by 3 2^-24 |y|, and the average of |y|
// by weight is at most log2 of the number of tokens, below 19: 2.4e-6; ex2.approx adds 2^-22, sums of up to 96 in a
// thread, in fours, 26 2^-24.
constexpr double kSumError = 5e-6;
constexpr float kWhole = 8388608.0f;    // 2^23: a sum with it is a whole number
constexpr int kWholeBits = 0x4b000000;

enum SearchState { kUnsure, kFound, kTooMany };

// What the blocks of a cluster tell each other; written for all, read behind the next barrier of the cluster.
struct Box {
  float top[kMaxCluster];
  int bad[kMaxCluster];
  float sum[kMaxCluster];            // of e^(x - m)
  u64 part[kMaxCluster];             // of a sum in order of i
  u64 higher[kMaxCluster];           // of weights above those noted
  float low[kMaxCluster], high[kMaxCluster];  // values in a bin
  int first;
  float border_value;
  int border_index;
  int state;  // of a search
};

struct Shared {
  Box box;
  unsigned table[kTable];     // 2^(i / 1024), units of 2^-31
  alignas(16) unsigned bins[3][kBins];  // the histogram: weights in three words of 15 bits and some, or counts
  union {
    u64 sums[kBins];              // of all blocks' histograms
    ulonglong2 own_list[kListed];  // (once a bin is chosen)
  };
  unsigned listed, noted;     // of the cluster's list (in the first block), of this block's
  ulonglong2 list[kListed];   // of the first block: order and weight
  uint16_t spots[kWarps][kSpots];  // from the warp's first token on
  u64 warp_part[kWarps];
  float warp_top[kWarps], warp_low[kWarps];
  int bad;
  int bin;
  u64 before, list_kept;
};

// The last token that stays.
struct Border {
  float value;
  int index;
  __device__ bool keeps(float x, int i) const { return x > value || (x == value && i <= index); }
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
#define s (*reinterpret_cast<Shared*>(dynamic_shared))  // (by name: a pointer in a register has no address space)

template <typename T>
struct Row {
  static constexpr int kElements = kVector / sizeof(T);
  int first;             // number of the token at the slice's first sixteen bytes
  int rank, size;        // of the cluster
  int warp, lane, begin, end;  // this warp's chunks of sixteen bytes
  int each_warp;         // chunks
  float top, lowest;     // the largest logit, the last that has a weight
  double scale;          // log2(e) / T
  float fast_scale;      // the same
  bool fast;             // sums in FP32 have their bound
  float ratio;           // of all tokens to those that guess() goes by
  int unit;              // weights are counted in 2^-unit

  // This block's slice; places beside it are -infinity.
  static __device__ __forceinline__ uint4* slice_at() {
    return reinterpret_cast<uint4*>(dynamic_shared + (sizeof(Shared) + 15) / 16 * 16);
  }
  __device__ __forceinline__ float value(int at) const { return static_cast<float>(reinterpret_cast<const T*>(slice_at())[at]); }
  // visit(x, index) of this warp's tokens, a lane each; all lanes together, with -infinity behind the end.
  template <typename Visit>
  __device__ __forceinline__ void each(Visit visit) const {
#pragma unroll 1
    for (int at = begin * kElements + lane; at < end * kElements + lane; at += 32) {
      visit(at < end * kElements ? value(at) : -INFINITY, first + at);
    }
  }
  // visit(x[4], index of x[0]), four at a time, all lanes together, with -infinity behind the end.
  template <typename Visit>
  __device__ __forceinline__ void each_four(Visit visit) const {
    constexpr int kFours = kElements / 4;
#pragma unroll 1
    for (int at = begin * kFours + lane; at < end * kFours + lane; at += 32) {
      float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (at < end * kFours) {
        if constexpr (sizeof(T) == 4) {
          const float4 v = reinterpret_cast<const float4*>(slice_at())[at];
          x[0] = v.x;
          x[1] = v.y;
          x[2] = v.z;
          x[3] = v.w;
        } else {
          const uint2 v = reinterpret_cast<const uint2*>(slice_at())[at];
          x[0] = __uint_as_float(v.x << 16);
          x[1] = __uint_as_float(v.x & 0xffff0000u);
          x[2] = __uint_as_float(v.y << 16);
          x[3] = __uint_as_float(v.y & 0xffff0000u);
        }
      }
      visit(x, first + 4 * at);
    }
  }

  // A token's weight.  z holds its logarithm to base 2 as a whole number of 2^-42, the upper word units of 2^-10.
  // 2^(that) is a power from the table, times 1 + q with q = 2^r - 1 a polynomial of the rest r < 2^-10 (its first
  // three terms: the fourth is 2^-46).  r is cut off at 2^-33, q rounded to 2^-31.
  __device__ __forceinline__ u64 weight(float x) const {
    constexpr float c1 = 6.7690154351557163e-4f, c2 = 2.2909784980808780e-7f, c3 = 5.1691529e-11f;  // ln(2)^n 2^-10n / n!
    const double z = fma(static_cast<double>(fmaxf(x, lowest)) - static_cast<double>(top), scale, kPoint);
    const int whole = __double2hiint(z) - kPointHigh;
    const float r = __uint_as_float(0x3f800000u | (static_cast<unsigned>(__double2loint(z)) >> 9)) - 1.0f;
    const float q = fmaf(fmaf(fmaf(c3, r, c2), r, c1), r, 0x1p-8f);
    const unsigned one_and_q = __float_as_uint(q) + (0x80000000u - 0x3b800000u);
    const u64 w = static_cast<u64>(s.table[whole & (kTable - 1)]) * one_and_q;  // units of 2^-62
    return x >= lowest ? ((w >> (61 - unit - (whole >> 10))) + 1) >> 1 : 0;
  }
  // Nearly 2^-unit of it, and that as a whole number.
  __device__ __forceinline__ float fast_weight(float x) const {
    return x >= lowest ? exp2_approx((x - top) * fast_scale) : 0.0f;
  }
  __device__ u64 whole_of(float w) const { return __double2ull_rn(static_cast<double>(w) * static_cast<double>(1ull << unit)); }
  __device__ float fast_sum() const {
    float sum = 0.0f;
    each_four([&](const float (&x)[4], int) {
      sum += (fast_weight(x[0]) + fast_weight(x[1])) + (fast_weight(x[2]) + fast_weight(x[3]));
    });
    return sum;
  }

  // visit(x, index) of the noted tokens, or of all for which `in` holds where they were too many to be noted.
  template <typename In, typename Visit>
  __device__ __forceinline__ void each_noted(int count, In in, Visit visit) const {
    const bool all = count > kSpots;
    const int stop = all ? (end - begin) * kElements : count;
#pragma unroll 1
    for (int j = lane; j < stop; j += 32) {
      const int at = begin * kElements + (all ? j : s.spots[warp][j]);
      const float x = value(at);
      if (!all || in(x, first + at)) visit(x, first + at);
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

  // Which tokens a sum in order of i counts, and what each one counts.
  enum Measure { kEqual, kExact, kFast };
  struct Counted {
    Measure measure;
    Border border;  // of what counts; kEqual: also the value
    Border stay;    // (kEqual)
  };
  __device__ __forceinline__ u64 measure(const Counted& what, float x, int i) const {
    if (what.measure == kEqual) return x == what.border.value && what.stay.keeps(x, i);
    const u64 w = what.measure == kFast ? whole_of(fast_weight(x)) : weight(x);
    return what.border.keeps(x, i) ? w : 0;
  }
  // The first token in order of i at which the sum exceeds u of the whole (kEqual: `target`).  `mine`: this thread's part of
  // the sum.  Left in box.first for all blocks, behind one more barrier; -1 where FP32 sums leave it open.
  __device__ __forceinline__ int locate(const Counted& what, u64 mine, float u, u64 target) {
    cg::cluster_group cluster = cg::this_cluster();
    tell_total(&s.box.part[rank], mine);
    if (threadIdx.x == 0) s.box.first = -1;  // (what was there has been read)
    sync();
    u64 before = 0, margin = 0;
    for (int r = 0; r < rank; ++r) before += s.box.part[r];
    const u64 whole = total(s.box.part);
    if (what.measure != kEqual) {
      const double at = u > 0.0f ? static_cast<double>(u) * static_cast<double>(whole) : 0.0;
      target = at < static_cast<double>(whole) ? min(static_cast<u64>(at), whole - 1) : whole - 1;
      if (what.measure == kFast) margin = static_cast<u64>(2.0 * kSumError * static_cast<double>(whole)) + 1;
    }
    if (target >= before && target < before + s.box.part[rank]) {  // this block, ...
      const u64 of_warp = lane < kWarps ? s.warp_part[lane] : 0, upto = warp_upto(of_warp, lane);
      const int owner = __ffs(__ballot_sync(0xffffffffu, target < before + upto)) - 1;
      before += __shfl_sync(0xffffffffu, upto - of_warp, owner);  // ... and this warp's tokens
      const int from = min(owner * each_warp, chunks()) * kElements, to = min((owner + 1) * each_warp, chunks()) * kElements;
#pragma unroll 1
      for (int start = from; start < to; start += kThreads) {
        const int at = start + static_cast<int>(threadIdx.x);
        const float x = at < to ? value(at) : -INFINITY;
        const u64 own = at < to ? measure(what, x, first + at) : 0;
        u64 sum = warp_upto(own, lane);
        __syncthreads();  // (what was there has been read)
        if (lane == 31) s.warp_part[warp] = sum;
        __syncthreads();
        sum += before + warp_total(lane < warp ? s.warp_part[lane & (kWarps - 1)] : 0);
        if (sum > target && sum - own <= target && sum > target + margin && sum - own + margin <= target) {
          for (int r = 0; r < size; ++r) *cluster.map_shared_rank(&s.box.first, r) = first + at;
        }
        before += warp_total(lane < kWarps ? s.warp_part[lane] : 0);
        if (before > target) break;
      }
    }
    sync();
    return s.box.first;
  }
  __device__ int chunks() const { return all_chunks; }
  int all_chunks;  // of the block

  // What a search by weights leaves for the sums of what stays: this warp's sum above the noted tokens, and these.
  struct Known {
    bool is;
    u64 above;
    int noted;
  };

  // About where the weights reach top_p of their sum, by one in `ratio` of the tokens: false where these say nothing, else
  // the bins of `bins` before which tokens surely stay and behind which none does, most likely.
  __device__ __forceinline__ bool guess(const Bins& bins, float top_p, int& from, int& to) {
    const u64 sum = whole_of(fast_sum());
    clear_histogram();
#pragma unroll 1
    for (int at = begin * kElements + lane, k = 0; k < kSamples && at < end * kElements; at += 32, ++k) {
      const float x = value(at);
      if (bins.has(x)) count_weight(bins.of(x), weight(x));
    }
    tell_total(&s.box.part[rank], sum);
    sync();
    merge_bins();
    u64 some = 0;
#pragma unroll 4
    for (int b = lane; b < kBins; b += 32) some += s.sums[b];
    some = warp_total(some);
    // the border is where what lies behind has these parts of it
    const double part = static_cast<double>(total(s.box.part)) / ratio;
    // (a sum of such parts of what lies behind is off by about the root of the sum of the weights' squares)
    const double behind = (1.0 - fmax(static_cast<double>(top_p), 0.0)) * part, middle = static_cast<double>(some) - behind;
    if (!choose_bin(middle >= 1.0 ? static_cast<u64>(middle) : 1)) return false;
    const double at_border = static_cast<double>(weight(bins.edge(s.bin)));
    const double width = fmin(4.0 * sqrt(at_border * behind), 0.5 * behind);
    __syncthreads();
    from = 0;
    if (middle - width >= 1.0) {
      if (!choose_bin(static_cast<u64>(middle - width))) return false;
      from = s.bin;
      __syncthreads();
    }
    if (!choose_bin(middle + width >= 1.0 ? static_cast<u64>(middle + width) : 1)) return false;
    to = s.bin;
    return true;
  }

  // Of the tokens that `stay` keeps, the last before which fewer than `target` of them lie, or (weights) before which
  // weights of less than top_p of their sum lie.  Its value is in [low, top].
  __device__ __forceinline__ Border search(bool weights, const Border stay, u64 target, float top_p, float low, Known& known) {
    Bins bins;
    bins.set(low, top);
    u64 before = 0;
    int noted = 0;  // of this warp
    float lower = low, upper = top;  // the values that are noted
    auto in_range = [&](float x, int i) { return x >= lower && x <= upper && stay.keeps(x, i); };
    known.is = false;
    bool near = weights && fast && stay.value < low;
    if (near) {
      int from, to;
      near = guess(bins, top_p, from, to);
      if (near) {
        lower = fmaxf(low, bins.edge(to + 1));
        if (from > 0) upper = bins.edge(from - 1);
        bins.set(lower, upper);
      }
    }
    bool whole = true;
#pragma unroll 1
    for (;;) {
      if (whole) {
        u64 exact = 0, above = 0;
        noted = 0;
        each_four([&](const float (&x)[4], int i) {
          const float largest = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          if (!__any_sync(0xffffffffu, largest >= fmaxf(fminf(lower, lowest), stay.value))) return;
          if (weights) {
            u64 w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = weight(x[k]);
            if (!near) {
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = stay.keeps(x[k], i + k) ? w[k] : 0;
            }
            exact += (w[0] + w[1]) + (w[2] + w[3]);
            if (__any_sync(0xffffffffu, largest > upper)) {
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = x[k] > upper ? w[k] : 0;
              above += (w[0] + w[1]) + (w[2] + w[3]);
            }
          }
          if (!__any_sync(0xffffffffu, largest >= lower)) return;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const bool mine = in_range(x[k], i + k);
            const unsigned all = __ballot_sync(0xffffffffu, mine);
            const int at = noted + __popc(all & ((1u << lane) - 1));
            if (mine && at < kSpots) s.spots[warp][at] = static_cast<uint16_t>(i + k - first - begin * kElements);
            noted += __popc(all);
          }
        });
        if (weights) {
          known.above = tell_total(&s.box.higher[rank], above);
          known.noted = noted;
          __syncthreads();
          tell_total(&s.box.part[rank], exact);
        }
      }
      clear_histogram();
      each_noted(noted, in_range, [&](float x, int) {
        if (!bins.has(x)) return;
        if (weights) {
          count_weight(bins.of(x), weight(x));
        } else {
          atomicAdd(&s.bins[0][bins.of(x)], 1u);
        }
      });
      sync();
      if (weights && whole) {
        target = part_of(top_p, total(s.box.part));
        before = total(s.box.higher);
      }
      merge_bins();
      if ((near && target <= before) || !choose_bin(target - before)) {
        if (!near) return stay;
        near = false;  // the guess was wrong: all of them
        lower = low;
        upper = top;
        bins.set(lower, upper);
        before = 0;
        continue;
      }
      whole = false;
      const int chosen = s.bin;
      before += s.before;
      auto in_bin = [&](float x) { return bins.has(x) && bins.of(x) == chosen; };
      each_noted(noted, in_range, [&](float x, int i) {
        if (in_bin(x)) list(x, i);
      });
      Border border;
      known.is = weights && noted <= kSpots;
      if (rank_listed(!weights, target, before, 1.0f, border) == kFound) return border;
      // too many in the bin: their range
      float lowest_of = INFINITY, highest_of = -INFINITY;
      each_noted(noted, in_range, [&](float x, int) {
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
        const Counted what{kEqual, {lowest_of, INT_MAX}, stay};
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
    // (of the threads that have one at all; each_four() gave them out)
    if (largest_of_thread >= bins.low && bins.of(largest_of_thread) <= chosen) {
#pragma unroll 1
      for (int four = begin * (kElements / 4) + lane; four < end * (kElements / 4); four += 32) {
#pragma unroll 1
        for (int at = 4 * four; at < 4 * four + 4; ++at) {
          const float x = value(at);
          if (x >= bins.low && bins.of(x) <= chosen) list(x, first + at);
        }
      }
    }
    return rank_listed(true, k, 0, top_p, border) == kFound;
  }
};

// `slice`: elements to a block, a multiple of those in sixteen bytes.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs args, int slice, int unit) {
  uint4* data = Row<T>::slice_at();
  constexpr int kElements = kVector / sizeof(T);
  cg::cluster_group cluster = cg::this_cluster();
  Row<T> row;
  row.rank = static_cast<int>(cluster.block_rank());
  row.size = static_cast<int>(cluster.num_blocks());
  row.warp = threadIdx.x >> 5;
  row.lane = threadIdx.x & 31;
  const int number = blockIdx.x / row.size, lane = row.lane, warp = row.warp;
  if (threadIdx.x == 0) s.bad = 0;
  cluster_arrive();  // (the blocks' shared memory is there)
#pragma unroll 1
  for (int i = threadIdx.x; i < kTable; i += kThreads) s.table[i] = __double2uint_rn(exp2(31.0 + i * (1.0 / kTable)));
  wait_for_predecessor();
  release_successor();
  const T* logits = static_cast<const T*>(args.logits) + args.stride * number + static_cast<int64_t>(row.rank) * slice;
  const int tokens = min(max(args.vocab - row.rank * slice, 0), slice);
  // sixteen bytes at a time from the boundary below; what lies beside the slice is not read
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(logits) & (kVector - 1)) / sizeof(T));
  row.all_chunks = tokens > 0 ? (lead + tokens + kElements - 1) / kElements : 0;
  row.each_warp = (row.all_chunks + kWarps - 1) / kWarps;
  row.first = row.rank * slice - lead;
  row.begin = min(warp * row.each_warp, row.all_chunks);
  row.end = min(row.begin + row.each_warp, row.all_chunks);
  row.unit = unit;
  // (the same in all blocks)
  row.ratio = fmaxf(1.0f, static_cast<float>((slice / kElements + kWarps) / kWarps * kElements) / (32.0f * kSamples));
  float mine = -INFINITY;  // the largest
  bool bad = false;
  {
    const uint4* from = reinterpret_cast<const uint4*>(logits - lead);
    constexpr int kAtOnce = 8;
#pragma unroll 1
    for (int start = row.begin + lane; start < row.end; start += 32 * kAtOnce) {
      uint4 v[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int c = start + 32 * k;
        if (c < row.end && c * kElements >= lead && (c + 1) * kElements <= lead + tokens) v[k] = __ldcs(from + c);
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int c = start + 32 * k;
        if (c < row.end && c * kElements >= lead && (c + 1) * kElements <= lead + tokens) data[c] = v[k];
      }
    }
    if (lead > 0 || (lead + tokens) % kElements != 0) {  // the ends
#pragma unroll 1
      for (int c = row.begin + lane; c < row.end; c += 32) {
        if (c * kElements >= lead && (c + 1) * kElements <= lead + tokens) continue;
        T* some = reinterpret_cast<T*>(data + c);
#pragma unroll 1
        for (int i = 0; i < kElements; ++i) {
          const int at = c * kElements + i - lead;
          some[i] = at >= 0 && at < tokens ? logits[at] : static_cast<T>(-INFINITY);
        }
      }
    }
    row.each_four([&](const float (&x)[4], int) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        mine = fmaxf(mine, x[k]);
        bad |= x[k] != x[k];
      }
    });
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
  // (asked for meanwhile)
  const float temperature = args.temperature.of(number), top_p = args.top_p.of(number);
  const float least = args.min_p.of(number), u = args.uniform[number];
  const int top_k = args.top_k.of(number);
  row.sync();
  top = s.box.top[0];
  int any_bad = s.box.bad[0];
  for (int r = 1; r < row.size; ++r) {
    top = fmaxf(top, s.box.top[r]);
    any_bad |= s.box.bad[r];
  }
  row.top = top;
  const bool logprobs = args.logprobs != nullptr;
  if (any_bad || !(fabsf(top) < INFINITY)) {  // no distribution
    if (row.rank == 0 && threadIdx.x == 0) {
      args.tokens[number] = -1;
      if (logprobs) args.logprobs[number] = NAN;
    }
    return;  // (behind a barrier that all blocks have passed; nobody reads a neighbour any more)
  }
  if (logprobs) {
    float sum = 0.0f;
    row.each_four([&](const float (&x)[4], int) {
      float e[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) e[k] = exp2_approx((x[k] - top) * kLog2e);
      sum += (e[0] + e[1]) + (e[2] + e[3]);
    });
    auto over_warp = [&] {
#pragma unroll 1
      for (int step = 16; step > 0; step /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, step);
    };
    over_warp();
    if (lane == 0) s.warp_low[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      sum = lane < kWarps ? s.warp_low[lane] : 0.0f;
      over_warp();
      row.tell(&s.box.sum[row.rank], sum);  // (read behind a barrier that is still to come)
    }
    __syncthreads();
  }
  typename Row<T>::Counted what{Row<T>::kEqual, {top, INT_MAX}, {-INFINITY, INT_MAX}};  // the first of the largest
  typename Row<T>::Known known;
  known.is = false;
  if (temperature > 0.0f) {
    row.scale = 1.4426950408889634 / static_cast<double>(temperature);
    row.fast_scale = static_cast<float>(row.scale);
    row.fast = temperature >= 1e-30f && temperature <= 1e30f;
    // 2^-1.5 of a unit and less is 0 (so shifts in weight() stay below 64)
    const double reach = (unit + 1.5) * 0.6931471805599453 * static_cast<double>(temperature);
    row.lowest = fmaxf(__double2float_ru(static_cast<double>(top) - reach), -FLT_MAX);
    Border border{-INFINITY, INT_MAX};
    const bool some_k = top_k >= 1 && top_k < args.vocab;
    bool done = false;
    if (some_k && top_k <= kFewK) done = row.search_few(mine, top_k, top_p, border);
#pragma unroll 1
    for (int by_weight = 0; by_weight < 2 && !done; ++by_weight) {
      if (by_weight ? !(top_p < 1.0f) : !some_k) continue;
      float low = border.value;
      if (by_weight && !some_k && row.fast) {
        // what lies lower never stays (a hundredth less than that, and nothing for the rounding of weights)
        const double cut = 0.99 * (1.0 - fmax(static_cast<double>(top_p), 0.0)) / args.vocab;
        low = __double2float_rd(static_cast<double>(top) + static_cast<double>(temperature) * log(cut));
      }
      border = row.search(by_weight != 0, border, top_k, top_p, fmaxf(low, row.lowest), known);
    }
    if (least > 0.0f && temperature < INFINITY) {  // w >= p where x - m >= T ln p
      const double below = least < 1.0f ? static_cast<double>(temperature) * log(static_cast<double>(least)) : 0.0;
      const float value = __double2float_ru(static_cast<double>(top) + below);
      if (value > border.value) {
        border = {fminf(value, top), INT_MAX};
        known.is = false;
      }
    }
    what = {!(border.value > -INFINITY) && row.fast ? Row<T>::kFast : Row<T>::kExact, border, border};
  }
  int token = -1;
#pragma unroll 1
  for (int attempt = 0; attempt < 2 && token < 0; ++attempt) {
    u64 stays = 0;
    if (what.measure == Row<T>::kFast) {
      stays = row.whole_of(row.fast_sum());
    } else if (known.is) {
      stays = lane == 0 ? known.above : 0;
      row.each_noted(known.noted, [](float, int) { return false; }, [&](float x, int i) { stays += row.measure(what, x, i); });
    } else {
      row.each_four([&](const float (&x)[4], int i) {
        if (!__any_sync(0xffffffffu, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= what.border.value)) return;
        u64 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = row.measure(what, x[k], i + k);
        stays += (w[0] + w[1]) + (w[2] + w[3]);
      });
    }
    token = row.locate(what, stays, u, 0);
    what.measure = Row<T>::kExact;
  }
  if (row.rank == 0 && threadIdx.x == 0) {
    args.tokens[number] = token;
    if (logprobs) {
      double all = 0.0;
      for (int r = 0; r < row.size; ++r) all += s.box.sum[r];
      const float x = static_cast<float>(static_cast<const T*>(args.logits)[args.stride * number + token]);
      args.logprobs[number] = static_cast<float>(static_cast<double>(x) - static_cast<double>(top) - log(all));
    }
  }
}

#undef s

size_t shared_bytes(int slice, int size) { return (sizeof(Shared) + 15) / 16 * 16 + static_cast<size_t>(slice) * size + kVector; }

static_assert((sizeof(Shared) + 15) / 16 * 16 + kMostSliceBytes + kVector <= kMaxSharedBytes);

template <typename T>
cudaError_t launch(const SampleArgs& args, cudaStream_t stream) {
  // As few blocks to a row as hold it; more where rows are few, so that all SMs read.
  const int64_t bytes = static_cast<int64_t>(args.vocab) * sizeof(T);
  const int64_t limit = bytes > static_cast<int64_t>(kSliceBytes) * kMaxCluster ? kMostSliceBytes : kSliceBytes;
  int size = 1;
  while (size < kMaxCluster && (bytes > limit * size || (args.rows * size * 2 <= device_sms() && bytes > 8192 * size))) size *= 2;
  constexpr int kElements = kVector / sizeof(T);
  const int slice = ((args.vocab + size - 1) / size + kElements - 1) / kElements * kElements;
  int bits = 0;
  while ((1ll << bits) < args.vocab) ++bits;
  const int unit = std::min(kMostUnit, 63 - bits);  // so that the sum of all weights has 64 bits
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t err = allow_shared_memory_once(sample_kernel<T>, allowed);
  if (err != cudaSuccess) return err;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim = {static_cast<unsigned>(size), 1, 1};
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(args.rows) * size);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = shared_bytes(slice, sizeof(T));
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, sample_kernel<T>, args, slice, unit);
}

}  // namespace

bool sample_supported(int vocab, bool bf16) {
  return static_cast<int64_t>(vocab) * (bf16 ? 2 : 4) <= static_cast<int64_t>(kMostSliceBytes) * kMaxCluster;
}

cudaError_t launch_sample(const SampleArgs& args, bool bf16, cudaStream_t stream) {
  return bf16 ? launch<__nv_bfloat16>(args, stream) : launch<float>(args, stream);
}

}  // namespace nmoe
