// Tokens from logits: temperature, top-k, top-p, min-p, and the token on which a given random number falls.
//
// For a row x with largest value m the weights are w_i = e^((x_i - m) / T).  In falling order of x, ties by rising i:
// the first k tokens; of these as many as reach p of their sum (a token stays if those before it sum up to less);
// of these those with w_i >= min_p.  The token is the first in rising order of i at which the sum of what stays
// exceeds u times the whole.
//
// Which token that is changes with the last bits of a sum when a row has many likely tokens: of n equal ones an error
// of e in the sum moves n e of the random numbers to a neighbour, and FP32 sums of 131072 weights would give another
// token than the formula in one of a hundred such rows.  So weights are whole numbers of 2^-44, from exponentials in
// FP64, and sums are 64-bit integers: they do not depend on an order, and rows come out the same whatever the split.
// (Weights below 2^-45 of the largest are 0.)
//
// What bounds it is reading the logits once.  A cluster of blocks holds a row in its shared memory and goes over it as
// often as the parameters ask: the largest; a histogram of counts and weights over (m - x) / T; the few tokens in the
// bin at the border, ranked one by one (a bin with too many is split again by its bits; equal values by their place);
// the sums of what stays in order of i.  No sort.
#include <cooperative_groups.h>

#include <climits>
#include <cmath>

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
constexpr float kBinsPerUnit = 32.0f;      // of (m - x) / T: weights end at 31.2
constexpr double kOne = 17592186044416.0;  // 2^44, a weight of 1
constexpr int kListed = 256;               // tokens ranked one by one
constexpr int kVector = 16;                // bytes
constexpr int kSliceBytes = 64 * 1024;     // of a row to a block where clusters suffice: two blocks to an SM
constexpr int kMostSliceBytes = 192 * 1024;

// What the blocks of a cluster tell each other; written for all, read behind the next barrier of the cluster.
struct Box {
  float top[kMaxCluster];
  int bad[kMaxCluster];
  double sum[kMaxCluster];                      // of e^(x - m)
  u64 segment_weight[kMaxCluster];              // of the histogram
  unsigned segment_count[kMaxCluster];
  u64 part[kMaxCluster];                        // of a sum in order of i
  unsigned low[kMaxCluster], high[kMaxCluster];  // keys in a bin
  int first[kMaxCluster];
  int bin;
  unsigned bin_count, before_count;
  u64 before_weight;
  unsigned border_key;
  int border_index;
  u64 kept;
};

struct Shared {
  Box box;
  unsigned low[kBins], high[kBins], count[kBins];  // the histogram: weights in two words
  unsigned listed;
  unsigned list_key[kListed];
  int list_index[kListed];
  u64 list_weight[kListed];
  u64 warp_part[kWarps];
  float warp_top[kWarps];
  double warp_sum[kWarps];
  unsigned warp_low[kWarps], warp_high[kWarps];
  int warp_first[kWarps];
  int bad;
};

// Floats as whole numbers of the same order; both zeros are one.
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned bits = __float_as_uint(x + 0.0f);
  return bits ^ ((bits >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float(key ^ ((key >> 31) != 0 ? 0x80000000u : 0xffffffffu));
}

// The last token that stays.
struct Border {
  unsigned key;
  int index;
  __device__ bool keeps(unsigned k, int i) const { return k > key || (k == key && i <= index); }
};

template <typename T>
struct Row {
  static constexpr int kElements = kVector / sizeof(T);
  Shared& s;
  const uint4* data;     // this block's slice; places beside it are -infinity
  int chunks, first;     // sixteen bytes each; number of the token at the first one's begin
  int rank, size;        // of the cluster
  int warp, lane, begin, end;  // this warp's chunks
  float top;
  double inverse;        // 1 / T
  float bin_scale;
  bool level_one;        // the histogram is that of bins of (m - x) / T

  __device__ Row(Shared& shared) : s(shared) {}

  // visit(x, index) of this warp's tokens in order, lanes side by side.
  template <typename Visit>
  __device__ __forceinline__ void each(Visit visit) const {
#pragma unroll 2
    for (int c = begin + lane; c < end; c += 32) chunk(c, visit);
  }
  template <typename Visit>
  __device__ __forceinline__ void chunk(int c, Visit visit) const {
    const uint4 v = data[c];
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
    const int at = first + c * kElements;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        visit(__uint_as_float(w[i]), at + i);
      } else {
        visit(__uint_as_float(w[i] << 16), at + 2 * i);
        visit(__uint_as_float(w[i] & 0xffff0000u), at + 2 * i + 1);
      }
    }
  }

  __device__ double weight(float x) const { return exp((static_cast<double>(x) - static_cast<double>(top)) * inverse); }
  static __device__ u64 fixed(double w) { return __double2ull_rn(w * kOne); }
  // of a token's weight, kBins where that is certainly 0
  __device__ int bin_of(float x) const {
    const float at = x == top ? 0.0f : (top - x) * bin_scale;
    return at < static_cast<float>(kBins) ? static_cast<int>(at) : kBins;  // (-infinity with T infinite: none)
  }

  __device__ void sync() const {
    __syncthreads();
    cluster_sync_all();
  }
  // Each block's value to all of them; one thread calls it.
  template <typename V>
  __device__ void tell(V* box, V value) const {
    cg::cluster_group cluster = cg::this_cluster();
    for (int r = 0; r < size; ++r) *cluster.map_shared_rank(box, r) = value;
  }

  // The histogram of the tokens that `bin` gives one below kBins, each block's share of the bins summed over all.
  template <typename Bin>
  __device__ void histogram(Bin bin) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) s.low[b] = s.high[b] = s.count[b] = 0;
    __syncthreads();
    each([&](float x, int) {
      const int b = bin(x);
      if (b >= kBins) return;
      const u64 w = fixed(weight(x));
      if (w == 0) return;
      const unsigned low = static_cast<unsigned>(w);
      const unsigned before = atomicAdd(&s.low[b], low);
      const unsigned rest = static_cast<unsigned>(w >> 32) + (before + low < before);
      if (rest != 0) atomicAdd(&s.high[b], rest);
      atomicAdd(&s.count[b], 1u);
    });
    sync();
    // (nobody else reads this block's share of its own histogram)
    cg::cluster_group cluster = cg::this_cluster();
    const int share = kBins / size;
    u64 weight_sum = 0;
    unsigned count_sum = 0;
    for (int b = rank * share + threadIdx.x; b < (rank + 1) * share; b += kThreads) {
      u64 w = 0;
      unsigned n = 0;
      for (int r = 0; r < size; ++r) {
        w += *cluster.map_shared_rank(&s.low[b], r) + (static_cast<u64>(*cluster.map_shared_rank(&s.high[b], r)) << 32);
        n += *cluster.map_shared_rank(&s.count[b], r);
      }
      s.low[b] = static_cast<unsigned>(w);
      s.high[b] = static_cast<unsigned>(w >> 32);
      s.count[b] = n;
      weight_sum += w;
      count_sum += n;
    }
#pragma unroll
    for (int step = 16; step > 0; step /= 2) {
      weight_sum += __shfl_xor_sync(0xffffffffu, weight_sum, step);
      count_sum += __shfl_xor_sync(0xffffffffu, count_sum, step);
    }
    if (lane == 0) {
      s.warp_part[warp] = weight_sum;
      s.warp_low[warp] = count_sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kWarps; ++w) {
        weight_sum += s.warp_part[w];
        count_sum += s.warp_low[w];
      }
      tell(&s.box.segment_weight[rank], weight_sum);
      tell(&s.box.segment_count[rank], count_sum);
    }
    sync();
  }

  // The tokens' measures (whole numbers) in order of i: the first token at which their sum exceeds target(sum of all),
  // to `told` of all blocks and behind a barrier, or by the block that has it alone.
  template <typename Measure, typename Target, typename Found>
  __device__ void locate(Measure measure, Target target_of, Found found) {
    u64 mine = 0;
    each([&](float x, int i) { mine += measure(x, i); });
#pragma unroll
    for (int step = 16; step > 0; step /= 2) mine += __shfl_xor_sync(0xffffffffu, mine, step);
    if (lane == 0) s.warp_part[warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 all = 0;
      for (int w = 0; w < kWarps; ++w) all += s.warp_part[w];
      tell(&s.box.part[rank], all);
    }
    sync();
    u64 total = 0, before = 0;
    for (int r = 0; r < size; ++r) {
      if (r < rank) before += s.box.part[r];
      total += s.box.part[r];
    }
    const u64 target = target_of(total);
    for (int w = 0; w < warp; ++w) before += s.warp_part[w];
    if (target < before || target >= before + mine) return;
    // this warp
#pragma unroll 1
    for (int c = begin; c < end; c += 32) {
      u64 own = 0;
      if (c + lane < end) chunk(c + lane, [&](float x, int i) { own += measure(x, i); });
      u64 upto = own;
#pragma unroll
      for (int step = 1; step < 32; step *= 2) {
        const u64 other = __shfl_up_sync(0xffffffffu, upto, step);
        if (lane >= step) upto += other;
      }
      const unsigned beyond = __ballot_sync(0xffffffffu, before + upto > target);
      if (beyond != 0) {
        if (lane == __ffs(beyond) - 1) {
          u64 at = before + upto - own;
          bool done = false;
          chunk(c + lane, [&](float x, int i) {
            at += measure(x, i);
            if (!done && at > target) {
              found(i);
              done = true;
            }
          });
        }
        return;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }

  // The last token, in falling order, before which fewer than `target` tokens, or weights that sum up to less, lie;
  // `kept`: the sum of weights up to it.  Where there are not as many: all.
  __device__ Border search(bool by_count, u64 target, u64& kept) {
    unsigned low = 0, high = 0xffffffffu;  // keys
    int shift = -1;                        // of the bins; -1: of (m - x) / T
    u64 before_weight = 0, before_count = 0;
#pragma unroll 1
    for (;;) {
      auto bin = [&](float x) {
        if (shift < 0) return bin_of(x);
        const unsigned key = key_of(x);
        return key >= low && key <= high ? static_cast<int>((high - key) >> shift) : kBins;
      };
      if (shift >= 0 || !level_one) {
        histogram(bin);
        level_one = shift < 0;
      }
      const int share = kBins / size;
      int owner = -1;
      for (int r = 0; r < size; ++r) {
        const u64 w = s.box.segment_weight[r], n = s.box.segment_count[r];
        if (target <= (by_count ? before_count + n : before_weight + w)) {
          owner = r;
          break;
        }
        before_weight += w;
        before_count += n;
      }
      if (owner < 0) {
        kept = before_weight;
        return {0, INT_MAX};
      }
      if (rank == owner && warp == 0) {
        for (int start = rank * share; start < (rank + 1) * share; start += 32) {
          const int b = start + lane;
          const bool there = b < (rank + 1) * share;
          const u64 w = there ? s.low[b] + (static_cast<u64>(s.high[b]) << 32) : 0, n = there ? s.count[b] : 0;
          u64 upto_w = w, upto_n = n;
#pragma unroll
          for (int step = 1; step < 32; step *= 2) {
            const u64 other_w = __shfl_up_sync(0xffffffffu, upto_w, step), other_n = __shfl_up_sync(0xffffffffu, upto_n, step);
            if (lane >= step) {
              upto_w += other_w;
              upto_n += other_n;
            }
          }
          const unsigned reached = __ballot_sync(0xffffffffu, target <= (by_count ? before_count + upto_n : before_weight + upto_w));
          if (reached != 0) {
            if (lane == __ffs(reached) - 1) {
              tell(&s.box.bin, b);
              tell(&s.box.bin_count, static_cast<unsigned>(n));
              tell(&s.box.before_count, static_cast<unsigned>(before_count + upto_n - n));
              tell(&s.box.before_weight, before_weight + upto_w - w);
            }
            break;
          }
          before_weight += __shfl_sync(0xffffffffu, upto_w, 31);
          before_count += __shfl_sync(0xffffffffu, upto_n, 31);
        }
      }
      if (threadIdx.x == 0) s.listed = 0;
      sync();
      const int chosen = s.box.bin;
      const unsigned inside = s.box.bin_count;
      before_weight = s.box.before_weight;
      before_count = s.box.before_count;
      auto in_bin = [&](float x) { return bin(x) == chosen && (shift >= 0 || fixed(weight(x)) != 0); };
      if (inside <= kListed) {
        rank_listed(in_bin, by_count, target, before_count, before_weight, static_cast<int>(inside));
        kept = s.box.kept;
        return {s.box.border_key, s.box.border_index};
      }
      // too many: their keys' range
      unsigned lowest = 0xffffffffu, highest = 0;
      each([&](float x, int) {
        if (in_bin(x)) {
          lowest = min(lowest, key_of(x));
          highest = max(highest, key_of(x));
        }
      });
      lowest = __reduce_min_sync(0xffffffffu, lowest);
      highest = __reduce_max_sync(0xffffffffu, highest);
      if (lane == 0) {
        s.warp_low[warp] = lowest;
        s.warp_high[warp] = highest;
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        for (int w = 1; w < kWarps; ++w) {
          lowest = min(lowest, s.warp_low[w]);
          highest = max(highest, s.warp_high[w]);
        }
        tell(&s.box.low[rank], lowest);
        tell(&s.box.high[rank], highest);
      }
      sync();
      low = 0xffffffffu;
      high = 0;
      for (int r = 0; r < size; ++r) {
        low = min(low, s.box.low[r]);
        high = max(high, s.box.high[r]);
      }
      if (low == high) {  // equal values: by their places
        const u64 w = fixed(weight(value_of(low)));
        const u64 stay = by_count ? target - before_count : (target - before_weight + w - 1) / w;
        locate([&](float x, int) -> u64 { return key_of(x) == low; }, [&](u64) { return stay - 1; },
               [&](int i) { tell(&s.box.border_index, i); });
        sync();
        kept = before_weight + stay * w;
        return {low, s.box.border_index};
      }
      shift = max(0, 32 - __clz(high - low) - 10);
    }
  }

  template <typename InBin>
  __device__ __forceinline__ void rank_listed(InBin in_bin, bool by_count, u64 target, u64 before_count, u64 before_weight, int n) {
    cg::cluster_group cluster = cg::this_cluster();
    each([&](float x, int i) {
      if (in_bin(x)) {
        const unsigned at = atomicAdd(cluster.map_shared_rank(&s.listed, 0), 1u);
        *cluster.map_shared_rank(&s.list_key[at], 0) = key_of(x);
        *cluster.map_shared_rank(&s.list_index[at], 0) = i;
      }
    });
    sync();
    if (rank == 0) {
      const int mine = threadIdx.x;
      unsigned key = 0;
      int index = 0;
      u64 own = 0;
      if (mine < n) {
        key = s.list_key[mine];
        index = s.list_index[mine];
        own = fixed(weight(value_of(key)));
        s.list_weight[mine] = own;
      }
      __syncthreads();
      if (mine < n) {
        u64 count = before_count, weights = before_weight;
        for (int j = 0; j < n; ++j) {
          const bool before = Border{key, index - 1}.keeps(s.list_key[j], s.list_index[j]);
          count += before;
          weights += before ? s.list_weight[j] : 0;
        }
        const u64 before = by_count ? count : weights, upto = by_count ? count + 1 : weights + own;
        if (before < target && target <= upto) {
          tell(&s.box.border_key, key);
          tell(&s.box.border_index, index);
          tell(&s.box.kept, weights + own);
        }
      }
    }
    sync();
  }
};

// `slice`: elements to a block, a multiple of those in sixteen bytes.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs args, int slice) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared& s = *reinterpret_cast<Shared*>(raw);
  uint4* data = reinterpret_cast<uint4*>(raw + (sizeof(Shared) + 15) / 16 * 16);
  constexpr int kElements = kVector / sizeof(T);
  cg::cluster_group cluster = cg::this_cluster();
  Row<T> row(s);
  row.rank = static_cast<int>(cluster.block_rank());
  row.size = static_cast<int>(cluster.num_blocks());
  row.warp = threadIdx.x >> 5;
  row.lane = threadIdx.x & 31;
  const int number = blockIdx.x / row.size, lane = row.lane, warp = row.warp;
  wait_for_predecessor();
  release_successor();
  const T* logits = static_cast<const T*>(args.logits) + args.stride * number + static_cast<int64_t>(row.rank) * slice;
  const int tokens = min(max(args.vocab - row.rank * slice, 0), slice);
  // sixteen bytes at a time from the boundary below; what lies beside the slice is not read
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(logits) & (kVector - 1)) / sizeof(T));
  row.data = data;
  row.chunks = tokens > 0 ? (lead + tokens + kElements - 1) / kElements : 0;
  row.first = row.rank * slice - lead;
  const int each = (row.chunks + kWarps - 1) / kWarps;
  row.begin = min(warp * each, row.chunks);
  row.end = min(row.begin + each, row.chunks);
  row.level_one = false;
  float top = -INFINITY;
  bool bad = false;
  {
    const uint4* from = reinterpret_cast<const uint4*>(logits - lead);
    auto see = [&](float x, int) {
      top = fmaxf(top, x);
      bad |= x != x;
    };
#pragma unroll 8
    for (int c = row.begin + lane; c < row.end; c += 32) {
      uint4 v;
      if (c * kElements >= lead && (c + 1) * kElements <= lead + tokens) {
        v = __ldcs(from + c);
      } else {
        alignas(kVector) T some[kElements];
#pragma unroll
        for (int i = 0; i < kElements; ++i) {
          const int at = c * kElements + i - lead;
          some[i] = at >= 0 && at < tokens ? logits[at] : static_cast<T>(-INFINITY);
        }
        v = *reinterpret_cast<uint4*>(some);
      }
      data[c] = v;
      row.chunk(c, see);
    }
  }
#pragma unroll
  for (int step = 16; step > 0; step /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
  bad = __any_sync(0xffffffffu, bad);
  if (threadIdx.x == 0) s.bad = 0;
  __syncthreads();
  if (lane == 0) {
    s.warp_top[warp] = top;
    if (bad) s.bad = 1;
  }
  cluster_sync_all();  // (the boxes of all blocks of the cluster are there from here on)
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s.warp_top[w]);
    row.tell(&s.box.top[row.rank], top);
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
  const float temperature = args.temperature.of(number), top_p = args.top_p.of(number);
  const float least = args.min_p.of(number), u = args.uniform[number];
  const int top_k = args.top_k.of(number);
  int* token = args.tokens + number;
  if (any_bad || !(fabsf(top) < INFINITY)) {  // no distribution
    if (row.rank == 0 && threadIdx.x == 0) {
      *token = -1;
      if (args.logprobs != nullptr) args.logprobs[number] = NAN;
    }
    return;  // (behind a barrier that all blocks have passed; nobody reads a neighbour any more)
  }
  double log_sum = 0.0;
  if (args.logprobs != nullptr) {
    float sum = 0.0f;
    row.each([&](float x, int) { sum += exp2_approx((x - top) * kLog2e); });
    double all = sum;
#pragma unroll
    for (int step = 16; step > 0; step /= 2) all += __shfl_xor_sync(0xffffffffu, all, step);
    if (lane == 0) s.warp_sum[warp] = all;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kWarps; ++w) all += s.warp_sum[w];
      row.tell(&s.box.sum[row.rank], all);
    }
    row.sync();
    for (int r = 0; r < row.size; ++r) log_sum += s.box.sum[r];
    log_sum = log(log_sum);
  }
  auto answer = [&](int i) {
    *token = i;
    if (args.logprobs != nullptr) {
      const float x = static_cast<float>(static_cast<const T*>(args.logits)[args.stride * number + i]);
      args.logprobs[number] = static_cast<float>(static_cast<double>(x) - static_cast<double>(top) - log_sum);
    }
  };
  if (!(temperature > 0.0f)) {  // the first of the largest
    int first = INT_MAX;
    row.each([&](float x, int i) {
      if (x == top) first = min(first, i);
    });
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) s.warp_first[warp] = first;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kWarps; ++w) first = min(first, s.warp_first[w]);
      *cluster.map_shared_rank(&s.box.first[row.rank], 0) = first;
    }
    row.sync();
    if (row.rank == 0 && threadIdx.x == 0) {
      for (int r = 0; r < row.size; ++r) first = min(first, s.box.first[r]);
      answer(first);
    }
    return;
  }
  row.inverse = 1.0 / static_cast<double>(temperature);
  row.bin_scale = kBinsPerUnit / temperature;
  Border border{0, INT_MAX};
  u64 kept = 0;
  bool whole = true;
  if (top_k >= 1 && top_k < args.vocab) {
    border = row.search(true, static_cast<u64>(top_k), kept);
    whole = false;
  }
  if (top_p < 1.0f) {
    if (whole) {
      row.histogram([&](float x) { return row.bin_of(x); });
      row.level_one = true;
      for (int r = 0; r < row.size; ++r) kept += s.box.segment_weight[r];
    }
    const double part = ceil(static_cast<double>(top_p) * static_cast<double>(kept));
    border = row.search(false, part >= 1.0 ? static_cast<u64>(part) : 1, kept);
  }
  const double lowest = least > 0.0f ? fmin(static_cast<double>(least), 1.0) : 0.0;
  row.locate(
      [&](float x, int i) -> u64 {
        if (!(x > -INFINITY) || !border.keeps(key_of(x), i)) return 0;
        const double w = row.weight(x);
        return w >= lowest ? Row<T>::fixed(w) : 0;
      },
      [&](u64 total) {
        const double at = u > 0.0f ? static_cast<double>(u) * static_cast<double>(total) : 0.0;
        return at < static_cast<double>(total) ? min(static_cast<u64>(at), total - 1) : total - 1;
      },
      answer);
}

size_t shared_bytes(int slice, int size) { return (sizeof(Shared) + 15) / 16 * 16 + static_cast<size_t>(slice) * size + kVector; }

template <typename T>
cudaError_t launch(const SampleArgs& args, cudaStream_t stream) {
  // As few blocks to a row as hold it; more where rows are few, so that all SMs read.
  const int64_t bytes = static_cast<int64_t>(args.vocab) * sizeof(T);
  const int64_t limit = bytes > static_cast<int64_t>(kSliceBytes) * kMaxCluster ? kMostSliceBytes : kSliceBytes;
  int size = 1;
  while (size < kMaxCluster && (bytes > limit * size || (args.rows * size * 2 <= device_sms() && bytes > 8192 * size))) size *= 2;
  constexpr int kElements = kVector / sizeof(T);
  const int slice = ((args.vocab + size - 1) / size + kElements - 1) / kElements * kElements;
  const cudaError_t err = allow_shared_memory(sample_kernel<T>);
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
  return cudaLaunchKernelEx(&config, sample_kernel<T>, args, slice);
}

}  // namespace

bool sample_supported(int vocab, bool bf16) {
  return static_cast<int64_t>(vocab) * (bf16 ? 2 : 4) <= static_cast<int64_t>(kMostSliceBytes) * kMaxCluster;
}

cudaError_t launch_sample(const SampleArgs& args, bool bf16, cudaStream_t stream) {
  return bf16 ? launch<__nv_bfloat16>(args, stream) : launch<float>(args, stream);
}

}  // namespace nmoe
