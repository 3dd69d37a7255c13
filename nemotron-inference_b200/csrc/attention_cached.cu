// Attention of new rows over the paged 8-bit cache.
//
// For a row with query q at position x of its sequence, over the tokens j <= x whose keys and values are
// codes times powers of two (a power per page and head):
//   s_j = scale 2^(key power) q . kcode_j,   o = sum_j e^s_j 2^(value power) vcode_j / sum_j e^s_j
//
// What bounds it is reading the cache once.  So the codes go from memory to the tensor cores as they lie
// in their pages: what they are multiplied by is made 8-bit as well, as a sum of two E4M3 terms, a and
// b / 16.  A bf16 query's eight bits of significand fit the two terms exactly (scaled to its row's
// largest element; what lies 2^14 below that ends at 2^-21 of it), a weight e^(s - max) is rounded to
// within 2^-8 of itself.  With R query rows (new rows x heads that share the key head), tiles of 128
// tokens:
//   S^T = K [a | b]^T   M = 128 tokens, N = 2R, K = 128: four MMAs, both operands in shared memory
//   softmax             a thread per token: a row's scores lie in one column of TMEM
//   O^T += V^T [a | b]  M = 128 dimensions, N = 2R, K = 128 tokens: the values' tile is read along its
//                       rows, so nothing is transposed
// The powers of keys enter the scores and those of values the exponents of the weights, relative to a
// running maximum of both together: the largest weight is always near 2^8, however far powers lie
// apart.  The sums of the weights without the values' powers are kept in FP32 beside.
//
// A group of four warps runs a pipeline of its own, with its own S, weights and O: up to 32 rows against
// every tile (few rows: two blocks of one group to an SM), or, in blocks of four groups, up to 128 rows
// with all groups at one tile, 64 with two tiles at a time, 32 with four.  One tile's softmax is a chain of
// some 3500 cycles, in which the memory brings two and a half more: pipelines side by side hide it.
//
// Blocks share all tiles of all sequences evenly, whatever
// the sequences' lengths: block g of G takes the tiles [W g / G, W (g + 1) / G) of the W in order, a tile
// counting for what its rows cost.  Where
// a (sequence, key head) is cut, each piece leaves its sums in the workspace and the last to finish
// joins them, in order, so results do not depend on who that is.
#include <cuda_fp16.h>

#include <algorithm>

#include "attention.h"
#include "attention_mma.cuh"
#include "kernels.h"

namespace nmoe {
namespace {

constexpr int kTile = 128;  // tokens
constexpr int kTileBytes = kTile * kHeadDim;
constexpr int kMaxPagesPerTile = kTile / 16;
constexpr int kMaxRows = 128;
constexpr int kSoftmaxRegisters = 104, kOtherRegisters = 64;  // 4 * 104 + 64 = 5 * 96, as launched
constexpr int kSegments = 4;
constexpr int kSlotsPerBlock = 3;       // of the workspace: a piece that began before, one that goes on, one's own
constexpr float kWeightBits = 7.0f;    // a row's largest weight is 2^7 when its reference is set ...
constexpr float kLargestBits = 8.8f;   // ... and less than 2^8.8 < 448 before it is set anew

// R query rows; `Groups` times four warps that take R / Groups of them each.
template <int R, int Groups>
struct Shape {
  static constexpr int kRows = R, kGroups = Groups, kGroupRows = R / Groups;
  static constexpr int kWidth = 2 * kGroupRows;  // columns of a group's S and O, bytes of a token's weights
  static constexpr int kBlocks = Groups == 1 ? 2 : 1;  // on an SM
  static constexpr int kScores = Groups == 1 ? 2 : 1;  // buffers of a group's S
  // Tiles in flight; values are held from the tile's softmax on, of as many tiles as there are pipelines.
  static constexpr int kKeySlots = 3, kValueSlots = Groups == 1 ? 3 : 6;
  static constexpr int kSoftmaxWarps = 4 * Groups;
  static constexpr int kRowsPerWarp = R / kSoftmaxWarps;  // of queries
  // Four groups and two warps more have 96 registers a thread; the groups take 8 from four others.
  static constexpr bool kSplitRegisters = Groups > 1;
  static constexpr int kThreads = 32 * (kSoftmaxWarps + (kSplitRegisters ? 4 : 2));
  static constexpr int kColumnsUsed = (kScores + 1) * Groups * kWidth;
  static constexpr int kColumns = kColumnsUsed <= 64 ? 64 : kColumnsUsed <= 128 ? 128 : 512;
  static constexpr uint32_t kQueryBytes = 2 * R * kHeadDim, kWeightBytes = 2 * R * kTile;
};

// Groups that work on one tile together when `groups` of them have rows (three leave the fourth idle).
template <typename S>
__host__ __device__ constexpr int groups_per_tile(int groups) {
  return S::kGroups == 1 || groups == 1 ? 1 : groups == 2 ? 2 : S::kGroups;
}
// What a tile counts for when blocks share them: with all four groups at it, twice as much as with one.
template <typename S>
__host__ __device__ constexpr int tile_cost(int groups) {
  return S::kGroups == 1 ? 1 : groups <= 2 ? 1 : 2;
}

// The tiles of one (sequence, key head, rows) that a block works on.
struct Segment {
  int first, rows, length;  // of the batch entry
  int kv_head, row0;        // first of the query rows
  int groups, step;         // groups of rows that there are; groups to a tile: group g has the rows of g % step
  int tile, tiles;          // group g takes every (groups / step)th, from g / step on
  int part;                 // -1: no other block has any; else the slot of the workspace for its sums
  int lead, parts;          // the first block with a part, and how many have one
};

template <typename S>
struct Control {
  uint64_t k_full[S::kKeySlots], k_empty[S::kKeySlots], v_full[S::kValueSlots], v_empty[S::kValueSlots];
  uint64_t s_full[S::kGroups][S::kScores], s_empty[S::kGroups][S::kScores];
  uint64_t p_full[S::kGroups], p_empty[S::kGroups], q_full, drained;
  uint64_t segment_full[kSegments], segment_empty[kSegments];
  Segment segment[kSegments];  // a place is given back when the segment is done
  int has_segment[kSegments];
  Segment to_join[2];          // the (at most two) that other blocks have pieces of
  int powers[S::kValueSlots][2][kMaxPagesPerTile];  // of a tile's pages, keys and values
  // by row
  alignas(16) float factor[S::kRows];  // what a row's product of codes is multiplied by
  int out_row[S::kRows];               // of the result, -1: none
  int limit[S::kRows];                 // a row's position: the last token it sees
  // by group and row
  alignas(16) float shift[S::kRows];                 // kWeightBits - the reference
  alignas(16) float rise[S::kRows], fade[S::kRows];  // of a reference, and what that leaves of its sums
  int highest[S::kRows];                             // largest exponents of a tile, as ordered()
  uint32_t risen[S::kGroups];                        // the rows whose references have changed
  float warp_sum[S::kSoftmaxWarps][S::kGroupRows];
  float sum[S::kRows], inverse[S::kRows];
  int first_bad[kHeadDim];  // position of the first masked value that is no number
  int failed[S::kGroups];
  int joined;
  uint32_t tmem;
  int64_t before[S::kThreads / 32];
  int most[S::kThreads / 32];
  int64_t total, found_before;  // cost of all tiles, and of those of the entries before:
  BatchEntry entry;             // the entry in which this block's tiles begin
  int found, blocks;            // which it is; blocks that have any tiles
};

template <typename S>
constexpr size_t shared_bytes() {
  return 1024 + (S::kKeySlots + S::kValueSlots) * kTileBytes + S::kQueryBytes + S::kWeightBytes + sizeof(Control<S>);
}

// All blocks of a launch run at once.
template <typename S>
constexpr bool fits_on_sm() {
  return S::kBlocks * (shared_bytes<S>() + 1024) <= 228 * 1024 && S::kBlocks * S::kColumns <= 512;
}

// What a block leaves for the join: by group and row 128 sums, then the references and the sums of weights.
__host__ __device__ constexpr size_t slot_floats(int rows) { return static_cast<size_t>(rows) * (kHeadDim + 2); }

struct Split {
  int* counters;  // by the block in which a (sequence, key head) begins: pieces that are done, twice
  float* slots;
};

// Instruction descriptor of kind::f8f6f4 on E4M3 operands, FP32 sums, M = 128.
__host__ __device__ constexpr uint32_t make_idesc_e4m3(uint32_t n, bool along_rows) {
  return (1u << 4) | (along_rows ? 3u << 15 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

// (no calls where registers are handed over between warps: see wait_warp())
template <typename S>
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
  if constexpr (S::kSplitRegisters) return wait_warp(bar, parity);
  return mbar_wait_warp(bar, parity);
}

// Floats as integers of the same order (no NaN), and back.
__device__ __forceinline__ int ordered(float x) {
  const int bits = __float_as_int(x);
  return bits ^ ((bits >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
constexpr int kLowest = static_cast<int>(0x807fffffu);  // of -infinity

// The largest over the warp, in all lanes.
__device__ __forceinline__ float warp_max(float x) {
  return from_ordered(__reduce_max_sync(0xffffffffu, ordered(x)));
}

__device__ __forceinline__ void group_sync(int group) {
  asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
}
__device__ __forceinline__ bool group_any(int group, bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "bar.red.or.pred q, %1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(group + 1), "r"(static_cast<uint32_t>(mine))
      : "memory");
  return any != 0;
}
template <typename S>
__device__ __forceinline__ void softmax_sync() {
  asm volatile("bar.sync 5, %0;" ::"n"(S::kSoftmaxWarps * 32) : "memory");
}

// Sums N values over the warp: lane L holds in v[0..] the totals of the rows sum_row<N>(L, 0..).  Half of
// the values change hands in each step.
template <int N>
__device__ __forceinline__ void warp_sums(float (&v)[N], int lane) {
  int count = N;
#pragma unroll
  for (int stride = 16; stride > 0; stride /= 2) {
    if (count > 1) {
      count /= 2;
      const bool upper = (lane & stride) != 0;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < count) {
          const float send = upper ? v[i] : v[i + count], keep = upper ? v[i + count] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, stride);
        }
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], stride);
    }
  }
}
template <int N>
__device__ __forceinline__ int sum_row(int lane, int i) {
  int row = 0, count = N;
#pragma unroll
  for (int stride = 16; stride > 0; stride /= 2) {
    if (count > 1) {
      count /= 2;
      if (lane & stride) row += count;
    }
  }
  return row + i;
}

// Two E4M3 codes, `lo` in the low byte, of two binary16 values, and back.
__device__ __forceinline__ uint32_t codes_of(__half2 x) {
  uint16_t codes;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(codes) : "r"(*reinterpret_cast<const uint32_t*>(&x)));
  return codes;
}
__device__ __forceinline__ __half2 halves_of(uint32_t codes) {
  uint32_t two;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"(static_cast<uint16_t>(codes)));
  return *reinterpret_cast<const __half2*>(&two);
}
// Two values as two terms each, a + b / 16.
__device__ __forceinline__ void two_terms(float x, float y, uint32_t& a, uint32_t& b) {
  const __half2 v = __floats2half2_rn(x, y);
  a = codes_of(v);
  b = codes_of(__hmul2(__hsub2(v, halves_of(a)), __float2half2_rn(16.0f)));
}

// How a batch entry's tiles lie in the order of all: by key head, then by rows, kRows at a time.
template <typename S>
struct EntryTiles {
  int tiles, row_tiles, last_groups;  // of tokens; of rows, and the groups of the last of them
  int64_t head_cost;

  __device__ EntryTiles(const CachedArgs& args, const BatchEntry& e) {
    const int rows = e.rows * (args.heads / args.cache.kv_heads);
    tiles = (e.length + kTile - 1) / kTile;
    row_tiles = (rows + S::kRows - 1) / S::kRows;
    last_groups = (rows - (row_tiles - 1) * S::kRows + S::kGroupRows - 1) / S::kGroupRows;
    head_cost = static_cast<int64_t>(tiles) *
                ((row_tiles - 1) * tile_cost<S>(S::kGroups) + (row_tiles > 0 ? tile_cost<S>(last_groups) : tile_cost<S>(S::kGroups)));
    if (row_tiles == 0) head_cost = 0;
  }
};

// All threads: the cost of all tiles, and the entry in which this block's begin.
template <typename S>
__device__ void find_begin(const CachedArgs& args, Control<S>* c) {
  const int n = args.batch.count, each = (n + S::kThreads - 1) / S::kThreads, heads = args.cache.kv_heads;
  const int begin = min(n, static_cast<int>(threadIdx.x) * each), end = min(n, begin + each);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t mine = 0;
  int most = 1;  // of a tile
  BatchEntry e;
#pragma unroll 1
  for (int i = begin; i < end; ++i) {
    e = batch_entry(args.cache, args.batch, i);
    if (!e.valid && blockIdx.x == 0) report_cache_error(args.cache.error, kCacheBadSequence);
    const EntryTiles<S> tiles(args, e);
    mine += heads * tiles.head_cost;
    if (tiles.row_tiles > 0) most = max(most, tile_cost<S>(tiles.row_tiles > 1 ? S::kGroups : tiles.last_groups));
  }
  int64_t upto = mine;
#pragma unroll
  for (int step = 1; step < 32; step *= 2) {
    const int64_t other = __shfl_up_sync(0xffffffffu, upto, step);
    if (lane >= step) upto += other;
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 31) {
    c->before[warp] = upto;
    c->most[warp] = most;
  }
  __syncthreads();
  int64_t total = 0, below = upto - mine;
#pragma unroll 1
  for (int w = 0; w < S::kThreads / 32; ++w) {
    if (w < warp) below += c->before[w];
    total += c->before[w];
    most = max(most, c->most[w]);
  }
  // Every block's share is at least one tile, so that between a (sequence, key head)'s first block and its
  // last each has some of it.
  const int blocks = total == 0 ? 0 : static_cast<int>(max(min(total / most, static_cast<int64_t>(gridDim.x)), static_cast<int64_t>(1)));
  if (threadIdx.x == 0) {
    c->total = total;
    c->blocks = blocks;
  }
  if (static_cast<int>(blockIdx.x) >= blocks) return;
  const int64_t start = total * blockIdx.x / blocks;
  if (start >= below && start < below + mine) {  // one thread's
#pragma unroll 1
    for (int i = begin; i < end; ++i) {
      if (each > 1) e = batch_entry(args.cache, args.batch, i);
      const int64_t cost = heads * EntryTiles<S>(args, e).head_cost;
      if (start < below + cost) {
        c->found = i;
        c->found_before = below;
        c->entry = e;
        break;
      }
      below += cost;
    }
  }
}

// The block in whose share place `at` of `total` lies, of `blocks` with [total g / blocks, total (g + 1) / blocks).
__device__ __forceinline__ int block_of(int64_t at, int64_t total, int blocks) {
  const uint64_t x = static_cast<uint64_t>(at + 1) * blocks - 1;
  if ((x | static_cast<uint64_t>(total)) >> 32) return static_cast<int>(x / static_cast<uint64_t>(total));
  return static_cast<int>(static_cast<uint32_t>(x) / static_cast<uint32_t>(total));
}

// The warp that brings keys and values in, a page at a time.
template <typename S>
__device__ void load_role(const CachedArgs& args, const CUtensorMap* map, uint32_t keys_at, uint32_t values_at, Control<S>* c) {
  const PagedCache& cache = args.cache;
  const int lane = threadIdx.x & 31, blocks = c->blocks, g = blockIdx.x;
  const int64_t total = c->total;
  const int64_t begin = g < blocks ? total * g / blocks : 0, stop = g < blocks ? total * (g + 1) / blocks : 0;
  const int pages_per_tile = kTile >> cache.page_shift;
  const uint32_t page_bytes = kHeadDim << cache.page_shift;
  uint32_t no = 0, segments = 0;  // tiles, segments so far
  int i = c->found;
  int64_t entry_at = c->found_before;
  BatchEntry e = c->entry;
  bool ok = true;
#pragma unroll 1
  while (entry_at < stop && ok) {
    const EntryTiles<S> t(args, e);
    const int units = cache.kv_heads * t.row_tiles;
    // the first unit that reaches into this block's share
    const int64_t skip = max(begin - entry_at, static_cast<int64_t>(0));
    int head = 0, row_tile = 0;
    int64_t unit_at = entry_at;
    if (skip > 0) {
      head = static_cast<int>(skip / t.head_cost);
      unit_at += head * t.head_cost;
      const int full = t.tiles * tile_cost<S>(S::kGroups);
      row_tile = min(static_cast<int>((begin - unit_at) / full), t.row_tiles - 1);
      unit_at += static_cast<int64_t>(row_tile) * full;
    }
    const int last_page = pages_of(cache, e.length);
#pragma unroll 1
    for (int unit = head * t.row_tiles + row_tile; unit < units && unit_at < stop && ok; ++unit) {
      const int groups = row_tile == t.row_tiles - 1 ? t.last_groups : S::kGroups, cost = tile_cost<S>(groups);
      Segment s;
      s.first = e.first;
      s.rows = e.rows;
      s.length = e.length;
      s.kv_head = head;
      s.row0 = row_tile * S::kRows;
      s.groups = groups;
      s.step = groups_per_tile<S>(groups);
      s.tile = begin > unit_at ? static_cast<int>((begin - unit_at + cost - 1) / cost) : 0;
      s.tiles = static_cast<int>(min((stop - unit_at + cost - 1) / cost, static_cast<int64_t>(t.tiles))) - s.tile;
      s.lead = block_of(unit_at, total, blocks);
      s.parts = block_of(unit_at + static_cast<int64_t>(t.tiles - 1) * cost, total, blocks) - s.lead + 1;
      s.part = s.parts == 1 ? -1 : kSlotsPerBlock * g + (g == s.lead);
      unit_at += static_cast<int64_t>(t.tiles) * cost;
      if (++row_tile == t.row_tiles) {
        row_tile = 0;
        ++head;
      }
      if (s.tiles <= 0) continue;
      const uint32_t place = segments % kSegments;
      if (!(ok = wait<S>(smem_u32(&c->segment_empty[place]), ((segments / kSegments) & 1) ^ 1))) break;
      if (lane == 0) {
        c->segment[place] = s;
        c->has_segment[place] = 1;
        mbar_arrive(&c->segment_full[place]);
      }
      __syncwarp();
      ++segments;
      int first_page = -1, page = 0, k_power = 0, v_power = 0;  // a lane per page, 32 at a time
#pragma unroll 1
      for (int tile = s.tile; tile < s.tile + s.tiles; ++tile, ++no) {
        const int wanted = tile * pages_per_tile;
        const bool new_pages = first_page < 0 || wanted >= first_page + 32;
        if (new_pages) {
          first_page = wanted;
          if (wanted + lane < last_page) {
            page = page_at(cache, e.sequence, wanted + lane);
            if (page < 0) {
              report_cache_error(cache.error, kCacheBadSequence);
              page = 0;
            }
          }
        }
        const int count = min(pages_per_tile, last_page - wanted), from = wanted - first_page;
        const uint32_t k_slot = no % S::kKeySlots, v_slot = no % S::kValueSlots;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          const uint32_t empty = smem_u32(half ? &c->v_empty[v_slot] : &c->k_empty[k_slot]);
          const uint32_t round = half ? no / S::kValueSlots : no / S::kKeySlots;
          if (!(ok = wait<S>(empty, (round & 1) ^ 1))) break;
          const uint32_t bar = smem_u32(half ? &c->v_full[v_slot] : &c->k_full[k_slot]);
          const uint32_t to = half ? values_at + v_slot * kTileBytes : keys_at + k_slot * kTileBytes;
#pragma unroll 1
          for (int j = 0; j < count; ++j) {
            const int id = __shfl_sync(0xffffffffu, page, from + j);
            const int row = static_cast<int>(block_of_page(cache, args.layer, id, half, s.kv_head) << cache.page_shift);
            if (elect_one()) tma_load_2d_at(to + j * page_bytes, map, 0, row, bar);
            __syncwarp();
          }
          if (half) {  // the values are there once the tile's powers are as well
            if (new_pages && wanted + lane < last_page) {
              k_power = cache.exponents[block_of_page(cache, args.layer, page, 0, s.kv_head)];
              v_power = cache.exponents[block_of_page(cache, args.layer, page, 1, s.kv_head)];
            }
            const int p = __shfl_sync(0xffffffffu, k_power, (from + lane) & 31);
            const int z = __shfl_sync(0xffffffffu, v_power, (from + lane) & 31);
            if (lane < count) {
              c->powers[v_slot][0][lane] = p;
              c->powers[v_slot][1][lane] = z;
            }
            __syncwarp();
          }
          if (elect_one()) mbar_arrive_expect_tx_at(bar, count * page_bytes);
          __syncwarp();
        }
        if (!ok) break;
      }
    }
    entry_at += cache.kv_heads * t.head_cost;
    if (entry_at < stop && ok) e = batch_entry(cache, args.batch, ++i);
  }
  if (ok) {
    const uint32_t place = segments % kSegments;
    ok = wait<S>(smem_u32(&c->segment_empty[place]), ((segments / kSegments) & 1) ^ 1);
    if (ok && lane == 0) {
      c->has_segment[place] = 0;
      mbar_arrive(&c->segment_full[place]);
    }
  }
  if (ok) return;
  if (lane == 0) report_cache_error(cache.error, kDevWaitTimeout);
  // what is in flight arrives before the block's shared memory is given up
#pragma unroll 1
  for (uint32_t back = 0; back < S::kValueSlots; ++back) {
    const uint32_t tile = no - back;
    if (back > no) break;
    wait<S>(smem_u32(&c->k_full[tile % S::kKeySlots]), (tile / S::kKeySlots) & 1);
    wait<S>(smem_u32(&c->v_full[tile % S::kValueSlots]), (tile / S::kValueSlots) & 1);
  }
}

// Small counters, one per group, in one word.
__device__ __forceinline__ uint32_t count_of(uint32_t counters, int g) { return (counters >> (8 * g)) & 0xffu; }
__device__ __forceinline__ uint32_t counted(uint32_t counters, int g) {
  return (counters & ~(0xffu << (8 * g))) | (((count_of(counters, g) + 1) & 0xffu) << (8 * g));
}

template <typename S>
__device__ bool mma_role(uint32_t keys_at, uint32_t values_at, uint32_t q_at, uint32_t weights_at, uint32_t tmem, Control<S>* c) {
  constexpr uint32_t kScoresDesc = make_idesc_e4m3(S::kWidth, false), kValuesDesc = make_idesc_e4m3(S::kWidth, true);
  // a token's weights are 16, 32 or 64 bytes, swizzled in as many
  constexpr uint32_t kSwizzle = S::kWidth == 64 ? 4 : S::kWidth == 32 ? 6 : 0;
  const uint32_t o = tmem + S::kGroups * S::kScores * S::kWidth;
  uint32_t first_no = 0;  // of the segment's tiles among all
  uint32_t s_uses = 0, p_uses = 0;
#pragma unroll 1
  for (uint32_t segments = 0;; ++segments) {
    const uint32_t place = segments % kSegments;
    if (!wait<S>(smem_u32(&c->segment_full[place]), (segments / kSegments) & 1)) return false;
    const int some = c->has_segment[place];
    const int tiles = warp_uniform(c->segment[place].tiles), groups = warp_uniform(c->segment[place].groups);
    const int step = warp_uniform(c->segment[place].step), streams = S::kGroups / step;
    __syncwarp();
    if (!some) return true;
    if (elect_one()) mbar_arrive(&c->segment_empty[place]);
    __syncwarp();
    if (!wait<S>(smem_u32(&c->q_full), segments & 1)) return false;
    tcgen05_fence_after();
    // scores are ahead of the values by a tile for each pipeline
#pragma unroll 1
    for (int j = 0; j < tiles + streams; ++j) {
      if (j < tiles) {
        const uint32_t no = first_no + j, slot = no % S::kKeySlots;
        if (!wait<S>(smem_u32(&c->k_full[slot]), (no / S::kKeySlots) & 1)) return false;
        const uint64_t k_desc = make_smem_desc(keys_at + slot * kTileBytes, 16, 1024, 2);
#pragma unroll 1
        for (int rows = 0; rows < groups; ++rows) {
          const int g = j % streams * step + rows;
          const uint32_t use = count_of(s_uses, g), buffer = use % S::kScores;
          s_uses = counted(s_uses, g);
          if (!wait<S>(smem_u32(&c->s_empty[g][buffer]), ((use / S::kScores) & 1) ^ 1)) return false;
          tcgen05_fence_after();
          if (elect_one()) {
            const uint64_t q_desc = make_smem_desc(q_at + rows * S::kWidth * kHeadDim, 16, 1024, 2);
            const uint32_t d = tmem + (g * S::kScores + buffer) * S::kWidth;
#pragma unroll
            for (int k = 0; k < kHeadDim / 32; ++k) {
              mma_e4m3(d, advance_smem_desc(k_desc, k * 32), advance_smem_desc(q_desc, k * 32), kScoresDesc, k > 0);
            }
            tcgen05_commit(&c->s_full[g][buffer]);
            if (rows == groups - 1) tcgen05_commit(&c->k_empty[slot]);
          }
          __syncwarp();
        }
      }
      if (j >= streams) {
        const int tile = j - streams;
        const uint32_t no = first_no + tile, slot = no % S::kValueSlots;
        if (!wait<S>(smem_u32(&c->v_full[slot]), (no / S::kValueSlots) & 1)) return false;
        // (eight tokens are 1024 bytes of values)
        const uint64_t v_desc = make_smem_desc(values_at + slot * kTileBytes, 16, 1024, 2);
#pragma unroll 1
        for (int rows = 0; rows < groups; ++rows) {
          const int g = tile % streams * step + rows;
          if (!wait<S>(smem_u32(&c->p_full[g]), count_of(p_uses, g) & 1)) return false;
          p_uses = counted(p_uses, g);
          tcgen05_fence_after();
          if (elect_one()) {
            const uint32_t at = weights_at + g * kTile * S::kWidth;
            const uint64_t p_desc = S::kWidth == 16 ? make_smem_desc(at, 128, 128, 0) : make_smem_desc(at, 16, 8 * S::kWidth, kSwizzle);
#pragma unroll
            for (int k = 0; k < kTile / 32; ++k) {
              mma_e4m3(o + g * S::kWidth, advance_smem_desc(v_desc, k * 4096), advance_smem_desc(p_desc, k * 32 * S::kWidth),
                       kValuesDesc, tile >= streams || k > 0);
            }
            tcgen05_commit(&c->p_empty[g]);
            if (rows == groups - 1) tcgen05_commit(&c->v_empty[slot]);
          }
          __syncwarp();
        }
      }
    }
    first_no += tiles;
  }
}

// Eight columns of this warp's 32 lanes, without the wait.
__device__ __forceinline__ void tmem_ld_x8_async(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

__device__ __forceinline__ float power_of_two(int e) {  // -126 <= e <= 127
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// The queries of a segment, a warp per row: read ...
template <typename S>
__device__ __forceinline__ void load_queries(const CachedArgs& args, const Segment& s, uint2 (&raw)[S::kRowsPerWarp]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = args.heads / args.cache.kv_heads;
#pragma unroll
  for (int k = 0; k < S::kRowsPerWarp; ++k) {
    const int row = s.row0 + k * S::kSoftmaxWarps + warp, token = row / group;
    raw[k] = make_uint2(0, 0);
    if (token < s.rows) {
      raw[k] = *reinterpret_cast<const uint2*>(args.q + static_cast<int64_t>(s.first + token) * args.q_stride +
                                               (s.kv_head * group + row % group) * kHeadDim + lane * 4);
    }
  }
}

// ... and put into shared memory as two terms, each row scaled by a power of two: the first terms of a
// group's rows, then the second terms.
template <typename S>
__device__ __forceinline__ void store_queries(const CachedArgs& args, const Segment& s,
                                              const uint2 (&raw)[S::kRowsPerWarp], uint8_t* q, Control<S>* c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = args.heads / args.cache.kv_heads;
#pragma unroll
  for (int k = 0; k < S::kRowsPerWarp; ++k) {
    const int r = k * S::kSoftmaxWarps + warp;
    if (r >= s.groups * S::kGroupRows) break;
    float x[4];
    x[0] = __uint_as_float(raw[k].x << 16);
    x[1] = __uint_as_float(raw[k].x & 0xffff0000u);
    x[2] = __uint_as_float(raw[k].y << 16);
    x[3] = __uint_as_float(raw[k].y & 0xffff0000u);
    // (magnitudes as whole numbers: what is no number is beyond them all)
    const uint32_t m = max(max(raw[k].x & 0x7fffu, (raw[k].x >> 16) & 0x7fffu),
                           max(raw[k].y & 0x7fffu, (raw[k].y >> 16) & 0x7fffu));
    const int largest = static_cast<int>(__reduce_max_sync(0xffffffffu, m));
    // the largest element's exponent becomes 7: below 256
    const int power = max(largest >> 7, 1) - 134;
    const int some = max(power, -100), rest = power - some;  // (2^-power may be beyond FP32)
    const float down = power_of_two(-some), downer = power_of_two(-rest);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = x[i] * down * downer;
    uint32_t a[2], b[2];
    two_terms(x[0], x[1], a[0], b[0]);
    two_terms(x[2], x[3], a[1], b[1]);
    const int chunk = lane >> 2, inside = (lane & 3) * 4;
    const int r1 = r / S::kGroupRows * S::kWidth + r % S::kGroupRows, r2 = r1 + S::kGroupRows;
    *reinterpret_cast<uint32_t*>(q + r1 * 128 + ((chunk ^ (r1 & 7)) << 4) + inside) = a[0] | (a[1] << 16);
    *reinterpret_cast<uint32_t*>(q + r2 * 128 + ((chunk ^ (r2 & 7)) << 4) + inside) = b[0] | (b[1] << 16);
    if (lane == 0) {
      // (a row that is no number: its scores are none)
      c->factor[r] = largest < 0x7f80 ? args.scale * kLog2e * power_of_two(some) * power_of_two(rest) : NAN;
      const int token = (s.row0 + r) / group;
      const bool valid = token < s.rows;
      c->limit[r] = s.length - s.rows + (valid ? token : 0);
      c->out_row[r] = valid ? (s.first + token) * args.heads + s.kv_head * group + (s.row0 + r) % group : -1;
    }
  }
  if (threadIdx.x < S::kRows) {
    c->shift[threadIdx.x] = 0.0f;
    c->highest[threadIdx.x] = kLowest;
  }
}

// The values of a tile at the end of a sequence: places behind it hold anything and become 0; where a
// value that only some rows see is no number, it becomes 0 as well, and the rows that see it get it in
// the end (a weight of 0 times such a value would be none either).  A thread per token.
template <typename S>
__device__ __forceinline__ void clean_values(uint8_t* values, int token, int position, const Segment& s, Control<S>* c) {
  uint4* row = reinterpret_cast<uint4*>(values + token * kHeadDim);
  if (position >= s.length) {
#pragma unroll
    for (int i = 0; i < 8; ++i) row[i] = make_uint4(0, 0, 0, 0);
  } else if (position > s.length - s.rows) {
    uint32_t* words = reinterpret_cast<uint32_t*>(row);
#pragma unroll 1
    for (int i = 0; i < kHeadDim / 4; ++i) {
      const uint32_t x = words[i];
      if ((((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) == 0) continue;
#pragma unroll 1
      for (int k = 0; k < 4; ++k) {
        if (((x >> (8 * k)) & 0x7fu) != 0x7fu) continue;
        atomicMin(&c->first_bad[(((i >> 2) ^ (token & 7)) << 4) + 4 * (i & 3) + k], position);
        reinterpret_cast<uint8_t*>(words + i)[k] = 0;
      }
    }
  }
  fence_proxy_async_smem();
}

// Where byte `column` (a multiple of 8) of a token's weights lies in its group's.
template <typename S>
__device__ __forceinline__ uint32_t weight_offset(int token, int column) {
  const uint32_t at = token * S::kWidth + column;
  constexpr uint32_t mask = (S::kWidth / 16 - 1) << 4;
  return at ^ ((at >> 3) & mask);
}

// Joins the pieces of a (sequence, key head): `parts` slots, a group of rows for each stream in each; this
// block takes share `piece` of the rows, a warp per row.
template <typename S>
__device__ void join(const CachedArgs& args, const Split& split, const Segment& s, int parts, int piece, Control<S>* c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = args.heads / args.cache.kv_heads, streams = S::kGroups / s.step, pieces = parts * streams;
  const int rows = min(S::kRows, s.rows * group - s.row0);
  // the sums of row 0 in piece p
  auto sums_of = [&](int p) {
    const int part = p / streams;
    const int slot = parts == 1 ? kSlotsPerBlock * static_cast<int>(blockIdx.x) + 2
                                : kSlotsPerBlock * (s.lead + part) + (part == 0);
    return split.slots + slot_floats(S::kRows) * slot;
  };
  auto row_of = [&](int p) { return p % streams * s.step * S::kGroupRows; };
  const int end = rows * (piece + 1) / parts;
#pragma unroll 1
  for (int r = rows * piece / parts + warp; r < end; r += S::kSoftmaxWarps) {
    // references and sums of weights, a lane per piece; the maximum so far is raised where there are over 32
    float top = -INFINITY, sum = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int start = 0; start < pieces; start += 32) {
      const int count = min(32, pieces - start);
      float reference = -INFINITY, weight = 0.0f;
      if (lane < count) {
        const float* at = sums_of(start + lane) + S::kRows * kHeadDim + row_of(start + lane) + r;
        reference = __ldcg(at);
        weight = __ldcg(at + S::kRows);
      }
      float scale = 0.0f;
#pragma unroll 1
      for (int first = 0; first < count; first += 8) {
        float4 x[8];  // (what is behind the last is read again, with no weight)
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const int of = min(start + first + p, pieces - 1);
          x[p] = __ldcg(reinterpret_cast<const float4*>(sums_of(of) + (row_of(of) + r) * kHeadDim) + lane);
        }
        if (first == 0) {
          const float higher = fmaxf(top, warp_max(reference));
          const float keep = top > -INFINITY ? exp2_approx(top - higher) : 0.0f;
          top = higher;
          sum *= keep;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] *= keep;
          if (reference > -INFINITY) scale = exp2_approx(reference - top);
          weight = scale != 0.0f ? weight * scale : 0.0f;
        }
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const float f = __shfl_sync(0xffffffffu, scale, first + p);
          if (first + p >= count || f == 0.0f) continue;
          sum += __shfl_sync(0xffffffffu, weight, first + p);
          o[0] = fmaf(x[p].x, f, o[0]);
          o[1] = fmaf(x[p].y, f, o[1]);
          o[2] = fmaf(x[p].z, f, o[2]);
          o[3] = fmaf(x[p].w, f, o[3]);
        }
      }
    }
    const float inverse = 1.0f / sum;
    const int row = s.row0 + r;
    const size_t at = static_cast<size_t>(s.first + row / group) * args.heads + s.kv_head * group + row % group;
    *reinterpret_cast<uint2*>(args.out + at * kHeadDim + lane * 4) =
        make_uint2(pack_bf16(o[0] * inverse, o[1] * inverse), pack_bf16(o[2] * inverse, o[3] * inverse));
  }
}

// Waits until every piece of a segment's (sequence, key head) has left its sums, then joins.  All blocks
// with tiles run at once (as many as the SMs hold, and none waits before its own tiles are done).  The
// counter is 0 again when the last of them has joined.
template <typename S>
__device__ bool wait_and_join(const CachedArgs& args, const Split& split, const Segment& s, Control<S>* c) {
  if (threadIdx.x == 0) {
    volatile int* done = split.counters + s.lead;
    const long long start = clock64();
    bool there = *done >= s.parts;
    while (!there && clock64() - start < (1ll << 31)) there = *done >= s.parts;
    __threadfence();
    c->joined = there;
  }
  softmax_sync<S>();
  if (!c->joined) return false;
  join<S>(args, split, s, s.parts, static_cast<int>(blockIdx.x) - s.lead, c);
  softmax_sync<S>();
  if (threadIdx.x == 0 && atomicAdd(&split.counters[s.lead], 1) == 2 * s.parts - 1) split.counters[s.lead] = 0;
  return true;
}

template <typename S>
__device__ bool softmax_role(const CachedArgs& args, const Split& split, uint8_t* values, uint8_t* q, uint8_t* all_weights,
                             uint32_t tmem, Control<S>* c) {
  constexpr int RG = S::kGroupRows, RH = RG < 16 ? RG : 16;  // rows of a group; of those, at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = warp >> 2;
  const int token = threadIdx.x & (kTile - 1), r0 = group * RG;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
  const uint32_t s_at = lanes + group * S::kScores * S::kWidth;
  const uint32_t o_at = lanes + (S::kGroups * S::kScores + group) * S::kWidth;
  uint8_t* weights = all_weights + group * kTile * S::kWidth;
  const int page_shift = args.cache.page_shift;
  const uint64_t* shifts = reinterpret_cast<const uint64_t*>(c->shift + r0);
  const uint64_t* rises = reinterpret_cast<const uint64_t*>(c->rise + r0);
  const uint64_t* fades = reinterpret_cast<const uint64_t*>(c->fade + r0);
  volatile int* failed = &c->failed[group];
  int joins = 0;
  uint32_t first_no = 0, uses = 0;  // tiles of the segments before; this group's own
  bool ok = wait<S>(smem_u32(&c->segment_full[0]), 0);
  int some = ok && c->has_segment[0];
  uint2 queries[S::kRowsPerWarp];
  if (some) load_queries<S>(args, c->segment[0], queries);
#pragma unroll 1
  for (uint32_t segments = 0;; ++segments) {
    const Segment& s = c->segment[segments % kSegments];
    if (!ok) *failed = 1;
    softmax_sync<S>();
#pragma unroll
    for (int i = 0; i < S::kGroups; ++i) ok = ok && c->failed[i] == 0;
    if (!ok) return false;
    if (!some) break;
    if (threadIdx.x < kHeadDim) c->first_bad[threadIdx.x] = INT32_MAX;
    store_queries<S>(args, s, queries, q, c);
    fence_proxy_async_smem();
    softmax_sync<S>();
    if (lane == 0) mbar_arrive(&c->q_full);
    const int streams = S::kGroups / s.step, stream = group / s.step, my_rows = group % s.step;
    const bool has_rows = my_rows < s.groups;
    const uint64_t* factors = reinterpret_cast<const uint64_t*>(c->factor + my_rows * RG);
    const int* limits = c->limit + my_rows * RG;
    uint64_t sum[RG / 2];
#pragma unroll
    for (int r = 0; r < RG / 2; ++r) sum[r] = 0;
    const int clear = s.length - s.rows;  // the last token that every row sees
#pragma unroll 1
    for (int j = has_rows ? stream : s.tiles; j < s.tiles; j += streams, ++uses) {
      const uint32_t no = first_no + j, slot = no % S::kValueSlots, buffer = uses % S::kScores;
      const int first = (s.tile + j) * kTile, position = first + token;
      const bool at_end = first + kTile - 1 > clear, is_first = j == stream;
      ok = wait<S>(smem_u32(&c->v_full[slot]), (no / S::kValueSlots) & 1);
      ok = wait<S>(smem_u32(&c->s_full[group][buffer]), (uses / S::kScores) & 1) && ok;
      tcgen05_fence_after();
      // (places behind the sequence may lie in pages that it does not have)
      const int page = token >> page_shift;
      const float k_scale = exp2_approx(static_cast<float>(position < s.length ? c->powers[slot][0][page] : 0));
      const float v_power = static_cast<float>(position < s.length ? c->powers[slot][1][page] : 0);
      const uint64_t k2 = pack2(k_scale, k_scale), k2_16 = pack2(k_scale * 0.0625f, k_scale * 0.0625f);
      const uint64_t v2 = pack2(v_power, v_power);
      const float v_inverse = exp2_approx(-v_power);
      const uint64_t v2_inverse = pack2(v_inverse, v_inverse);
      // (its weights are the first that the tensor cores multiply with this tile's values)
      if (at_end && my_rows == 0) clean_values<S>(values + slot * kTileBytes, token, position, s, c);
      bool stop = false;
#pragma unroll
      for (int h = 0; h < RG; h += RH) {
        // exponents of the weights, rows in pairs: score + power of the values - reference + kWeightBits
        uint64_t y[RH / 2];
        float high = -INFINITY;
        {
          uint32_t a[RH], b[RH];
#pragma unroll
          for (int i = 0; i < RH; i += 8) {
            tmem_ld_x8_async(s_at + buffer * S::kWidth + h + i, a + i);
            tmem_ld_x8_async(s_at + buffer * S::kWidth + RG + h + i, b + i);
          }
          tmem_ld_wait();
          registers_loaded<RH>(a);
          registers_loaded<RH>(b);
#pragma unroll
          for (int i = 0; i < RH / 2; ++i) {
            const uint64_t product =
                fma2(pack2(__uint_as_float(b[2 * i]), __uint_as_float(b[2 * i + 1])), k2_16,
                     mul2(pack2(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1])), k2));
            y[i] = fma2(product, factors[h / 2 + i], add2(shifts[h / 2 + i], v2));
          }
        }
        if (h + RH == RG) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&c->s_empty[group][buffer]);
        }
        if (at_end) {
#pragma unroll
          for (int r = 0; r < RH; r += 2) {
            float y0, y1;
            unpack2(y[r / 2], y0, y1);
            if (position > limits[h + r]) y0 = -INFINITY;
            if (position > limits[h + r + 1]) y1 = -INFINITY;
            y[r / 2] = pack2(y0, y1);
          }
        }
#pragma unroll
        for (int r = 0; r < RH / 2; ++r) {
          float y0, y1;
          unpack2(y[r], y0, y1);
          high = fmaxf(high, fmaxf(y0, y1));
        }
        if (h == 0) {  // the weights of the tile before have been read, and O holds it
          ok = wait<S>(smem_u32(&c->p_empty[group]), (uses & 1) ^ 1) && ok;
          tcgen05_fence_after();
          if (!ok) *failed = 1;
        }
        const bool rise = group_any(group, is_first || high > kLargestBits);
        stop = *failed != 0;
        if (stop) break;
        if (rise) {
          // the largest of each row that it may be, eight rows at a time
#pragma unroll
          for (int i = 0; i < RH; i += 8) {
            float z[8];
#pragma unroll
            for (int k = 0; k < 8; k += 2) unpack2(y[(i + k) / 2], z[k], z[k + 1]);
            const float of_eight = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])),
                                         fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7])));
            if (!__any_sync(0xffffffffu, is_first || of_eight > kLargestBits)) continue;
            int mine = kLowest;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int largest = __reduce_max_sync(0xffffffffu, ordered(z[k]));
              if (lane == k) mine = largest;
            }
            if (lane < 8 && (is_first || mine > ordered(kLargestBits))) atomicMax(&c->highest[r0 + h + i + lane], mine);
          }
          group_sync(group);
          if (token < 32) {
            bool risen = false;
            if (token < RH) {
              const int r = r0 + h + token;
              const float top = from_ordered(c->highest[r]);
              c->highest[r] = kLowest;
              risen = top > -INFINITY;
              const float by = risen ? top - kWeightBits : 0.0f;  // (in a first tile a reference may fall, too)
              c->rise[r] = -by;
              c->fade[r] = is_first ? 1.0f : exp2_approx(-by);
              c->shift[r] -= by;
            }
            const uint32_t rows = __ballot_sync(0xffffffffu, risen);
            if (lane == 0) c->risen[group] = rows;
          }
          group_sync(group);
#pragma unroll
          for (int r = 0; r < RH / 2; ++r) {
            y[r] = add2(y[r], rises[h / 2 + r]);
            sum[h / 2 + r] = mul2(sum[h / 2 + r], fades[h / 2 + r]);
          }
          if (!is_first) {
#pragma unroll 1
            for (int i = 0; i < RH; i += 8) {
              if ((c->risen[group] >> i & 0xffu) == 0) continue;
              uint32_t o[16];
              tmem_ld_x8_async(o_at + h + i, o);
              tmem_ld_x8_async(o_at + RG + h + i, o + 8);
              tmem_ld_wait();
              registers_loaded<16>(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * c->fade[r0 + h + i + (k & 7)]);
              tmem_st_x8(o_at + h + i, o);
              tmem_st_x8(o_at + RG + h + i, o + 8);
            }
            tmem_st_wait();
          }
        }
#pragma unroll
        for (int i = 0; i < RH; i += 8) {
          uint32_t a[4], b[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float p0, p1;
            unpack2(y[i / 2 + k], p0, p1);
            p0 = exp2_approx(p0);
            p1 = exp2_approx(p1);
            sum[(h + i) / 2 + k] = fma2(pack2(p0, p1), v2_inverse, sum[(h + i) / 2 + k]);
            two_terms(p0, p1, a[k], b[k]);
          }
          *reinterpret_cast<uint2*>(weights + weight_offset<S>(token, h + i)) =
              make_uint2(a[0] | (a[1] << 16), a[2] | (a[3] << 16));
          *reinterpret_cast<uint2*>(weights + weight_offset<S>(token, RG + h + i)) =
              make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
        }
      }
      if (stop) break;  // (the whole group; all groups leave together, at the top)
      fence_proxy_async_smem();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->p_full[group]);
    }
    first_no += s.tiles;
    // the next segment's queries are on their way during the end of this one
    const uint32_t following = segments + 1;
    const bool known = wait<S>(smem_u32(&c->segment_full[following % kSegments]), (following / kSegments) & 1);
    some = known && c->has_segment[following % kSegments];
    if (some) load_queries<S>(args, c->segment[following % kSegments], queries);
    // the rows' sums of weights over the 128 threads, in a fixed order
    float each[RG];
#pragma unroll
    for (int r = 0; r < RG; r += 2) unpack2(sum[r / 2], each[r], each[r + 1]);
    warp_sums<RG>(each, lane);
    c->warp_sum[warp][sum_row<RG>(lane, 0)] = each[0];
    ok = wait<S>(smem_u32(&c->p_empty[group]), (uses & 1) ^ 1) && known;
    tcgen05_fence_after();
    if (!ok) *failed = 1;
    group_sync(group);
    if (token < RG) {
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) x += c->warp_sum[group * 4 + w][token];
      c->sum[r0 + token] = x;
      c->inverse[r0 + token] = 1.0f / x;
    }
    if (streams > 1) {
      softmax_sync<S>();  // (values that are no numbers may have been found in any stream)
    } else {
      group_sync(group);
    }
    // a thread per dimension now
    const bool alone = s.part < 0, direct = alone && streams == 1;
    float* slot = split.slots + slot_floats(S::kRows) * (alone ? kSlotsPerBlock * blockIdx.x + 2 : s.part);
    const int bad = c->first_bad[token];
    if (has_rows) {
      const int* out_rows = c->out_row + my_rows * RG;
#pragma unroll 1
      for (int i = 0; i < RG && out_rows[i] >= 0; i += 8) {
        uint32_t a[16];
        tmem_ld_x8_async(o_at + i, a);
        tmem_ld_x8_async(o_at + RG + i, a + 8);
        tmem_ld_wait();
        registers_loaded<16>(a);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = i + k, to = out_rows[r];
          float o = fmaf(__uint_as_float(a[k + 8]), 0.0625f, __uint_as_float(a[k]));
          if (limits[r] >= bad) o = NAN;
          if (to < 0) continue;
          if (direct) {
            args.out[static_cast<size_t>(to) * kHeadDim + token] = __float2bfloat16(o * c->inverse[r0 + r]);
          } else {
            __stcg(slot + (r0 + r) * kHeadDim + token, o);
          }
        }
      }
      if (!direct && token < RG) {
        // (a row that has seen no token, for want of a tile or behind its mask, leaves nothing)
        const int r = r0 + token;
        __stcg(slot + S::kRows * kHeadDim + r, c->sum[r] == 0.0f ? -INFINITY : -c->shift[r]);
        __stcg(slot + S::kRows * (kHeadDim + 1) + r, c->sum[r]);
      }
    }
    tcgen05_fence_before();
    if (!alone) {
      if (threadIdx.x == 0) c->to_join[joins] = s;
      ++joins;
    } else if (!direct) {
      __threadfence_block();
      softmax_sync<S>();
      join<S>(args, split, s, 1, 0, c);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&c->segment_empty[segments % kSegments]);
  }
  if (joins == 0) return true;
  // (all threads' sums are behind the barrier at the top of the loop, so one thread speaks for them)
  if (threadIdx.x == 0) {
    __threadfence();
#pragma unroll 1
    for (int i = 0; i < joins; ++i) atomicAdd(&split.counters[c->to_join[i].lead], 1);
  }
#pragma unroll 1
  for (int i = 0; i < joins; ++i) {
    if (!wait_and_join<S>(args, split, c->to_join[i], c)) return false;
  }
  return true;
}

template <typename S>
__global__ void __launch_bounds__(S::kThreads, S::kBlocks)
    cached_kernel(const __grid_constant__ CUtensorMap map, const CachedArgs args, const Split split) {
  static_assert(fits_on_sm<S>());
  extern __shared__ uint8_t raw[];
  uint8_t* keys = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint8_t* values = keys + S::kKeySlots * kTileBytes;
  uint8_t* q = values + S::kValueSlots * kTileBytes;
  uint8_t* weights = q + S::kQueryBytes;
  Control<S>* c = reinterpret_cast<Control<S>*>(weights + S::kWeightBytes);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int i = 0; i < S::kKeySlots; ++i) {
      mbar_init(&c->k_full[i], 1);
      mbar_init(&c->k_empty[i], 1);
    }
#pragma unroll 1
    for (int i = 0; i < S::kValueSlots; ++i) {
      mbar_init(&c->v_full[i], 1);
      mbar_init(&c->v_empty[i], 1);
    }
#pragma unroll 1
    for (int g = 0; g < S::kGroups; ++g) {
      for (int i = 0; i < S::kScores; ++i) {
        mbar_init(&c->s_full[g][i], 1);
        mbar_init(&c->s_empty[g][i], 4);
      }
      mbar_init(&c->p_full[g], 4);
      mbar_init(&c->p_empty[g], 1);
      c->failed[g] = 0;
    }
    mbar_init(&c->q_full, S::kSoftmaxWarps);
    mbar_init(&c->drained, 1);
#pragma unroll 1
    for (int i = 0; i < kSegments; ++i) {
      mbar_init(&c->segment_full[i], 1);
      mbar_init(&c->segment_empty[i], S::kSoftmaxWarps + 1);
    }
    c->found = 0;
    c->found_before = 0;
    fence_barrier_init();
  }
  if (warp == S::kSoftmaxWarps) {
    tmem_alloc(&c->tmem, S::kColumns);
    tmem_relinquish();
  }
  find_begin<S>(args, c);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = c->tmem;
  if constexpr (S::kSplitRegisters) {
    if (warp < S::kSoftmaxWarps) {
      more_registers<kSoftmaxRegisters>();
    } else {
      fewer_registers<kOtherRegisters>();
    }
  }
  if (warp < S::kSoftmaxWarps) {
    if (!softmax_role<S>(args, split, values, q, weights, tmem, c) && (threadIdx.x & 31) == 0) {
      report_cache_error(args.cache.error, kDevWaitTimeout);
    }
  } else if (warp == S::kSoftmaxWarps) {
    const bool ok = mma_role<S>(smem_u32(keys), smem_u32(values), smem_u32(q), smem_u32(weights), tmem, c);
    if (elect_one()) {
      if (!ok) report_cache_error(args.cache.error, kDevWaitTimeout);
      tcgen05_commit(&c->drained);
    }
    __syncwarp();
    wait<S>(smem_u32(&c->drained), 0);
  } else if (warp == S::kSoftmaxWarps + 1) {
    load_role<S>(args, &map, smem_u32(keys), smem_u32(values), c);
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == S::kSoftmaxWarps) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, S::kColumns);
  }
}

template <typename S>
cudaError_t launch(const CUtensorMap& map, const CachedArgs& args, const Split& split, int sms, cudaStream_t stream) {
  cudaError_t err = allow_shared_memory(cached_kernel<S>);
  if (err != cudaSuccess) return err;
  cached_kernel<S><<<sms * S::kBlocks, S::kThreads, shared_bytes<S>(), stream>>>(map, args, split);
  return cudaGetLastError();
}

}  // namespace

size_t attention_cached_workspace_bytes() {
  // (two blocks of 16 rows need less than one of 128)
  return kAttendCounterBytes + sizeof(float) * slot_floats(kMaxRows) * kSlotsPerBlock * device_sms();
}

cudaError_t launch_attention_cached(const CachedArgs& args, cudaStream_t stream) {
  const int sms = device_sms();
  if (sms * 2 * sizeof(int) > kAttendCounterBytes) return cudaErrorInvalidValue;
  CUtensorMap map;
  if (!pages_tensor_map(args.cache, &map)) return cudaErrorInvalidValue;
  const Split split{reinterpret_cast<int*>(args.cache.attend_workspace),
                    reinterpret_cast<float*>(args.cache.attend_workspace + kAttendCounterBytes)};
  // By the query rows that the entries have on average.  Entries with more are taken 8, 16 or 128 at a time
  // and read their keys and values again each time.
  const int64_t rows = (args.batch.rows + args.batch.count - 1) / args.batch.count *
                       static_cast<int64_t>(args.heads / args.cache.kv_heads);
  if (rows <= 8) return launch<Shape<8, 1>>(map, args, split, sms, stream);
  if (rows <= 16) return launch<Shape<16, 1>>(map, args, split, sms, stream);
  return launch<Shape<128, 4>>(map, args, split, sms, stream);
}

}  // namespace nmoe
