// What the two kernels of attention over the 8-bit cache share: how the tiles of all sequences are shared
// by the blocks, how keys and values get into shared memory, and how the pieces of a sequence are joined.
//
// For a row with query q at position x of its sequence, over the tokens j <= x whose keys and values are
// codes times powers of two (a power per page and head):
//   s_j = scale 2^(key power) q . kcode_j,   o = sum_j e^s_j 2^(value power) vcode_j / sum_j e^s_j
//
// What bounds it is reading the cache once.  So the codes go from memory to the tensor cores as they lie
// in their pages, and what they are multiplied by is made 8-bit as well, as a sum of two E4M3 terms: a bf16
// query's eight bits of significand fit the two exactly where it lies within 2^13 of its row's largest element (2^9
// in the kernel for many rows) and are off by 2^-21 (2^-17) of that at most where it does not; a weight
// e^(s - reference) is rounded to within 2^-8 of itself, or 2^-22 (2^-20.5 of the row's largest, which is 2^-1.5 at
// least).  The keys' powers enter the
// scores and those of the values the exponents of the weights, whose reference is a running maximum of both
// together, so it does not matter how far powers lie apart.  The sums of the weights without the values'
// powers are kept in FP32 beside.
//
// With R rows of queries (new rows x heads that share the key head) at a time, W tiles of 128 tokens in all (and
// some more for what each sequence, key head and rows cost beside) and G blocks, block g takes the tiles [W g / G, W (g + 1) / G)
// in order, whatever the sequences' lengths.
// Where a (sequence, key head) is cut, each piece leaves its sums in the workspace.  When all have, these blocks
// join them, a share of the rows at a time; each row is joined piece by piece in order, so results never depend
// on timing or on who joins.  Nobody has to wait: a block that sees pieces missing for some 30 us leaves, and the
// one that brings the last piece joins what nobody else does.  (All blocks run at once only if no other kernel
// holds SMs; two calls on two streams could otherwise each wait for blocks that the other keeps out.)
#pragma once

#include <cuda_fp16.h>

#include "attention.h"
#include "attention_mma.cuh"
#include "kernels.h"

namespace nmoe {

constexpr int kKeyTile = 128;  // tokens
constexpr int kKeyTileBytes = kKeyTile * kHeadDim;
constexpr int kMaxPagesPerTile = kKeyTile / 16;
constexpr int kMaxRows = 128;
constexpr int kSegments = 4;
constexpr int kSlotsPerBlock = 2;      // of the workspace: a piece that began in a block before, one that goes on
constexpr float kWeightBits = -1.5f;  // a row's largest weight is 2^-1.5 when its reference is set ...
constexpr float kLargestBits = 0.0f;  // ... and at most 1 before it is set anew
constexpr float kCodeScale = 256.0f;  // of weights as codes
// An exponent is score - reference by one fma, off by 2^-24 of what comes out.  In a tile that lies this many orders
// above its row's reference so far (keys before it that are masked by values of their own), that would be 2^-10 and
// more: what the row has summed up is worth nothing there, and it begins anew.
constexpr float kFarBits = 8192.0f;
constexpr float kNoReference = -3e38f;  // of a row whose scores so far are all -infinity

// The tiles of one (sequence, key head, rows) that a block works on.
struct Segment {
  int first, rows, length;  // of the batch entry
  int kv_head, row0;        // first of the query rows
  int tile, tiles;
  int part;                 // -1: all of them; else the slot of the workspace for its sums
  int lead, parts;          // the first block with a part, and how many have one
};

// Tiles 0 .. total - 1 shared by blocks: the first `more` have one more than `each`.
struct Shares {
  int total, blocks, each, more;

  __device__ int begin(int block) const { return block >= blocks ? total : block * each + min(block, more); }
  __device__ int block_of(int tile) const {
    const int ahead = tile - more * (each + 1);
    return ahead < 0 ? tile / (each + 1) : more + ahead / each;
  }
};

// Shared memory of a block that the warps of all roles use.
template <typename S>
struct WorkControl {
  uint64_t k_full[S::kKeySlots], k_empty[S::kKeySlots], v_full[S::kValueSlots], v_empty[S::kValueSlots];
  uint64_t segment_full[kSegments], segment_empty[kSegments], q_full, drained;
  Segment segment[kSegments];  // a place is given back when the segment is done
  int has_segment[kSegments];
  Segment to_join[2];          // the (at most two) that other blocks have pieces of
  int powers[S::kValueSlots][2][kMaxPagesPerTile];  // of a tile's pages, keys and values
  // of this segment's rows and the next one's
  alignas(16) float factor[2][S::kRows];  // what a row's product of codes is multiplied by
  int out_row[2][S::kRows];               // of the result, -1: none
  int limit[2][S::kRows];                 // a row's position: the last token it sees
  int first_bad[kHeadDim];             // position of the first masked value that is no number, by dimension
  int found_bad;
  int share, pieces;  // of a join
  uint32_t tmem;
  int64_t before[S::kThreads / 32];
  int stopped;        // an error was pending before this call
  int patience;       // cycles that a block waits for the pieces of a join
  Shares shares;      // of all tiles
  BatchEntry entry;   // the entry in which this block's begin,
  int found, found_before;  // which it is, and the tiles of those before it
};

// What a block leaves for the join: 128 sums a row, then the references and the sums of weights.
__host__ __device__ constexpr size_t slot_floats(int rows) { return static_cast<size_t>(rows) * (kHeadDim + 2); }

// By the block in which a (sequence, key head) begins, all 0 between calls.
struct JoinCounters {
  int pieces;  // that are there, and kLeft for each block that left before all were; stands once all are
  int taken;   // shares of rows, where a block has left
  int done;    // blocks that ask for nothing more
};
constexpr int kLeft = 1 << 16;
constexpr int kMaxBlocks = static_cast<int>(kAttendCounterBytes / sizeof(JoinCounters));
constexpr int kJoinPatience = 1 << 16;  // cycles

struct Split {
  JoinCounters* counters;
  float* slots;
};

// Instruction descriptor of kind::f8f6f4 on E4M3 operands, FP32 sums, M = 128; an operand may lie in rows of
// consecutive m or n instead of consecutive k.
__host__ __device__ constexpr uint32_t make_idesc_e4m3(uint32_t n, bool a_along_m, bool b_along_n) {
  return (1u << 4) | (a_along_m ? 1u << 15 : 0u) | (b_along_n ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// D[tmem] (+)= A B^T with A in shared memory ...
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

// ... or in TMEM, four codes to a column.
__device__ __forceinline__ void mma_e4m3_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

// Floats as integers of the same order (no NaN), and back.
__device__ __forceinline__ int ordered(float x) {
  const int bits = __float_as_int(x);
  return bits ^ ((bits >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
constexpr int kLowest = static_cast<int>(0x807fffffu);  // of -infinity

// All softmax warps.
template <typename S>
__device__ __forceinline__ void softmax_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(S::kSoftmaxWarps * 32) : "memory");
}
template <typename S>
__device__ __forceinline__ bool softmax_any(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(mine)), "n"(S::kSoftmaxWarps * 32)
      : "memory");
  return any != 0;
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
// Four weights w in [0, 1] as four codes each of two terms, 256 w = a + b / 16: a is cut off, b rounded, which
// leaves 2^-8 of w at most, or 2^-14.  A binary16 number of up to 1 has the exponent field and the first bits of
// the significand of the E4M3 number 256 times it, subnormal ones too, so whole-number operations do: the
// conversions to and from E4M3 run at the rate of the exponentials (with them a tile of 128 rows took 1860 cycles
// from exponents to codes, of which the exponentials are 1024).
__device__ __forceinline__ void weight_codes(const float (&w)[4], uint32_t& a, uint32_t& b) {
  uint32_t first[2], second[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2 v = __floats2half2_rn(w[2 * i], w[2 * i + 1]);
    const uint32_t bits = *reinterpret_cast<const uint32_t*>(&v), kept = bits & 0xff80ff80u;
    const __half2 rest = __hmul2(__hsub2(v, *reinterpret_cast<const __half2*>(&kept)), __float2half2_rn(16.0f));
    first[i] = bits >> 7;
    second[i] = (*reinterpret_cast<const uint32_t*>(&rest) + 0x00400040u) >> 7;
  }
  a = __byte_perm(first[0], first[1], 0x6420);
  b = __byte_perm(second[0], second[1], 0x6420);
}

__device__ __forceinline__ float power_of_two(int e) {  // -126 <= e <= 127
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Entry i of a part of the work: of the batch, or a group as one, whose rows are all its members' and whose tokens those
// that they share, as the first of them with rows has them.
__device__ __forceinline__ BatchEntry group_entry(const CachedArgs& args, int g) {
  const Batch& b = args.batch;
  BatchEntry e;
  e.sequence = e.first = e.rows = e.length = e.skip = 0;
  const int from = args.groups[g], to = args.groups[g + 1];
  e.valid = from >= 0 && from <= to && to <= b.count;
  if (!e.valid || from == to) return e;
  int leader = from;
  while (leader + 1 < to && b.offsets[leader + 1] <= b.offsets[leader]) ++leader;
  const int first = b.offsets[from], rows = b.offsets[to] - first, shared = args.shared[leader];
  const int sequence = b.sequences[leader];
  e.valid = first >= 0 && rows >= 0 && rows <= b.rows - first && shared >= 0 && shared % kKeyTile == 0 &&
            static_cast<unsigned>(sequence) < static_cast<unsigned>(args.cache.max_sequences);
  if (!e.valid || shared == 0) return e;
  const int64_t room = static_cast<int64_t>(args.cache.max_pages) << args.cache.page_shift;
  e.valid = shared <= args.cache.lengths[sequence] && shared <= room;
  if (!e.valid) return e;
  e.sequence = sequence;
  e.first = first;
  e.rows = rows;
  e.length = shared;
  return e;
}
template <Part P>
__device__ __forceinline__ BatchEntry part_entry(const CachedArgs& args, int i) {
  if constexpr (P == Part::kShared) return group_entry(args, i);
  BatchEntry e = batch_entry(args.cache, args.batch, i);
  if constexpr (P == Part::kOwn) {
    if (e.valid) {
      e.skip = args.shared[i];
      e.valid = e.skip >= 0 && e.skip % kKeyTile == 0 && e.skip <= e.length - e.rows;
    }
    if (!e.valid) e.rows = e.length = e.skip = 0;
  }
  return e;
}
template <Part P>
__device__ __forceinline__ int part_count(const CachedArgs& args) {
  return P == Part::kShared ? args.group_count : args.batch.count;
}

// How a batch entry's tiles lie in the order of all: by key head, then by rows, kRows at a time.
template <typename S>
struct EntryTiles {
  int tiles, row_tiles;  // of tokens, of rows
  int cost;              // of one (key head, rows): the tiles lie behind S::kUnitCost
  int64_t all;

  __device__ EntryTiles(const CachedArgs& args, const BatchEntry& e) {
    tiles = (e.length + kKeyTile - 1) / kKeyTile - e.skip / kKeyTile;
    row_tiles = (e.rows * (args.heads / args.cache.kv_heads) + S::kRows - 1) / S::kRows;
    cost = tiles + S::kUnitCost;
    all = static_cast<int64_t>(cost) * row_tiles * args.cache.kv_heads;
  }
};

// Rows that get no results become zeros, each block's share of them by one or all threads.
static __device__ __noinline__ void clear_rows(__nv_bfloat16* out, int heads, int from, int to, int thread, int threads) {
  const int64_t of_row = static_cast<int64_t>(heads) * (kHeadDim / 8);
  for (int64_t row = from + static_cast<int64_t>(blockIdx.x); row < to; row += gridDim.x) {
    for (int64_t i = thread; i < of_row; i += threads) reinterpret_cast<uint4*>(out)[row * of_row + i] = make_uint4(0, 0, 0, 0);
  }
}

// All threads: the number of tiles, and the entry in which this block's begin.
template <typename S, Part P>
__device__ void find_begin(const CachedArgs& args, WorkControl<S>* c) {
  const int n = part_count<P>(args), each = (n + S::kThreads - 1) / S::kThreads;
  const int begin = min(n, static_cast<int>(threadIdx.x) * each), end = min(n, begin + each);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // (one thread's word: a wait that runs out in another block of this launch writes it)
  CacheWords words{};
  if (threadIdx.x == 0) words = cache_words(args.cache);
  int64_t mine = 0;
  BatchEntry e;
#pragma unroll 1
  for (int i = begin; i < end; ++i) {
    e = part_entry<P>(args, i);
    if (!e.valid) {
      if (blockIdx.x == 0) report_cache_error(args.cache.raised, kCacheBadSequence);
      if (P != Part::kShared) {
        const int from = args.batch.offsets[i], to = args.batch.offsets[i + 1];
        if (from >= 0 && to <= args.batch.rows) clear_rows(args.out, args.heads, from, to, 0, 1);
      }
    }
    mine += EntryTiles<S>(args, e).all;
  }
  int64_t upto = mine;
#pragma unroll
  for (int step = 1; step < 32; step *= 2) {
    const int64_t other = __shfl_up_sync(0xffffffffu, upto, step);
    if (lane >= step) upto += other;
  }
  if (lane == 31) c->before[warp] = upto;
  if (threadIdx.x == 0) {
    c->stopped = words.error;
    c->patience = words.impatient ? 0 : kJoinPatience;
  }
  __syncthreads();
  int64_t total = 0, below = upto - mine;
#pragma unroll 1
  for (int w = 0; w < S::kThreads / 32; ++w) {
    if (w < warp) below += c->before[w];
    total += c->before[w];
  }
  // (more than 2^31 tiles are some 70 TB of codes to be read; with fewer tiles than blocks, the first blocks have
  // one each)
  if (total > INT32_MAX && threadIdx.x == 0) report_cache_error(args.cache.raised, kCacheBadSequence);
  if (total > INT32_MAX || c->stopped != 0) {
    total = 0;
    if (P != Part::kShared) {
      clear_rows(args.out, args.heads, max(args.batch.offsets[0], 0), min(args.batch.offsets[n], args.batch.rows), threadIdx.x,
                 S::kThreads);
    }
  }
  Shares shares;
  shares.total = static_cast<int>(total);
  shares.blocks = min(shares.total, static_cast<int>(gridDim.x));
  shares.each = shares.blocks > 0 ? shares.total / shares.blocks : 0;
  shares.more = shares.total - shares.blocks * shares.each;
  if (threadIdx.x == 0) c->shares = shares;
  if (static_cast<int>(blockIdx.x) >= shares.blocks) return;
  const int start = shares.begin(blockIdx.x);
  if (start >= below && start < below + mine) {  // one thread's
#pragma unroll 1
    for (int i = begin; i < end; ++i) {
      if (each > 1) e = part_entry<P>(args, i);
      const int64_t tiles = EntryTiles<S>(args, e).all;
      if (start < below + tiles) {
        c->found = i;
        c->found_before = static_cast<int>(below);
        c->entry = e;
        break;
      }
      below += tiles;
    }
  }
}

struct NoQueries {
  __device__ bool operator()(const Segment&, uint32_t) const { return true; }
};

// The warp that brings keys and values in, a page at a time, and by `load_queries(segment, number)` what else a segment
// needs.
template <typename S, Part P, typename Queries = NoQueries>
__device__ void load_role(const CachedArgs& args, const CUtensorMap* map, uint32_t keys_at, uint32_t values_at, WorkControl<S>* c,
                          Queries load_queries = Queries()) {
  const PagedCache& cache = args.cache;
  const int lane = threadIdx.x & 31, g = blockIdx.x;
  const Shares shares = c->shares;
  const int begin = shares.begin(g), stop = shares.begin(g + 1);
  const int pages_per_tile = kKeyTile >> cache.page_shift;
  const uint32_t page_bytes = kHeadDim << cache.page_shift;
  uint32_t no = 0, segments = 0;  // tiles, segments so far
  int i = c->found;
  int entry_at = begin < stop ? c->found_before : stop;
  BatchEntry e = c->entry;
  bool ok = true;
#pragma unroll 1
  while (entry_at < stop && ok) {
    const EntryTiles<S> t(args, e);
    // the first (key head, rows) that reach into this block's share
    const int unit = max(begin - entry_at, 0) / t.cost;
    int head = unit / t.row_tiles, row_tile = unit % t.row_tiles;
    int unit_at = entry_at + unit * t.cost;
    const int last_page = pages_of(cache, e.length);
#pragma unroll 1
    for (; head < cache.kv_heads && unit_at < stop && ok; unit_at += t.cost) {
      Segment s;
      s.first = e.first;
      s.rows = e.rows;
      s.length = e.length;
      s.kv_head = head;
      s.row0 = row_tile * S::kRows;
      const int tiles_at = unit_at + S::kUnitCost;
      s.tile = max(begin - tiles_at, 0);
      s.tiles = min(stop - tiles_at, t.tiles) - s.tile;
      s.lead = shares.block_of(tiles_at);
      s.parts = shares.block_of(tiles_at + t.tiles - 1) - s.lead + 1;
      s.part = s.parts == 1 ? -1 : kSlotsPerBlock * g + (g == s.lead);
      if (++row_tile == t.row_tiles) {
        row_tile = 0;
        ++head;
      }
      if (s.tiles <= 0) continue;
      s.tile += e.skip / kKeyTile;
      const uint32_t place = segments % kSegments;
      if (!(ok = mbar_wait_warp(smem_u32(&c->segment_empty[place]), ((segments / kSegments) & 1) ^ 1))) break;
      if (lane == 0) {
        c->segment[place] = s;
        c->has_segment[place] = 1;
        mbar_arrive(&c->segment_full[place]);
      }
      __syncwarp();
      if (!(ok = load_queries(s, segments))) break;
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
              report_cache_error(cache.raised, kCacheBadSequence);
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
          if (!(ok = mbar_wait_warp(empty, (round & 1) ^ 1))) break;
          const uint32_t bar = smem_u32(half ? &c->v_full[v_slot] : &c->k_full[k_slot]);
          const uint32_t to = half ? values_at + v_slot * kKeyTileBytes : keys_at + k_slot * kKeyTileBytes;
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
    entry_at += static_cast<int>(t.all);
    while (entry_at < stop && ok) {  // (entries without rows have no tiles)
      e = part_entry<P>(args, ++i);
      if (e.rows > 0) break;
    }
  }
  if (ok) {
    const uint32_t place = segments % kSegments;
    ok = mbar_wait_warp(smem_u32(&c->segment_empty[place]), ((segments / kSegments) & 1) ^ 1);
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
    mbar_wait_warp(smem_u32(&c->k_full[tile % S::kKeySlots]), (tile / S::kKeySlots) & 1);
    mbar_wait_warp(smem_u32(&c->v_full[tile % S::kValueSlots]), (tile / S::kValueSlots) & 1);
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

// kBatch rows of a segment's queries to each warp: read ...
template <typename S>
__device__ __forceinline__ void load_queries(const CachedArgs& args, const Segment& s, int batch, uint2 (&raw)[S::kBatch]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = args.heads / args.cache.kv_heads;
#pragma unroll
  for (int k = 0; k < S::kBatch; ++k) {
    const int row = s.row0 + (batch * S::kBatch + k) * S::kSoftmaxWarps + warp, token = row / group;
    raw[k] = make_uint2(0, 0);
    if (token < s.rows) {
      raw[k] = *reinterpret_cast<const uint2*>(args.q + static_cast<int64_t>(s.first + token) * args.q_stride +
                                               (s.kv_head * group + row % group) * kHeadDim + lane * 4);
    }
  }
}

// Four elements of a row of queries to a lane: their codes as two terms, the row scaled by a power of two, the second
// terms multiplied by `Second`; `factor`: what the row's products of codes are multiplied by.
template <int Second>
__device__ __forceinline__ void query_terms(const uint2& raw, float scale, uint32_t& first, uint32_t& second, float& factor) {
  float x[4];
  x[0] = __uint_as_float(raw.x << 16);
  x[1] = __uint_as_float(raw.x & 0xffff0000u);
  x[2] = __uint_as_float(raw.y << 16);
  x[3] = __uint_as_float(raw.y & 0xffff0000u);
  // (magnitudes as whole numbers: what is no number is beyond them all)
  const uint32_t m = max(max(raw.x & 0x7fffu, (raw.x >> 16) & 0x7fffu), max(raw.y & 0x7fffu, (raw.y >> 16) & 0x7fffu));
  const int largest = static_cast<int>(__reduce_max_sync(0xffffffffu, m));
  // the largest element's exponent becomes 7: below 256
  const int power = max(largest >> 7, 1) - 134;
  const int some = max(power, -100), rest = power - some;  // (2^-power may be beyond FP32)
  const float down = power_of_two(-some), downer = power_of_two(-rest);
  uint32_t a[2], b[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2 v = __floats2half2_rn(x[2 * i] * down * downer, x[2 * i + 1] * down * downer);
    a[i] = codes_of(v);
    b[i] = codes_of(__hmul2(__hsub2(v, halves_of(a[i])), __float2half2_rn(static_cast<float>(Second))));
  }
  first = a[0] | (a[1] << 16);
  second = b[0] | (b[1] << 16);
  // (a row that is no number: its scores are none)
  factor = largest < 0x7f80 ? scale * kLog2e * power_of_two(some) * power_of_two(rest) : NAN;
}

// ... and put into shared memory as two terms.  The second terms, kRows rows behind the first, are multiplied by
// `Second`.
template <typename S, int Second>
__device__ __forceinline__ void store_queries(const CachedArgs& args, const Segment& s, int which, int batch,
                                              const uint2 (&raw)[S::kBatch], uint8_t* q, WorkControl<S>* c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = args.heads / args.cache.kv_heads;
#pragma unroll
  for (int k = 0; k < S::kBatch; ++k) {
    const int r = (batch * S::kBatch + k) * S::kSoftmaxWarps + warp;
    uint32_t first, second;
    float factor;
    query_terms<Second>(raw[k], args.scale, first, second, factor);
    const int chunk = lane >> 2, inside = (lane & 3) * 4, r2 = S::kRows + r;
    *reinterpret_cast<uint32_t*>(q + r * 128 + ((chunk ^ (r & 7)) << 4) + inside) = first;
    *reinterpret_cast<uint32_t*>(q + r2 * 128 + ((chunk ^ (r2 & 7)) << 4) + inside) = second;
    if (lane == 0) {
      c->factor[which][r] = factor;
      const int token = (s.row0 + r) / group;
      const bool valid = token < s.rows;
      c->limit[which][r] = s.length - s.rows + (valid ? token : 0);
      c->out_row[which][r] = valid ? (s.first + token) * args.heads + s.kv_head * group + (s.row0 + r) % group : -1;
    }
  }
}

// All of them, the first batch having been read; `which` of the row arrays takes what belongs to them.
template <typename S, int Second>
__device__ __forceinline__ void prepare_queries(const CachedArgs& args, const Segment& s, int which, uint2 (&raw)[S::kBatch], uint8_t* q,
                                                WorkControl<S>* c) {
  const int rows = s.rows * (args.heads / args.cache.kv_heads) - s.row0;
#pragma unroll 1
  for (int batch = 0; batch < S::kRows / (S::kBatch * S::kSoftmaxWarps); ++batch) {
    // (rows of warps that have none are not read by anybody)
    if (batch * S::kBatch * S::kSoftmaxWarps >= (rows + 31) / 32 * 32) break;
    uint2 next[S::kBatch];
    if (batch + 1 < S::kRows / (S::kBatch * S::kSoftmaxWarps)) load_queries<S>(args, s, batch + 1, next);
    store_queries<S, Second>(args, s, which, batch, raw, q, c);
#pragma unroll
    for (int k = 0; k < S::kBatch; ++k) raw[k] = next[k];
  }
}


// The values of a tile at the end of a sequence: places behind it hold anything and become 0; where a
// value that only some rows see is no number, it becomes 0 as well, and the rows that see it get it in
// the end (a weight of 0 times such a value would be none either).  A thread per token.
template <typename S>
__device__ __forceinline__ void clean_values(uint8_t* values, int token, int position, const Segment& s, WorkControl<S>* c) {
  uint4* row = reinterpret_cast<uint4*>(values + token * kHeadDim);
  if (position >= s.length) {
#pragma unroll
    for (int i = 0; i < 8; ++i) row[i] = make_uint4(0, 0, 0, 0);
  } else if (position > s.length - s.rows) {
    uint32_t any = 0;  // bit 7 of a byte for a code that is no number
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 x = row[i];
      any |= ((x.x & 0x7f7f7f7fu) + 0x01010101u) | ((x.y & 0x7f7f7f7fu) + 0x01010101u) |
             ((x.z & 0x7f7f7f7fu) + 0x01010101u) | ((x.w & 0x7f7f7f7fu) + 0x01010101u);
    }
    if (any & 0x80808080u) {
      uint8_t* codes = reinterpret_cast<uint8_t*>(row);
#pragma unroll 1
      for (int i = 0; i < kHeadDim; ++i) {
        if ((codes[i] & 0x7fu) != 0x7fu) continue;
        atomicMin(&c->first_bad[(((i >> 4) ^ (token & 7)) << 4) + (i & 15)], position);
        codes[i] = 0;
        c->found_bad = 1;
      }
    }
  }
  fence_proxy_async_smem();
}

// Joins the pieces of a (sequence, key head), one of as many shares of the rows.  Lanes per row: all 32 where there are
// few rows, or eight, so that four of a warp's many rows are on their way at once (a row after the other, asked for one
// ahead, took 6500 cycles for three of them: 48 sequences of 8192 tokens 113 -> 101 us).  A share of no more rows than
// there are warps spreads a row's pieces over the four instead, a quarter each.
template <typename S>
__device__ void join(const CachedArgs& args, const Split& split, const Segment& s, int share) {
  constexpr int kLanes = S::kRows > 16 ? 8 : 32;
  constexpr int kVectors = kHeadDim / 4 / kLanes;   // of four dimensions, to a lane
  constexpr int kAtOnce = kLanes == 32 ? 16 : 2;    // pieces (of many rows four spill: 112 us where two take 100)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = lane & (kLanes - 1), leader = lane - mine;
  const int group = args.heads / args.cache.kv_heads;
  const int pieces = s.parts, rows = min(S::kRows, s.rows * group - s.row0);
  const int end = rows * (share + 1) / pieces, slot = lane / kLanes;
  const bool spread = kLanes < 32 && rows <= pieces * S::kSoftmaxWarps;
  const int at_once = spread ? 1 : 32 / kLanes;  // rows
  const int from = spread ? pieces * slot / (32 / kLanes) : 0, to = spread ? pieces * (slot + 1) / (32 / kLanes) : pieces;
  const int longest = spread ? (pieces + 32 / kLanes - 1) / (32 / kLanes) : pieces;
  auto sums_of = [&](int p) { return split.slots + slot_floats(S::kRows) * (kSlotsPerBlock * (s.lead + p) + (p == 0)); };
#pragma unroll 1
  for (int base = rows * share / pieces + warp * at_once; base < end; base += S::kSoftmaxWarps * at_once) {
    const int r = min(base + (spread ? 0 : slot), end - 1), row = s.row0 + r;
    // the maximum so far is raised from chunk to chunk of pieces
    float top = -INFINITY, sum = 0.0f, o[4 * kVectors];
#pragma unroll
    for (int i = 0; i < 4 * kVectors; ++i) o[i] = 0.0f;
#pragma unroll 1
    for (int start = from; start < from + longest; start += kLanes) {
      float reference = -INFINITY, weight = 0.0f;  // a lane per piece
      if (start + mine < to) {
        const float* at = sums_of(start + mine) + S::kRows * kHeadDim + r;
        reference = __ldcg(at);
        weight = __ldcg(at + S::kRows);
      }
      const int count = min(kLanes, from + longest - start);
      float scale = 0.0f;
#pragma unroll 1
      for (int first = 0; first < count; first += kAtOnce) {
        float4 x[kAtOnce][kVectors];
#pragma unroll
        for (int p = 0; p < kAtOnce; ++p) {
          const float4* at = reinterpret_cast<const float4*>(sums_of(start + first + p) + r * kHeadDim) + mine;
#pragma unroll
          for (int i = 0; i < kVectors; ++i) {
            if (start + first + p < to) x[p][i] = __ldcg(at + i * kLanes);
          }
        }
        if (first == 0) {
          float higher = reference;
#pragma unroll
          for (int step = kLanes / 2; step > 0; step /= 2) higher = fmaxf(higher, __shfl_xor_sync(0xffffffffu, higher, step));
          higher = fmaxf(higher, top);
          const float keep = top > -INFINITY ? exp2_approx(top - higher) : 0.0f;
          scale = reference > -INFINITY ? exp2_approx(reference - higher) : 0.0f;
          weight *= scale;  // (of a piece far below the others 0, or what is no number)
          top = higher;
          sum *= keep;
#pragma unroll
          for (int i = 0; i < 4 * kVectors; ++i) o[i] *= keep;
        }
#pragma unroll
        for (int p = 0; p < kAtOnce; ++p) {
          const float f = __shfl_sync(0xffffffffu, scale, leader + ((first + p) & (kLanes - 1)));
          const float w = __shfl_sync(0xffffffffu, weight, leader + ((first + p) & (kLanes - 1)));
          if (spread ? start + first + p >= to : first + p >= count) continue;
          sum += w;
#pragma unroll
          for (int i = 0; i < kVectors; ++i) {
            o[4 * i] = fmaf(x[p][i].x, f, o[4 * i]);
            o[4 * i + 1] = fmaf(x[p][i].y, f, o[4 * i + 1]);
            o[4 * i + 2] = fmaf(x[p][i].z, f, o[4 * i + 2]);
            o[4 * i + 3] = fmaf(x[p][i].w, f, o[4 * i + 3]);
          }
        }
      }
    }
    if (spread) {
#pragma unroll
      for (int step = kLanes; step < 32; step *= 2) {
        const float higher = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
        const float keep = top > -INFINITY ? exp2_approx(top - higher) : 0.0f;
        top = higher;
        sum *= keep;
        sum += __shfl_xor_sync(0xffffffffu, sum, step);
#pragma unroll
        for (int i = 0; i < 4 * kVectors; ++i) {
          o[i] *= keep;
          o[i] += __shfl_xor_sync(0xffffffffu, o[i], step);
        }
      }
    }
    if (spread ? slot > 0 : base + slot >= end) continue;
    const float inverse = 1.0f / sum;
    const size_t at = static_cast<size_t>(s.first + row / group) * args.heads + s.kv_head * group + row % group;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      *reinterpret_cast<uint2*>(args.out + at * kHeadDim + (mine + i * kLanes) * 4) =
          make_uint2(pack_bf16(o[4 * i] * inverse, o[4 * i + 1] * inverse), pack_bf16(o[4 * i + 2] * inverse, o[4 * i + 3] * inverse));
    }
  }
}

// (a fence behind a plain load took 900 cycles)
__device__ __forceinline__ int load_acquire(const int* p) {
  int x;
  asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(x) : "l"(p) : "memory");
  return x;
}

// One thread: waits a while for the pieces that are missing.  The counter's word when all are there, or -1: this block
// has left.
__device__ __forceinline__ int wait_for_pieces(JoinCounters* counters, int parts, int patience) {
  const long long start = clock64();
  int word = load_acquire(&counters->pieces);
  while ((word & (kLeft - 1)) < parts && clock64() - start < patience) word = load_acquire(&counters->pieces);
  while ((word & (kLeft - 1)) < parts) {  // (it can have changed as often as there are blocks)
    const int seen = atomicCAS(&counters->pieces, word, word + kLeft);
    if (seen == word) return -1;
    word = seen;
    __threadfence();
  }
  return word;
}

// A block's part in the join of a segment's (sequence, key head).  If nobody has left, each block has the share of its
// own piece; else they take them in turn.  The last block that is done sets the counters back.
template <typename S>
__device__ void help_join(const CachedArgs& args, const Split& split, const Segment& s, WorkControl<S>* c) {
  JoinCounters* counters = &split.counters[s.lead];
  if (threadIdx.x == 0) c->pieces = wait_for_pieces(counters, s.parts, c->patience);
  softmax_sync<S>();
  const int word = c->pieces;
  // The last warp counts the block as done; where it joins rows first, the counter's answer is on its way meanwhile.
  const bool counts = threadIdx.x == 32 * (S::kSoftmaxWarps - 1);
  int done = 0;
  auto count = [&] {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %2, 0;\n\t"
        "@p atom.global.add.u32 %0, [%1], 1;\n\t}"
        : "+r"(done)
        : "l"(&counters->done), "r"(static_cast<uint32_t>(counts))
        : "memory");
  };
  if (word < kLeft) count();
  int share = word < 0 ? s.parts : static_cast<int>(blockIdx.x) - s.lead;
#pragma unroll 1
  for (;;) {
    if (word >= kLeft) {
      if (threadIdx.x == 0) c->share = atomicAdd(&counters->taken, 1);
      softmax_sync<S>();
      share = c->share;
    }
    if (share >= s.parts) break;
    join<S>(args, split, s, share);
    if (word < kLeft) break;
    softmax_sync<S>();
  }
  if (word >= kLeft) count();
  if (counts && done == s.parts - 1) counters->pieces = counters->taken = counters->done = 0;
}

// The end of a block's softmax warps: its pieces are there (all threads' sums are behind a barrier, so one
// thread speaks for them), and are joined with the others'.
template <typename S>
__device__ void announce_and_join(const CachedArgs& args, const Split& split, int joins, WorkControl<S>* c) {
  if (joins == 0) return;
  if (threadIdx.x == 0) {
    __threadfence();
#pragma unroll 1
    for (int i = 0; i < joins; ++i) atomicAdd(&split.counters[c->to_join[i].lead].pieces, 1);
  }
#pragma unroll 1
  for (int i = 0; i < joins; ++i) {
    if (i > 0) softmax_sync<S>();  // (the counters' words of the first are read)
    help_join<S>(args, split, c->to_join[i], c);
  }
}

// What a row leaves of a part: where its sums are, and whether in pieces.
__device__ __forceinline__ void leave_row_part(const CachedArgs& args, const Segment& s, int to, int row, float reference, float sum) {
  if (to < 0 || (s.part >= 0 && static_cast<int>(blockIdx.x) != s.lead)) return;
  args.row_parts[to] = {reference, sum, s.part < 0 ? 1 : s.parts << 8 | row, s.lead};
}

// Barriers of WorkControl; one thread.
template <typename S>
__device__ void init_work(WorkControl<S>* c) {
#pragma unroll 1
  for (int i = 0; i < S::kKeySlots; ++i) {
    mbar_init(&c->k_full[i], 1);
    mbar_init(&c->k_empty[i], 1);
  }
#pragma unroll 1
  for (int i = 0; i < S::kValueSlots; ++i) {
    mbar_init(&c->v_full[i], 1);
    mbar_init(&c->v_empty[i], S::kValueReaders);
  }
#pragma unroll 1
  for (int i = 0; i < kSegments; ++i) {
    mbar_init(&c->segment_full[i], 1);
    mbar_init(&c->segment_empty[i], S::kSegmentReaders);
  }
  mbar_init(&c->q_full, S::kQueryWriters);
  mbar_init(&c->drained, 1);
  c->found = 0;
  c->found_before = 0;
}

// For the kernel of more than 16 rows.
cudaError_t launch_cached_rows(const CUtensorMap& map, const CachedArgs& args, Part part, const Split& split, int sms, cudaStream_t stream);

}  // namespace nmoe
