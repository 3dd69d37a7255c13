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
// Blocks (two to an SM, one where there are 128 rows) share all tiles of all sequences evenly, whatever
// the sequences' lengths: block g of G takes the tiles [W g / G, W (g + 1) / G) of the W in order (G no larger than W).  Where
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
constexpr float kWeightBits = 8.0f;  // the largest weight is 2^8 or less ...
constexpr float kSlack = 0.8f;       // ... until its maximum has risen by this: 2^8.8 < 448

// R query rows, `Groups` times four warps that take R / Groups of them each.
template <int R, int Groups>
struct Shape {
  static constexpr int kRows = R, kGroups = Groups, kGroupRows = R / Groups;
  static constexpr int kN = 2 * R;
  static constexpr int kBlocks = R == kMaxRows ? 1 : 2;                // on an SM
  static constexpr int kScores = R >= 64 ? 1 : 2;                      // buffers of S
  static constexpr int kStages = R == kMaxRows ? 4 : R == 64 ? 2 : 3;  // tiles of keys and values in flight
  static constexpr int kSoftmaxWarps = 4 * Groups;
  static constexpr int kThreads = 32 * (kSoftmaxWarps + 2);
  static constexpr int kPanel = kN < 128 ? kN : 128;  // bytes of a token's row of weights in a panel
  static constexpr int kColumnsUsed = (kScores + 1) * kN;
  static constexpr int kColumns = kColumnsUsed <= 64 ? 64 : kColumnsUsed <= 128 ? 128 : kColumnsUsed <= 256 ? 256 : 512;
};

// The tiles of one (sequence, key head, rows) that a block works on.
struct Segment {
  int first, rows, length;  // of the batch entry
  int kv_head, row0;        // first of the query rows
  int tile, tiles;
  int part;                 // -1: all of them; else where its sums go
  int lead, parts;          // the first block with a part, and how many have one
};

template <typename S>
struct Control {
  uint64_t k_full[S::kStages], k_empty[S::kStages], v_full[S::kStages], v_empty[S::kStages];
  uint64_t s_full[S::kScores], s_empty[S::kScores], p_full, p_empty, q_full, drained;
  uint64_t segment_full[2], segment_empty[2];
  Segment segment[2];
  int has_segment[2];
  int powers[S::kStages][2][kMaxPagesPerTile];  // of a tile's pages, keys and values
  alignas(16) float factor[S::kRows];           // what a row's product of codes is multiplied by
  alignas(16) float shift[S::kRows];            // kWeightBits - the row's reference
  float top[S::kRows], fade[S::kRows];
  float warp_top[S::kSoftmaxWarps][S::kGroupRows];
  float warp_sum[S::kSoftmaxWarps][S::kGroupRows];
  float sum[S::kRows];
  int limit[S::kRows];                          // a row's position: the last token it sees
  int first_bad[kHeadDim];                      // position of the first masked value that is no number
  int failed[2];
  int last;
  uint32_t tmem;
  int64_t before[S::kThreads / 32];
  int64_t total, found_before;
  int found, blocks;  // the entry in which this block's tiles begin; blocks that have any
};

template <typename S>
constexpr size_t shared_bytes() {
  return 1024 + S::kStages * 2 * kTileBytes + 2 * S::kN * kTile + sizeof(Control<S>);
}

// What a block leaves for the join: a row's 128 sums, then the references and the sums of weights.
__host__ __device__ constexpr size_t part_floats(int rows) { return static_cast<size_t>(rows) * (kHeadDim + 2); }

struct Split {
  int* counters;  // a block's part of the sequence that begins in it: pieces that are done
  float* parts;
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

// The largest over the warp, in all lanes.
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
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
  asm volatile("bar.sync 3, %0;" ::"n"(S::kSoftmaxWarps * 32) : "memory");
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

template <typename S>
__device__ __forceinline__ int row_tiles(const CachedArgs& args, const BatchEntry& e) {
  return (e.rows * (args.heads / args.cache.kv_heads) + S::kRows - 1) / S::kRows;
}
template <typename S>
__device__ __forceinline__ int64_t entry_tiles(const CachedArgs& args, const BatchEntry& e) {
  return static_cast<int64_t>((e.length + kTile - 1) / kTile) * args.cache.kv_heads * row_tiles<S>(args, e);
}

// All threads: the number of tiles there are, and the entry in which this block's begin.
template <typename S>
__device__ void find_begin(const CachedArgs& args, Control<S>* c) {
  const int n = args.batch.count, each = (n + S::kThreads - 1) / S::kThreads;
  const int begin = min(n, static_cast<int>(threadIdx.x) * each), end = min(n, begin + each);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t mine = 0;
  for (int i = begin; i < end; ++i) {
    const BatchEntry e = batch_entry(args.cache, args.batch, i);
    if (!e.valid && blockIdx.x == 0) report_cache_error(args.cache.error, kCacheBadSequence);
    mine += entry_tiles<S>(args, e);
  }
  int64_t upto = mine;
#pragma unroll
  for (int step = 1; step < 32; step *= 2) {
    const int64_t other = __shfl_up_sync(0xffffffffu, upto, step);
    if (lane >= step) upto += other;
  }
  if (lane == 31) c->before[warp] = upto;
  __syncthreads();
  int64_t total = 0, below = upto - mine;
  for (int w = 0; w < S::kThreads / 32; ++w) {
    if (w < warp) below += c->before[w];
    total += c->before[w];
  }
  // (with fewer tiles than blocks, the first blocks have one each)
  const int blocks = static_cast<int>(min(total, static_cast<int64_t>(gridDim.x)));
  if (threadIdx.x == 0) {
    c->total = total;
    c->blocks = blocks;
  }
  if (static_cast<int>(blockIdx.x) >= blocks) return;
  const int64_t start = total * blockIdx.x / blocks;
  if (start >= below && start < below + mine) {  // one thread's
    for (int i = begin; i < end; ++i) {
      const int64_t tiles = entry_tiles<S>(args, batch_entry(args.cache, args.batch, i));
      if (start < below + tiles) {
        c->found = i;
        c->found_before = below;
        break;
      }
      below += tiles;
    }
  }
}

// The warp that brings keys and values in, a page at a time.
template <typename S>
__device__ void load_role(const CachedArgs& args, const CUtensorMap* map, uint32_t stages_at, Control<S>* c) {
  const PagedCache& cache = args.cache;
  const int lane = threadIdx.x & 31, G = c->blocks, g = blockIdx.x;
  const int64_t total = c->total;
  const int64_t stop = g < G ? total * (g + 1) / G : 0;
  int64_t at = g < G ? total * g / G : 0;
  const int pages_per_tile = kTile >> cache.page_shift;
  const uint32_t page_bytes = kHeadDim << cache.page_shift;
  uint32_t stage = 0, phase = 0, segments = 0, loads = 0;
  int i = c->found;
  int64_t entry_at = c->found_before;
  bool ok = true;
  while (at < stop && ok) {
    const BatchEntry e = batch_entry(cache, args.batch, i);
    const int tiles = (e.length + kTile - 1) / kTile, rows = row_tiles<S>(args, e);
    const int64_t entry_end = entry_at + entry_tiles<S>(args, e);
    const int last_page = pages_of(cache, e.length);
    while (at < min(stop, entry_end) && ok) {
      const int unit = static_cast<int>((at - entry_at) / tiles);
      const int64_t unit_at = entry_at + static_cast<int64_t>(unit) * tiles;
      Segment s;
      s.first = e.first;
      s.rows = e.rows;
      s.length = e.length;
      s.kv_head = unit / rows;
      s.row0 = (unit % rows) * S::kRows;
      s.tile = static_cast<int>(at - unit_at);
      s.tiles = static_cast<int>(min(stop, unit_at + tiles) - at);
      s.lead = static_cast<int>(((unit_at + 1) * G - 1) / total);
      s.parts = static_cast<int>(((unit_at + tiles) * G - 1) / total) - s.lead + 1;
      s.part = s.parts == 1 ? -1 : 2 * g + (g == s.lead);
      const uint32_t place = segments & 1;
      if (!(ok = wait_warp(smem_u32(&c->segment_empty[place]), ((segments >> 1) & 1) ^ 1))) break;
      if (lane == 0) {
        c->segment[place] = s;
        c->has_segment[place] = 1;
        mbar_arrive(&c->segment_full[place]);
      }
      __syncwarp();
      ++segments;
      int first_page = -1, page = 0, k_power = 0, v_power = 0;  // a lane per page, 32 at a time
      for (int tile = s.tile; tile < s.tile + s.tiles; ++tile) {
        const int wanted = tile * pages_per_tile;
        if (first_page < 0 || wanted >= first_page + 32) {
          first_page = wanted;
          if (wanted + lane < last_page) {
            page = page_at(cache, e.sequence, wanted + lane);
            if (page < 0) {
              report_cache_error(cache.error, kCacheBadSequence);
              page = 0;
            }
            k_power = cache.exponents[block_of_page(cache, args.layer, page, 0, s.kv_head)];
            v_power = cache.exponents[block_of_page(cache, args.layer, page, 1, s.kv_head)];
          }
        }
        const int count = min(pages_per_tile, last_page - wanted), from = wanted - first_page;
        for (int half = 0; half < 2; ++half) {
          uint64_t* empty = half ? &c->v_empty[stage] : &c->k_empty[stage];
          if (!(ok = wait_warp(smem_u32(empty), phase ^ 1))) break;
          if (half == 0) {  // (read by the softmax warps before they let the values' place go)
            if (!(ok = wait_warp(smem_u32(&c->v_empty[stage]), phase ^ 1))) break;
            const int p = __shfl_sync(0xffffffffu, k_power, (from + lane) & 31);
            const int z = __shfl_sync(0xffffffffu, v_power, (from + lane) & 31);
            if (lane < count) {
              c->powers[stage][0][lane] = p;
              c->powers[stage][1][lane] = z;
            }
            __syncwarp();
          }
          const uint32_t bar = smem_u32(half ? &c->v_full[stage] : &c->k_full[stage]);
          const uint32_t to = stages_at + (2 * stage + half) * kTileBytes;
          if (elect_one()) mbar_arrive_expect_tx_at(bar, count * page_bytes);
          __syncwarp();
          for (int j = 0; j < count; ++j) {
            const int id = __shfl_sync(0xffffffffu, page, from + j);
            const int row = static_cast<int>(block_of_page(cache, args.layer, id, half, s.kv_head) << cache.page_shift);
            if (elect_one()) tma_load_2d_at(to + j * page_bytes, map, 0, row, bar);
            __syncwarp();
          }
          ++loads;
        }
        if (!ok) break;
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      at += s.tiles;
    }
    entry_at = entry_end;
    ++i;
  }
  if (ok) {
    const uint32_t place = segments & 1;
    ok = wait_warp(smem_u32(&c->segment_empty[place]), ((segments >> 1) & 1) ^ 1);
    if (ok && lane == 0) {
      c->has_segment[place] = 0;
      mbar_arrive(&c->segment_full[place]);
    }
  }
  if (ok) return;
  if (lane == 0) report_cache_error(cache.error, kDevWaitTimeout);
  // what is in flight arrives before the block's shared memory is given up
  for (uint32_t back = 1; back <= min(loads, 2u * S::kStages); ++back) {
    const uint32_t load = loads - back, of = (load >> 1) % S::kStages;
    wait_warp(smem_u32(load & 1 ? &c->v_full[of] : &c->k_full[of]), ((load >> 1) / S::kStages) & 1);
  }
}

template <typename S>
__device__ bool mma_role(uint32_t stages_at, uint32_t q_at, uint32_t p_at, uint32_t tmem, Control<S>* c) {
  constexpr uint32_t kScoresDesc = make_idesc_e4m3(S::kN, false), kValuesDesc = make_idesc_e4m3(S::kN, true);
  // rows of weights are 16, 32, 64 or 128 bytes, swizzled in as many
  constexpr uint32_t kSwizzle = S::kPanel == 128 ? 2 : S::kPanel == 64 ? 4 : S::kPanel == 32 ? 6 : 0;
  const uint64_t q_desc = make_smem_desc(q_at, 16, 1024, 2);
  const uint64_t p_desc = S::kPanel == 16 ? make_smem_desc(p_at, 128, 128, 0)
                                          : make_smem_desc(p_at, kTile * S::kPanel, 8 * S::kPanel, kSwizzle);
  const uint32_t o = tmem + S::kScores * S::kN;
  uint32_t tile_no = 0;  // of all segments
  for (uint32_t segments = 0;; ++segments) {
    const uint32_t place = segments & 1;
    if (!wait_warp(smem_u32(&c->segment_full[place]), (segments >> 1) & 1)) return false;
    const int some = c->has_segment[place];
    const int tiles = c->segment[place].tiles;
    __syncwarp();
    if (!some) return true;
    if (elect_one()) mbar_arrive(&c->segment_empty[place]);
    __syncwarp();
    if (!wait_warp(smem_u32(&c->q_full), segments & 1)) return false;
    tcgen05_fence_after();
    // scores one tile ahead of the values
    for (int j = 0; j <= tiles; ++j) {
      if (j < tiles) {
        const uint32_t no = tile_no + j, stage = no % S::kStages, buffer = no % S::kScores;
        if (!wait_warp(smem_u32(&c->k_full[stage]), (no / S::kStages) & 1)) return false;
        if (!wait_warp(smem_u32(&c->s_empty[buffer]), ((no / S::kScores) & 1) ^ 1)) return false;
        tcgen05_fence_after();
        if (elect_one()) {
          const uint64_t k_desc = make_smem_desc(stages_at + 2 * stage * kTileBytes, 16, 1024, 2);
#pragma unroll
          for (int k = 0; k < kHeadDim / 32; ++k) {
            mma_e4m3(tmem + buffer * S::kN, advance_smem_desc(k_desc, k * 32), advance_smem_desc(q_desc, k * 32),
                     kScoresDesc, k > 0);
          }
          tcgen05_commit(&c->s_full[buffer]);
          tcgen05_commit(&c->k_empty[stage]);
        }
        __syncwarp();
      }
      if (j > 0) {
        const uint32_t no = tile_no + j - 1, stage = no % S::kStages;
        if (!wait_warp(smem_u32(&c->v_full[stage]), (no / S::kStages) & 1)) return false;
        if (!wait_warp(smem_u32(&c->p_full), no & 1)) return false;
        tcgen05_fence_after();
        if (elect_one()) {
          // eight tokens are 1024 bytes of values
          const uint64_t v_desc = make_smem_desc(stages_at + (2 * stage + 1) * kTileBytes, 16, 1024, 2);
#pragma unroll
          for (int k = 0; k < kTile / 32; ++k) {
            mma_e4m3(o, advance_smem_desc(v_desc, k * 4096), advance_smem_desc(p_desc, k * 32 * S::kPanel),
                     kValuesDesc, j > 1 || k > 0);
          }
          tcgen05_commit(&c->p_empty);
          tcgen05_commit(&c->v_empty[stage]);
        }
        __syncwarp();
      }
    }
    tile_no += tiles;
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

// The queries of a segment as two terms, each row scaled by a power of two; a warp per row.
template <typename S>
__device__ __forceinline__ void prepare_queries(const CachedArgs& args, const Segment& s, uint8_t* q, Control<S>* c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = args.heads / args.cache.kv_heads;
  for (int r = warp; r < S::kRows; r += S::kSoftmaxWarps) {
    const int row = s.row0 + r, token = row / group;
    const bool valid = row < s.rows * group;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (valid) {
      const uint2 raw = *reinterpret_cast<const uint2*>(args.q + static_cast<int64_t>(s.first + token) * args.q_stride +
                                                        (s.kv_head * group + row % group) * kHeadDim + lane * 4);
      x[0] = __uint_as_float(raw.x << 16);
      x[1] = __uint_as_float(raw.x & 0xffff0000u);
      x[2] = __uint_as_float(raw.y << 16);
      x[3] = __uint_as_float(raw.y & 0xffff0000u);
    }
    const float largest = warp_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
    const bool finite = __all_sync(0xffffffffu, fabsf(x[0]) < INFINITY && fabsf(x[1]) < INFINITY &&
                                                    fabsf(x[2]) < INFINITY && fabsf(x[3]) < INFINITY);
    // the largest element's exponent becomes 7: below 256
    const int power = largest > 0.0f && finite ? ilogbf(largest) - 7 : 0;
    uint32_t a[2], b[2];
    two_terms(scalbnf(x[0], -power), scalbnf(x[1], -power), a[0], b[0]);
    two_terms(scalbnf(x[2], -power), scalbnf(x[3], -power), a[1], b[1]);
    const int chunk = lane >> 2, inside = (lane & 3) * 4;
    *reinterpret_cast<uint32_t*>(q + r * 128 + ((chunk ^ (r & 7)) << 4) + inside) = a[0] | (a[1] << 16);
    const int r2 = S::kRows + r;
    *reinterpret_cast<uint32_t*>(q + r2 * 128 + ((chunk ^ (r2 & 7)) << 4) + inside) = b[0] | (b[1] << 16);
    if (lane == 0) {
      // (a row that is no number: its scores are none)
      c->factor[r] = finite ? scalbnf(args.scale * kLog2e, power) : NAN;
      c->limit[r] = s.length - s.rows + (valid ? token : 0);
      c->top[r] = -INFINITY;
      c->shift[r] = 0.0f;
    }
  }
}

// The values of a tile at the end of a sequence: places behind it hold anything and become 0; where a
// value that only some rows see is no number, it becomes 0 as well, and the rows that see it get it in
// the end (a weight of 0 times such a value would be none either).  A thread per token.
template <typename S>
__device__ __forceinline__ void clean_values(uint8_t* values, int token, int position, const Segment& s, Control<S>* c) {
  uint4* row = reinterpret_cast<uint4*>(values + token * kHeadDim);
  if (position >= s.length) {
    for (int i = 0; i < 8; ++i) row[i] = make_uint4(0, 0, 0, 0);
  } else if (position > s.length - s.rows) {
    for (int i = 0; i < 8; ++i) {
      const uint4 x = row[i];
      const uint32_t words[4] = {x.x, x.y, x.z, x.w};
      for (int w = 0; w < 4; ++w) {
        if ((((words[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) == 0) continue;
        for (int k = 0; k < 4; ++k) {
          if (((words[w] >> (8 * k)) & 0x7fu) != 0x7fu) continue;
          atomicMin(&c->first_bad[((i ^ (token & 7)) << 4) + 4 * w + k], position);
          reinterpret_cast<uint8_t*>(row + i)[4 * w + k] = 0;
        }
      }
    }
  }
  fence_proxy_async_smem();
}

// Where byte `column` (a multiple of 8) of a token's weights lies.
template <typename S>
__device__ __forceinline__ uint32_t weight_offset(int token, int column) {
  const int panel = column / S::kPanel, inside = column % S::kPanel;
  const uint32_t at = panel * kTile * S::kPanel + token * S::kPanel + inside;
  constexpr uint32_t mask = (S::kPanel / 16 - 1) << 4;
  return at ^ ((at >> 3) & mask);
}

template <typename S>
__device__ void join(const CachedArgs& args, const Split& split, const Segment& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = args.heads / args.cache.kv_heads;
  const int rows = min(S::kRows, s.rows * group - s.row0);
  auto part_of = [&](int p) {
    return split.parts + part_floats(S::kRows) * (p == 0 ? 2 * s.lead + 1 : 2 * (s.lead + p));
  };
  for (int r = warp; r < rows; r += S::kSoftmaxWarps) {
    float top = -INFINITY;
    for (int p = lane; p < s.parts; p += 32) top = fmaxf(top, __ldcg(part_of(p) + S::kRows * kHeadDim + r));
    top = warp_max(top);
    if (top == -INFINITY) top = 0.0f;
    float sum = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int start = 0; start < s.parts; start += 32) {
      float scale = 0.0f, weight = 0.0f;
      if (start + lane < s.parts) {
        const float* part = part_of(start + lane) + S::kRows * kHeadDim;
        scale = exp2_approx(__ldcg(part + r) - top);
        weight = __ldcg(part + S::kRows + r) * scale;
      }
      const int count = min(32, s.parts - start);
#pragma unroll 8
      for (int p = 0; p < count; ++p) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(part_of(start + p) + r * kHeadDim) + lane);
        const float f = __shfl_sync(0xffffffffu, scale, p);
        sum += __shfl_sync(0xffffffffu, weight, p);
        o[0] += x.x * f;
        o[1] += x.y * f;
        o[2] += x.z * f;
        o[3] += x.w * f;
      }
    }
    const float inverse = 1.0f / sum;
    const int row = s.row0 + r;
    const size_t at = (static_cast<size_t>(s.first + row / group) * args.heads + s.kv_head * group + row % group);
    *reinterpret_cast<uint2*>(args.out + at * kHeadDim + lane * 4) =
        make_uint2(pack_bf16(o[0] * inverse, o[1] * inverse), pack_bf16(o[2] * inverse, o[3] * inverse));
  }
}

template <typename S>
__device__ bool softmax_role(const CachedArgs& args, const Split& split, uint8_t* stages, uint8_t* q, uint8_t* weights,
                             uint32_t tmem, Control<S>* c) {
  constexpr int RG = S::kGroupRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = warp >> 2;
  const int token = threadIdx.x & (kTile - 1), r0 = group * RG;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
  const uint32_t o_at = lanes + S::kScores * S::kN + r0;
  const int page_shift = args.cache.page_shift;
  volatile int* failed = &c->failed[group];
  uint32_t tile_no = 0;
  for (uint32_t segments = 0;; ++segments) {
    const uint32_t place = segments & 1;
    bool ok = wait_warp(smem_u32(&c->segment_full[place]), (segments >> 1) & 1);
    const int some = ok && c->has_segment[place];
    const Segment s = c->segment[place];
    if (!ok) *failed = 1;
    softmax_sync<S>();
    if (c->failed[0] || c->failed[S::kGroups - 1]) return false;
    if (!some) return true;
    if (lane == 0) mbar_arrive(&c->segment_empty[place]);
    if (threadIdx.x < kHeadDim) c->first_bad[threadIdx.x] = INT32_MAX;
    prepare_queries<S>(args, s, q, c);
    fence_proxy_async_smem();
    softmax_sync<S>();
    if (lane == 0) mbar_arrive(&c->q_full);
    float sum[RG];
#pragma unroll
    for (int r = 0; r < RG; ++r) sum[r] = 0.0f;
    const int clear = s.length - s.rows;  // the last token that every row sees
    for (int j = 0; j < s.tiles; ++j, ++tile_no) {
      const uint32_t stage = tile_no % S::kStages, buffer = tile_no % S::kScores;
      const int first = (s.tile + j) * kTile, position = first + token;
      const bool at_end = first + kTile - 1 > clear;
      ok = wait_warp(smem_u32(&c->k_full[stage]), (tile_no / S::kStages) & 1);
      ok = wait_warp(smem_u32(&c->s_full[buffer]), (tile_no / S::kScores) & 1) && ok;
      tcgen05_fence_after();
      if (at_end) ok = wait_warp(smem_u32(&c->v_full[stage]), (tile_no / S::kStages) & 1) && ok;
      // (places behind the sequence may lie in pages that it does not have)
      const int page = token >> page_shift;
      const float k_scale = exp2_approx(static_cast<float>(position < s.length ? c->powers[stage][0][page] : 0));
      const float v_power = static_cast<float>(position < s.length ? c->powers[stage][1][page] : 0);
      float y[RG];
#pragma unroll
      for (int part = 0; part < RG; part += 32) {
        constexpr int kChunk = RG < 32 ? RG : 32;
        uint32_t a[kChunk], b[kChunk];
#pragma unroll
        for (int i = 0; i < kChunk; i += 8) {
          tmem_ld_x8_async(lanes + buffer * S::kN + r0 + part + i, a + i);
          tmem_ld_x8_async(lanes + buffer * S::kN + S::kRows + r0 + part + i, b + i);
        }
        tmem_ld_wait();
        registers_loaded<kChunk>(a);
        registers_loaded<kChunk>(b);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          const float product = fmaf(__uint_as_float(b[i]), 0.0625f, __uint_as_float(a[i]));
          y[part + i] = fmaf(product, c->factor[r0 + part + i] * k_scale, v_power);
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->s_empty[buffer]);
      if (at_end) {
#pragma unroll
        for (int r = 0; r < RG; ++r) {
          if (position > c->limit[r0 + r]) y[r] = -INFINITY;
        }
        if (group == 0) clean_values<S>(stages + (2 * stage + 1) * kTileBytes, token, position, s, c);
      }
      // the largest of each row, row r in lane r
      bool higher = false;
      float mine[(RG + 31) / 32];
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        const float largest = warp_max(y[r]);
        if (lane == (r & 31)) mine[r / 32] = largest;
      }
#pragma unroll
      for (int r = lane, i = 0; i < (RG + 31) / 32; r += 32, ++i) {
        if (r < RG) {
          c->warp_top[warp][r] = mine[i];
          higher = higher || mine[i] > c->top[r0 + r] + kSlack;
        }
      }
      // the weights of the tile before have been read, and O holds it
      ok = wait_warp(smem_u32(&c->p_empty), (tile_no & 1) ^ 1) && ok;
      tcgen05_fence_after();
      if (!ok) *failed = 1;
      const bool rise = group_any(group, higher);
      if (*failed) return false;
      if (rise) {
        if (token < RG) {
          const int r = r0 + token;
          float top = c->top[r];
          const float was = top;
#pragma unroll
          for (int w = 0; w < 4; ++w) top = fmaxf(top, c->warp_top[group * 4 + w][token]);
          c->fade[r] = was == -INFINITY ? 0.0f : exp2_approx(was - top);
          c->top[r] = top;
          c->shift[r] = top == -INFINITY ? 0.0f : kWeightBits - top;
        }
        group_sync(group);
        if (j > 0) {
#pragma unroll 1
          for (int i = 0; i < RG; i += 8) {
#pragma unroll
            for (int term = 0; term < 2; ++term) {
              uint32_t o[8];
              tmem_ld_x8_async(o_at + term * S::kRows + i, o);
              tmem_ld_wait();
              registers_loaded<8>(o);
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * c->fade[r0 + i + k]);
              tmem_st_x8(o_at + term * S::kRows + i, o);
            }
          }
          tmem_st_wait();
#pragma unroll
          for (int r = 0; r < RG; ++r) sum[r] *= c->fade[r0 + r];
        }
      }
      const float v_inverse = exp2_approx(-v_power);
#pragma unroll
      for (int i = 0; i < RG; i += 8) {
        uint32_t a[4], b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = i + 2 * k;
          const float p0 = exp2_approx(y[r] + c->shift[r0 + r]);
          const float p1 = exp2_approx(y[r + 1] + c->shift[r0 + r + 1]);
          sum[r] = fmaf(p0, v_inverse, sum[r]);
          sum[r + 1] = fmaf(p1, v_inverse, sum[r + 1]);
          two_terms(p0, p1, a[k], b[k]);
        }
        *reinterpret_cast<uint2*>(weights + weight_offset<S>(token, r0 + i)) =
            make_uint2(a[0] | (a[1] << 16), a[2] | (a[3] << 16));
        *reinterpret_cast<uint2*>(weights + weight_offset<S>(token, S::kRows + r0 + i)) =
            make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
      }
      fence_proxy_async_smem();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->p_full);
    }
    // the rows' sums of weights over the 128 threads, in a fixed order
#pragma unroll
    for (int r = 0; r < RG; ++r) {
      float x = sum[r];
#pragma unroll
      for (int step = 16; step > 0; step /= 2) x += __shfl_xor_sync(0xffffffffu, x, step);
      if (lane == 0) c->warp_sum[warp][r] = x;
    }
    ok = wait_warp(smem_u32(&c->p_empty), (tile_no & 1) ^ 1);
    tcgen05_fence_after();
    if (!ok) *failed = 1;
    group_sync(group);
    if (*failed) return false;
    if (token < RG) {
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) x += c->warp_sum[group * 4 + w][token];
      c->sum[r0 + token] = x;
    }
    group_sync(group);
    // a thread per dimension now
    const int heads_per = args.heads / args.cache.kv_heads;
    const int rows = min(RG, s.rows * heads_per - s.row0 - r0);
    float* part = s.part < 0 ? nullptr : split.parts + part_floats(S::kRows) * s.part;
    const int bad = c->first_bad[token];
#pragma unroll 1
    for (int i = 0; i < RG; i += 8) {
      uint32_t a[8], b[8];
      tmem_ld_x8_async(o_at + i, a);
      tmem_ld_x8_async(o_at + S::kRows + i, b);
      tmem_ld_wait();
      registers_loaded<8>(a);
      registers_loaded<8>(b);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (i + k >= rows) break;
        const int r = r0 + i + k, row = s.row0 + r;
        float o = fmaf(__uint_as_float(b[k]), 0.0625f, __uint_as_float(a[k]));
        if (c->limit[r] >= bad) o = NAN;
        if (part != nullptr) {
          __stcg(part + r * kHeadDim + token, o);
        } else {
          const size_t at = static_cast<size_t>(s.first + row / heads_per) * args.heads + s.kv_head * heads_per + row % heads_per;
          args.out[at * kHeadDim + token] = __float2bfloat16(o / c->sum[r]);
        }
      }
    }
    tcgen05_fence_before();
    if (part != nullptr) {
      if (token < RG) {
        __stcg(part + S::kRows * kHeadDim + r0 + token, c->top[r0 + token]);
        __stcg(part + S::kRows * (kHeadDim + 1) + r0 + token, c->sum[r0 + token]);
      }
      __threadfence();
      softmax_sync<S>();
      if (threadIdx.x == 0) c->last = atomicAdd(&split.counters[s.lead], 1) == s.parts - 1;
      softmax_sync<S>();
      if (c->last) {
        __threadfence();
        if (threadIdx.x == 0) split.counters[s.lead] = 0;
        join<S>(args, split, s);
      }
    }
  }
}

template <typename S>
__global__ void __launch_bounds__(S::kThreads, S::kBlocks)
    cached_kernel(const __grid_constant__ CUtensorMap map, const CachedArgs args, const Split split) {
  extern __shared__ uint8_t raw[];
  uint8_t* stages = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint8_t* q = stages + S::kStages * 2 * kTileBytes;
  uint8_t* weights = q + S::kN * kHeadDim;
  Control<S>* c = reinterpret_cast<Control<S>*>(weights + S::kN * kTile);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&c->k_full[i], 1);
      mbar_init(&c->k_empty[i], 1);
      mbar_init(&c->v_full[i], 1);
      mbar_init(&c->v_empty[i], 1);
    }
    for (int i = 0; i < S::kScores; ++i) {
      mbar_init(&c->s_full[i], 1);
      mbar_init(&c->s_empty[i], S::kSoftmaxWarps);
    }
    mbar_init(&c->p_full, S::kSoftmaxWarps);
    mbar_init(&c->p_empty, 1);
    mbar_init(&c->q_full, S::kSoftmaxWarps);
    mbar_init(&c->drained, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c->segment_full[i], 1);
      mbar_init(&c->segment_empty[i], S::kSoftmaxWarps + 1);
      c->failed[i] = 0;
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
  if (warp < S::kSoftmaxWarps) {
    if (!softmax_role<S>(args, split, stages, q, weights, tmem, c) && (threadIdx.x & 31) == 0) {
      report_cache_error(args.cache.error, kDevWaitTimeout);
    }
  } else if (warp == S::kSoftmaxWarps) {
    const bool ok = mma_role<S>(smem_u32(stages), smem_u32(q), smem_u32(weights), tmem, c);
    if (elect_one()) {
      if (!ok) report_cache_error(args.cache.error, kDevWaitTimeout);
      tcgen05_commit(&c->drained);
    }
    __syncwarp();
    wait_warp(smem_u32(&c->drained), 0);
  } else {
    load_role<S>(args, &map, smem_u32(stages), c);
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == S::kSoftmaxWarps) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, S::kColumns);
  }
}

constexpr size_t kCounterBytes = 4096;

template <typename S>
cudaError_t launch(const CUtensorMap& map, const CachedArgs& args, const Split& split, int sms, cudaStream_t stream) {
  cudaError_t err = allow_shared_memory(cached_kernel<S>);
  if (err != cudaSuccess) return err;
  cached_kernel<S><<<sms * S::kBlocks, S::kThreads, shared_bytes<S>(), stream>>>(map, args, split);
  return cudaGetLastError();
}

}  // namespace

size_t attention_cached_workspace_bytes() {
  // two parts to a block, as many rows on an SM whatever the shape
  return kCounterBytes + sizeof(float) * part_floats(kMaxRows) * 2 * device_sms();
}

cudaError_t launch_attention_cached(const CachedArgs& args, cudaStream_t stream) {
  const int sms = device_sms();
  if (sms * 2 * sizeof(int) > kCounterBytes) return cudaErrorInvalidValue;
  CUtensorMap map;
  if (!pages_tensor_map(args.cache, &map)) return cudaErrorInvalidValue;
  const Split split{reinterpret_cast<int*>(args.cache.attend_workspace),
                    reinterpret_cast<float*>(args.cache.attend_workspace + kCounterBytes)};
  // as many query rows at a time as the entries have on average, up to 128: further rows of an entry
  // read its keys and values again
  const int64_t rows = (args.batch.rows + args.batch.count - 1) / args.batch.count *
                       static_cast<int64_t>(args.heads / args.cache.kv_heads);
  if (rows <= 8) return launch<Shape<8, 1>>(map, args, split, sms, stream);
  if (rows <= 16) return launch<Shape<16, 1>>(map, args, split, sms, stream);
  if (rows <= 32) return launch<Shape<32, 1>>(map, args, split, sms, stream);
  if (rows <= 64) return launch<Shape<64, 1>>(map, args, split, sms, stream);
  return launch<Shape<128, 2>>(map, args, split, sms, stream);
}

}  // namespace nmoe
