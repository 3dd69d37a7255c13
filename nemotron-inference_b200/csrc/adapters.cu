// Low-rank adapters of many requests beside a projection that they share: with the adapter of a row's request
//   out = y + scale (x A^T) B^T,   A [rank, inner], B [outer, rank]
//
// What bounds it is memory: x and y are read and out is written once, A and B of the adapters in use; a row costs
// 2 rank (inner + outer) operations, some tens to a byte.  Two launches:
//   inside   t = x A^T for a tile of rows of one request, the tensor cores taking A as the operand of 128 rows (the
//            ranks; those behind the rank are whatever lies there and their results are not read) and the rows of x as the
//            other, of 128 too, of which only the rows that there are get read: a tile of 16 was no faster for few rows
//            and slower from 12 on.  The contraction is cut into parts where tiles are few; each leaves FP32 sums.
//   outside  out = y + (scale t) B^T, a block to an SM with an even share of all tiles of 128 rows and 128 columns, y and B
//            on their way tiles ahead.  t, summed up in a fixed order, is two bf16 terms (within 2^-17 of it; as one it
//            would be off by 2^-9, of the size of what y's own rounding leaves), both multiplied with the same tile of B
//            into one sum; y is added in FP32 and the result rounded once.  Rows without an adapter are copied.
// Measured (B200, calls one after another): 23 requests of 356 rows, 2688 to 4608, rank 32, 44 us (4.0 TB/s); 64 of 4 rows,
// 4096 to 2688, rank 64, 25 us (1.6 TB/s: a block's first tiles are on their way for 5 us, in each launch, and a piece
// begins with t); one row 10.5 us in a graph, 17 called.
#include <algorithm>

#include "attention.h"
#include "attention_mma.cuh"
#include "common.cuh"
#include "kernels.h"
#include "serving.h"

namespace nmoe {
namespace {

constexpr int kTile = 128;
constexpr int kChunk = 64;  // columns of x and A at a time: rows of 128 bytes
constexpr int kMostSplits = 16;
constexpr int kMostStages = 8;
constexpr int kInsideThreads = 192;
constexpr uint32_t kPanelBytes = kTile * 128;  // 128 rows of 64 bf16

// A tile of rows of one entry.
struct RowsTile {
  int first, rows, adapter;  // adapter -1: none; rows 0: no such tile
};

struct Found {
  int before[32];
  RowsTile tile;
};

// All threads: tile `u` of the entries' tiles of rows.
__device__ RowsTile find_tile(const AdapterArgs& args, int u, Found* f) {
  const int threads = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (args.count + threads - 1) / threads;
  const int begin = min(static_cast<int>(threadIdx.x) * each, args.count), end = min(begin + each, args.count);
  auto tiles_of = [&](int i, int& from) {
    from = args.offsets[i];
    const int to = args.offsets[i + 1];
    return from >= 0 && from <= to && to <= args.rows ? (to - from + kTile - 1) / kTile : 0;
  };
  if (threadIdx.x == 0) f->tile = {0, 0, -1};
  int mine = 0, from;
  for (int i = begin; i < end; ++i) mine += tiles_of(i, from);
  int upto = mine;
#pragma unroll
  for (int step = 1; step < 32; step *= 2) {
    const int other = __shfl_up_sync(0xffffffffu, upto, step);
    if (lane >= step) upto += other;
  }
  if (lane == 31) f->before[warp] = upto;
  __syncthreads();
  int at = upto - mine;
  for (int w = 0; w < warp; ++w) at += f->before[w];
  if (u >= at && u < at + mine) {  // one thread's
    for (int i = begin; i < end; ++i) {
      const int tiles = tiles_of(i, from);
      if (u < at + tiles) {
        const int skip = (u - at) * kTile, id = args.ids[i];
        f->tile = {from + skip, min(args.offsets[i + 1] - from - skip, kTile),
                   static_cast<unsigned>(id) < static_cast<unsigned>(args.adapters) ? id : -1};
        break;
      }
      at += tiles;
    }
  }
  __syncthreads();
  return f->tile;
}

// Entries and ids that are none.
__device__ void report_entries(const AdapterArgs& args) {
  for (int i = threadIdx.x; i < args.count; i += blockDim.x) {
    const int from = args.offsets[i], to = args.offsets[i + 1], id = args.ids[i];
    if (from < 0 || to < from || to > args.rows || id < -1 || id >= args.adapters) report_cache_error(args.error, kCacheBadSequence);
  }
}

struct InsideControl {
  uint64_t full[kMostStages], empty[kMostStages], done;
  uint32_t tmem;
  Found found;
};

__global__ void __launch_bounds__(kInsideThreads)
    inside_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const AdapterArgs args,
                  int chunks_each, int stages) {
  extern __shared__ uint8_t raw[];
  InsideControl* c = reinterpret_cast<InsideControl*>(raw);
  uint8_t* ring = raw + sizeof(InsideControl);
  ring += (1024 - (smem_u32(ring) & 1023)) & 1023;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMostStages; ++i) {
      mbar_init(&c->full[i], 1);
      mbar_init(&c->empty[i], 1);
    }
    mbar_init(&c->done, 1);
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(&c->tmem, kTile);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  wait_for_predecessor();
  const RowsTile t = find_tile(args, blockIdx.x, &c->found);
  release_successor();  // (the columns of TMEM are there)
  tcgen05_fence_after();
  if (blockIdx.x == 0 && blockIdx.y == 0) report_entries(args);
  const uint32_t tmem = c->tmem;
  const int chunks = (args.inner + kChunk - 1) / kChunk, from = blockIdx.y * chunks_each;
  const int count = t.rows > 0 && t.adapter >= 0 ? min(chunks_each, chunks - from) : 0;
  const uint32_t a_bytes = args.rank * 128, stage_bytes = a_bytes + kTile * 128;
  const int boxes = (t.rows + 7) / 8;
  if (warp == 4) {
    bool ok = true;
    int i = 0;
    for (; i < count && ok; ++i) {
      const int stage = i % stages;
      ok = mbar_wait_warp(smem_u32(&c->empty[stage]), ((i / stages) & 1) ^ 1);
      if (ok && elect_one()) {
        const uint32_t bar = smem_u32(&c->full[stage]), to = smem_u32(ring) + stage * stage_bytes;
        mbar_arrive_expect_tx_at(bar, a_bytes + boxes * 1024);
        tma_load_2d_at(to, &map_a, (from + i) * kChunk, t.adapter * args.rank, bar);
        for (int k = 0; k < boxes; ++k) tma_load_2d_at(to + a_bytes + k * 1024, &map_x, (from + i) * kChunk, t.first + 8 * k, bar);
      }
      __syncwarp();
    }
    if (!ok) {  // what is in flight arrives before the block's shared memory is given up
      if (lane == 0) report_cache_error(args.error, kDevWaitTimeout);
      for (int back = max(0, i - 1 - stages); back < i - 1; ++back) {
        mbar_wait_warp(smem_u32(&c->full[back % stages]), (back / stages) & 1);
      }
    }
  } else if (warp == 5) {
    constexpr uint32_t kDesc = make_idesc_bf16(kTile, false);
    bool ok = true;
    for (int i = 0; i < count && ok; ++i) {
      const int stage = i % stages;
      ok = mbar_wait_warp(smem_u32(&c->full[stage]), (i / stages) & 1);
      tcgen05_fence_after();
      if (ok && elect_one()) {
        const uint32_t at = smem_u32(ring) + stage * stage_bytes;
        const uint64_t a_desc = make_smem_desc(at, 16, 1024, 2), x_desc = make_smem_desc(at + a_bytes, 16, 1024, 2);
#pragma unroll
        for (int k = 0; k < kChunk / 16; ++k) {
          mma_f16_ss(tmem, advance_smem_desc(a_desc, k * 32), advance_smem_desc(x_desc, k * 32), kDesc, i > 0 || k > 0);
        }
        tcgen05_commit(&c->empty[stage]);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) report_cache_error(args.error, kDevWaitTimeout);
    if (elect_one()) tcgen05_commit(&c->done);
    __syncwarp();
  }
  // a warp per 32 of the ranks; sums of a row side by side
  const bool ok = mbar_wait_warp(smem_u32(&c->done), 0);
  tcgen05_fence_after();
  const int rank = warp * 32 + lane;
  if (warp < 4 && warp * 32 < args.rank && count > 0 && ok) {
    float* to = args.inside + (static_cast<size_t>(blockIdx.y) * args.rows + t.first) * args.rank + rank;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp) << 21);
    for (int r = 0; r < t.rows; r += 16) {
      uint32_t v[16];
      tmem_ld_x16_async(lanes + r, v);
      tmem_ld_wait();
      registers_loaded<16>(v);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        if (rank < args.rank && r + k < t.rows) __stcg(to + static_cast<size_t>(r + k) * args.rank, __uint_as_float(v[k]));
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 5) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, kTile);
  }
}

// Rows of one entry that a block works on, and their tiles of columns.
struct Piece {
  int first, rows, adapter;  // adapter -1: none
  int from, to;              // tiles of columns
};

constexpr int kPieces = 4;  // known ahead
constexpr int kMostOutsideStages = 3;
constexpr int kSumWarps = 8, kTermWarps = 4;
constexpr int kLoadWarp = kSumWarps, kMmaWarp = kSumWarps + 1, kFirstTermWarp = kSumWarps + 2;
constexpr int kOutsideThreads = 32 * (kSumWarps + 2 + kTermWarps);
constexpr uint32_t kTileBytes = 2 * kPanelBytes;  // 128 rows of 128 columns of y

struct OutsideControl {
  uint64_t piece_full[kPieces], piece_empty[kPieces];
  uint64_t y_full[kMostOutsideStages], y_empty[kMostOutsideStages], b_full[kMostOutsideStages], b_empty[kMostOutsideStages];
  uint64_t d_full[2], d_empty[2], t_full[2], t_empty[2], drained;
  Piece piece[kPieces];
  int some[kPieces];
  uint32_t tmem;
  int before[32];
  int64_t begin, end;        // this block's tiles, in order of the rows
  int entry;                 // the entry in which they begin, and the first tile of its
  int64_t entry_begin;
};

// Stages of a block's shared memory, by the panels of 64 ranks.
struct OutsideLayout {
  int panels, stages, terms;  // stages of y and B, buffers of t
  __host__ __device__ explicit OutsideLayout(int rank) : panels((rank + kChunk - 1) / kChunk), stages(panels > 1 ? 2 : 3), terms(panels > 1 ? 1 : 2) {}
  __host__ __device__ uint32_t b_bytes() const { return panels * kPanelBytes; }
  __host__ __device__ uint32_t t_bytes() const { return 2 * panels * kPanelBytes; }
  __host__ __device__ uint32_t total() const { return stages * (kTileBytes + b_bytes()) + terms * t_bytes(); }
};

// 16 bytes of y and sums of eight columns.
__device__ __forceinline__ uint4 add_eight(const uint4& y, const uint32_t* d) {
  const uint32_t w[4] = {y.x, y.y, y.z, y.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[i] = pack_bf16(__uint_as_float(w[i] << 16) + __uint_as_float(d[2 * i]),
                     __uint_as_float(w[i] & 0xffff0000u) + __uint_as_float(d[2 * i + 1]));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Entry i, empty where its offsets do not rise within the rows.
__device__ __forceinline__ Piece entry_of(const AdapterArgs& args, int i) {
  Piece p;
  const int from = args.offsets[i], to = args.offsets[i + 1], id = args.ids[i];
  p.first = from;
  p.rows = from >= 0 && from <= to && to <= args.rows ? to - from : 0;
  p.adapter = static_cast<unsigned>(id) < static_cast<unsigned>(args.adapters) ? id : -1;
  p.from = p.to = 0;
  return p;
}

// All threads: this block's share of all tiles of 128 rows and columns.
__device__ void find_share(const AdapterArgs& args, int columns, OutsideControl* c) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (args.count + kOutsideThreads - 1) / kOutsideThreads;
  const int begin = min(static_cast<int>(threadIdx.x) * each, args.count), end = min(begin + each, args.count);
  int mine = 0;
#pragma unroll 4
  for (int i = begin; i < end; ++i) mine += (entry_of(args, i).rows + kTile - 1) / kTile;
  int upto = mine;
#pragma unroll
  for (int step = 1; step < 32; step *= 2) {
    const int other = __shfl_up_sync(0xffffffffu, upto, step);
    if (lane >= step) upto += other;
  }
  if (lane == 31) c->before[warp] = upto;
  __syncthreads();
  int at = upto - mine, total = 0;
  for (int w = 0; w < kOutsideThreads / 32; ++w) {
    if (w < warp) at += c->before[w];
    total += c->before[w];
  }
  const int64_t all = static_cast<int64_t>(total) * columns;
  const int64_t from = all * blockIdx.x / gridDim.x, to = all * (blockIdx.x + 1) / gridDim.x;
  if (threadIdx.x == 0) {
    c->begin = from;
    c->end = to;
  }
  if (from < to && from >= static_cast<int64_t>(at) * columns && from < static_cast<int64_t>(at + mine) * columns) {  // one thread's
    for (int i = begin; i < end; ++i) {
      const int tiles = (entry_of(args, i).rows + kTile - 1) / kTile;
      if (from < static_cast<int64_t>(at + tiles) * columns) {
        c->entry = i;
        c->entry_begin = static_cast<int64_t>(at) * columns;
        break;
      }
      at += tiles;
    }
  }
  __syncthreads();
}

// The warp that finds the block's pieces, and brings in y and B.
__device__ bool load_role(const AdapterArgs& args, const CUtensorMap* y_rows, const CUtensorMap* y_few, const CUtensorMap* b_map, uint32_t y_at,
                          uint32_t b_at, const OutsideLayout& layout, int columns, OutsideControl* c) {
  const int lane = threadIdx.x & 31;
  const bool in_place = args.out == args.y;
  uint32_t pieces = 0, units = 0, adapted = 0;
  int64_t at = c->begin;
  const int64_t stop = c->end;
  int64_t entry_at = c->entry_begin;
  bool ok = true;
#pragma unroll 1
  for (int i = c->entry; at < stop && i < args.count; ++i) {
    const Piece e = entry_of(args, i);
    const int row_tiles = (e.rows + kTile - 1) / kTile;
#pragma unroll 1
    for (int tile = static_cast<int>((at - entry_at) / columns); tile < row_tiles && at < stop; ++tile) {
      const int64_t tile_at = entry_at + static_cast<int64_t>(tile) * columns;
      Piece p;
      p.first = e.first + tile * kTile;
      p.rows = min(e.rows - tile * kTile, kTile);
      p.adapter = e.adapter;
      p.from = static_cast<int>(at - tile_at);
      p.to = static_cast<int>(min(stop - tile_at, static_cast<int64_t>(columns)));
      at = tile_at + p.to;
      if (in_place && p.adapter < 0) continue;  // (these stay)
      const uint32_t place = pieces % kPieces;
      if (!mbar_wait_warp(smem_u32(&c->piece_empty[place]), ((pieces / kPieces) & 1) ^ 1)) return false;
      if (lane == 0) {
        c->piece[place] = p;
        c->some[place] = 1;
        mbar_arrive(&c->piece_full[place]);
      }
      __syncwarp();
      ++pieces;
      const int boxes = p.rows > kTile / 2 ? 1 : (p.rows + 7) / 8;  // of 128 rows, or of 8
      const uint32_t bytes = boxes == 1 && p.rows > 8 ? kTileBytes : boxes * 2048;
#pragma unroll 1
      for (int column = p.from; column < p.to; ++column, ++units) {
        const uint32_t stage = units % layout.stages, y_bar = smem_u32(&c->y_full[stage]), to = y_at + stage * kTileBytes;
        if (!mbar_wait_warp(smem_u32(&c->y_empty[stage]), ((units / layout.stages) & 1) ^ 1)) return false;
        if (elect_one()) {
          fence_proxy_async_smem();  // (here: in the warps that add up it would wait for their stores to memory)
          mbar_arrive_expect_tx_at(y_bar, bytes);
          for (int half = 0; half < 2; ++half) {
            if (bytes == kTileBytes) {
              tma_load_2d_at(to + half * kPanelBytes, y_rows, column * kTile + half * 64, p.first, y_bar);
            } else {
              for (int k = 0; k < boxes; ++k) {
                tma_load_2d_at(to + half * kPanelBytes + k * 1024, y_few, column * kTile + half * 64, p.first + 8 * k, y_bar);
              }
            }
          }
        }
        __syncwarp();
        if (p.adapter < 0) continue;
        const uint32_t b_stage = adapted % layout.stages, b_bar = smem_u32(&c->b_full[b_stage]);
        if (!mbar_wait_warp(smem_u32(&c->b_empty[b_stage]), ((adapted / layout.stages) & 1) ^ 1)) return false;
        if (elect_one()) {
          mbar_arrive_expect_tx_at(b_bar, layout.b_bytes());
          for (int k = 0; k < layout.panels; ++k) {
            tma_load_2d_at(b_at + b_stage * layout.b_bytes() + k * kPanelBytes, b_map, k * kChunk, p.adapter * args.outer + column * kTile,
                           b_bar);
          }
        }
        __syncwarp();
        ++adapted;
      }
    }
    entry_at += static_cast<int64_t>(row_tiles) * columns;
  }
  const uint32_t place = pieces % kPieces;
  if (!mbar_wait_warp(smem_u32(&c->piece_empty[place]), ((pieces / kPieces) & 1) ^ 1)) return false;
  if (lane == 0) {
    c->some[place] = 0;
    mbar_arrive(&c->piece_full[place]);
  }
  return ok;
}

// The next piece; false behind the last. `ok` falls where the wait runs out.
__device__ __forceinline__ bool next_piece(OutsideControl* c, uint32_t pieces, Piece& p, bool& ok) {
  const uint32_t place = pieces % kPieces;
  ok = mbar_wait_warp(smem_u32(&c->piece_full[place]), (pieces / kPieces) & 1);
  if (!ok || !c->some[place]) return false;
  p = c->piece[place];
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&c->piece_empty[place]);
  return true;
}

__device__ bool mma_role(uint32_t t_at, uint32_t b_at, uint32_t tmem, const OutsideLayout& layout, int rank, OutsideControl* c) {
  constexpr uint32_t kDesc = make_idesc_bf16(kTile, false);
  const int steps = (rank + 15) / 16;
  uint32_t adapted = 0, records = 0;
  bool ok;
  Piece p;
#pragma unroll 1
  for (uint32_t pieces = 0; next_piece(c, pieces, p, ok); ++pieces) {
    if (p.adapter < 0) continue;
    const uint32_t buffer_t = records % layout.terms;
    if (!mbar_wait_warp(smem_u32(&c->t_full[buffer_t]), (records / layout.terms) & 1)) return false;
    const uint64_t t_desc = make_smem_desc(t_at + buffer_t * layout.t_bytes(), 16, 1024, 2);
#pragma unroll 1
    for (int column = p.from; column < p.to; ++column, ++adapted) {
      const uint32_t stage = adapted % layout.stages, buffer = adapted & 1;
      if (!mbar_wait_warp(smem_u32(&c->b_full[stage]), (adapted / layout.stages) & 1)) return false;
      if (!mbar_wait_warp(smem_u32(&c->d_empty[buffer]), ((adapted >> 1) & 1) ^ 1)) return false;
      tcgen05_fence_after();
      if (elect_one()) {
        const uint64_t b_desc = make_smem_desc(b_at + stage * layout.b_bytes(), 16, 1024, 2);
        for (int term = 0; term < 2; ++term) {
          for (int k = 0; k < steps; ++k) {
            const uint32_t at = k / 4 * kPanelBytes + k % 4 * 32;
            mma_f16_ss(tmem + buffer * kTile, advance_smem_desc(t_desc, term * layout.b_bytes() + at), advance_smem_desc(b_desc, at), kDesc,
                       term > 0 || k > 0);
          }
        }
        tcgen05_commit(&c->d_full[buffer]);
        tcgen05_commit(&c->b_empty[stage]);
        if (column + 1 == p.to) tcgen05_commit(&c->t_empty[buffer_t]);
      }
      __syncwarp();
    }
    ++records;
  }
  return ok;
}

// Four warps that sum up t and put it into shared memory as two bf16 terms.
__device__ bool term_role(const AdapterArgs& args, uint8_t* terms, const OutsideLayout& layout, int splits, OutsideControl* c) {
  const int thread = threadIdx.x - 32 * kFirstTermWarp;
  const int eights = (args.rank + 15) / 16 * 2;  // of ranks, filled up to whole steps of an MMA
  const size_t split = static_cast<size_t>(args.rows) * args.rank;
  uint32_t records = 0;
  bool ok;
  Piece p;
#pragma unroll 1
  for (uint32_t pieces = 0; next_piece(c, pieces, p, ok); ++pieces) {
    if (p.adapter < 0) continue;
    if (records == 0) wait_for_predecessor();  // (the first launch; all else was there before that)
    const uint32_t buffer = records % layout.terms;
    if (!mbar_wait_warp(smem_u32(&c->t_empty[buffer]), ((records / layout.terms) & 1) ^ 1)) return false;
    const float scale = args.scales[p.adapter];
    const float* inside = args.inside + static_cast<size_t>(p.first) * args.rank;
    const int all = p.rows * eights;
    constexpr int kAtOnce = 2, kSplitsAtOnce = 4;  // (their loads wait side by side)
#pragma unroll 1
    for (int start = thread; start < all; start += kAtOnce * 32 * kTermWarps) {
      float v[kAtOnce][8];
#pragma unroll
      for (int m = 0; m < kAtOnce; ++m) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[m][k] = 0.0f;
      }
#pragma unroll 1
      for (int s = 0; s < splits; s += kSplitsAtOnce) {
        float4 part[kAtOnce][kSplitsAtOnce][2];
#pragma unroll
        for (int m = 0; m < kAtOnce; ++m) {
          const int i = start + m * 32 * kTermWarps, row = i / eights, eight = i - row * eights;
          const float4* from = reinterpret_cast<const float4*>(inside + s * split + static_cast<size_t>(row) * args.rank + eight * 8);
#pragma unroll
          for (int j = 0; j < kSplitsAtOnce; ++j) {
            part[m][j][0] = part[m][j][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i < all && eight * 8 < args.rank && s + j < splits) {
              part[m][j][0] = __ldcg(from);
              part[m][j][1] = __ldcg(from + 1);
            }
            from = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(from) + split);
          }
        }
#pragma unroll
        for (int m = 0; m < kAtOnce; ++m) {
#pragma unroll
          for (int j = 0; j < kSplitsAtOnce; ++j) {
            const float4 lo = part[m][j][0], hi = part[m][j][1];
            v[m][0] += lo.x, v[m][1] += lo.y, v[m][2] += lo.z, v[m][3] += lo.w;
            v[m][4] += hi.x, v[m][5] += hi.y, v[m][6] += hi.z, v[m][7] += hi.w;
          }
        }
      }
#pragma unroll
      for (int m = 0; m < kAtOnce; ++m) {
        const int i = start + m * 32 * kTermWarps, row = i / eights, eight = i - row * eights;
        if (i >= all) break;
        uint32_t first[4], second[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x = v[m][2 * k] * scale, z = v[m][2 * k + 1] * scale;
          first[k] = pack_bf16(x, z);
          const float x1 = __uint_as_float(first[k] << 16), z1 = __uint_as_float(first[k] & 0xffff0000u);
          // (nothing is left of what has become infinite)
          second[k] = pack_bf16(fabsf(x1) < INFINITY ? x - x1 : 0.0f, fabsf(z1) < INFINITY ? z - z1 : 0.0f);
        }
        uint8_t* to = terms + buffer * layout.t_bytes() + (eight >> 3) * kPanelBytes + row * 128 + (((eight & 7) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4*>(to) = make_uint4(first[0], first[1], first[2], first[3]);
        *reinterpret_cast<uint4*>(to + layout.b_bytes()) = make_uint4(second[0], second[1], second[2], second[3]);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&c->t_full[buffer]);
    ++records;
  }
  return ok;
}

// Eight warps that add up: a thread to a row and half of a tile's columns, whose results go over y's in shared memory
// and from there, by the same warp, to memory, whole lines at a time.
__device__ bool sum_role(const AdapterArgs& args, uint8_t* y, uint32_t tmem, const OutsideLayout& layout, OutsideControl* c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = (warp & 3) * 32, row = row0 + lane, half = warp >> 2;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21) + half * 64;
  uint32_t units = 0, adapted = 0;
  bool ok;
  Piece p;
#pragma unroll 1
  for (uint32_t pieces = 0; next_piece(c, pieces, p, ok); ++pieces) {
    const bool some = row0 < p.rows, with = p.adapter >= 0;
    __nv_bfloat16* out = args.out + static_cast<int64_t>(p.first) * args.out_stride;
#pragma unroll 1
    for (int column = p.from; column < p.to; ++column, ++units) {
      const uint32_t stage = units % layout.stages, buffer = adapted & 1;
      uint8_t* tile = y + stage * kTileBytes + half * kPanelBytes;
      if (!mbar_wait_warp(smem_u32(&c->y_full[stage]), (units / layout.stages) & 1)) return false;
      if (with) {
        uint4 own[8];  // (all before the first is written: the compiler does not know that they lie apart)
        auto at = [&](int k) { return reinterpret_cast<uint4*>(tile + row * 128 + ((k ^ (row & 7)) << 4)); };
        if (some) {
#pragma unroll
          for (int k = 0; k < 8; ++k) own[k] = *at(k);
        }
        if (!mbar_wait_warp(smem_u32(&c->d_full[buffer]), (adapted >> 1) & 1)) return false;
        tcgen05_fence_after();
        if (some) {
#pragma unroll
          for (int k = 0; k < 8; k += 4) {
            uint32_t d[32];
            tmem_ld_x32_async(lanes + buffer * kTile + k * 8, d);
            tmem_ld_wait();
            registers_loaded<32>(d);
#pragma unroll
            for (int j = 0; j < 4; ++j) *at(k + j) = add_eight(own[k + j], d + 8 * j);
          }
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&c->d_empty[buffer]);
        ++adapted;
      }
      uint4 line[8];
      if (some) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = row0 + k * 4 + (lane >> 3);
          line[k] = *reinterpret_cast<const uint4*>(tile + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->y_empty[stage]);
      if (some) {
        const int at = column * kTile + half * 64 + (lane & 7) * 8;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = row0 + k * 4 + (lane >> 3);
          if (r < p.rows && at < args.outer) *reinterpret_cast<uint4*>(out + r * args.out_stride + at) = line[k];
        }
      }
    }
  }
  return ok;
}

// A block to an SM, each with its share of the tiles of 128 rows and columns.
__global__ void __launch_bounds__(kOutsideThreads, 1)
    outside_kernel(const __grid_constant__ CUtensorMap y_rows, const __grid_constant__ CUtensorMap y_few,
                   const __grid_constant__ CUtensorMap b_map, const AdapterArgs args, int splits) {
  extern __shared__ uint8_t raw[];
  OutsideControl* c = reinterpret_cast<OutsideControl*>(raw);
  const OutsideLayout layout(args.rank);
  uint8_t* y = raw + sizeof(OutsideControl);
  y += (1024 - (smem_u32(y) & 1023)) & 1023;
  uint8_t* b = y + layout.stages * kTileBytes;
  uint8_t* terms = b + layout.stages * layout.b_bytes();
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPieces; ++i) {
      mbar_init(&c->piece_full[i], 1);
      mbar_init(&c->piece_empty[i], kSumWarps + 1 + kTermWarps);
    }
    for (int i = 0; i < kMostOutsideStages; ++i) {
      mbar_init(&c->y_full[i], 1);
      mbar_init(&c->y_empty[i], kSumWarps);
      mbar_init(&c->b_full[i], 1);
      mbar_init(&c->b_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c->d_full[i], 1);
      mbar_init(&c->d_empty[i], kSumWarps);
      mbar_init(&c->t_full[i], kTermWarps);
      mbar_init(&c->t_empty[i], 1);
    }
    mbar_init(&c->drained, 1);
    c->entry = 0;
    c->entry_begin = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&c->tmem, 2 * kTile);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  const int columns = (args.outer + kTile - 1) / kTile;
  // (the lists, y and B were there before the first launch, whose blocks have all waited for that when this one's begin)
  find_share(args, columns, c);
  release_successor();  // (the columns of TMEM are there)
  tcgen05_fence_after();
  const uint32_t tmem = c->tmem;
  bool ok;
  if (warp < kSumWarps) {
    ok = sum_role(args, y, tmem, layout, c);
  } else if (warp == kLoadWarp) {
    ok = load_role(args, &y_rows, &y_few, &b_map, smem_u32(y), smem_u32(b), layout, columns, c);
  } else if (warp == kMmaWarp) {
    ok = mma_role(smem_u32(terms), smem_u32(b), tmem, layout, args.rank, c);
    if (elect_one()) tcgen05_commit(&c->drained);
    __syncwarp();
    mbar_wait_warp(smem_u32(&c->drained), 0);
  } else {
    ok = term_role(args, terms, layout, splits, c);
  }
  if (!ok && (threadIdx.x & 31) == 0) report_cache_error(args.error, kDevWaitTimeout);
  wait_for_predecessor();  // (this launch ends behind the first)
  tcgen05_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, 2 * kTile);
  }
}

// How a call is cut.
struct Plan {
  int tiles;        // of rows, at most
  int chunks_each, splits, stages;
  size_t inside_shared;

  Plan(int64_t rows, int count, int inner, int rank, int sms) {
    tiles = static_cast<int>(std::min<int64_t>(rows, rows / kTile + count));
    // Two blocks to an SM, so that one's results go out while the other reads (4096 x 4096, rank 16: 64 entries of 4 rows
    // 32 us, of 30 rows 38, 23 of 356 50; with four blocks' parts 36, 40, 56, with one 46, - and 60).
    const int chunks = (inner + kChunk - 1) / kChunk;
    splits = std::clamp(2 * sms / tiles, 1, std::min(kMostSplits, std::max(chunks / 3, 1)));
    chunks_each = (chunks + splits - 1) / splits;
    splits = (chunks + chunks_each - 1) / chunks_each;
    const size_t stage = static_cast<size_t>(rank + kTile) * 128;
    stages = static_cast<int>(std::min<size_t>(std::min(kMostStages, chunks_each), 92 * 1024 / stage));
    inside_shared = sizeof(InsideControl) + 1024 + stages * stage + kPanelBytes;  // (128 rows are read of the last A, too)
  }
};

}  // namespace

size_t adapter_workspace_bytes(int64_t rows, int count, int inner, int rank) {
  return sizeof(float) * static_cast<size_t>(Plan(rows, count, inner, rank, device_sms()).splits) * rows * rank;
}

cudaError_t launch_adapters(const AdapterArgs& args, cudaStream_t stream) {
  const int sms = device_sms();
  const Plan plan(args.rows, args.count, args.inner, args.rank, sms);
  CUtensorMap map_x, map_a, map_b, y_rows, y_few;
  if (!matrix_tensor_map(args.x, args.rows, args.inner, args.x_stride, 8, &map_x) ||
      !matrix_tensor_map(args.a, static_cast<int64_t>(args.adapters) * args.rank, args.inner, args.inner, args.rank, &map_a) ||
      !matrix_tensor_map(args.b, static_cast<int64_t>(args.adapters) * args.outer, args.rank, args.rank, kTile, &map_b) ||
      !matrix_tensor_map(args.y, args.rows, args.outer, args.y_stride, kTile, &y_rows) ||
      !matrix_tensor_map(args.y, args.rows, args.outer, args.y_stride, 8, &y_few)) {
    return cudaErrorInvalidValue;
  }
  static std::atomic<uint64_t> allowed[2];
  cudaError_t err = allow_shared_memory_once(inside_kernel, allowed[0]);
  if (err == cudaSuccess) err = allow_shared_memory_once(outside_kernel, allowed[1]);
  if (err != cudaSuccess) return err;
  err = launch_kernel(inside_kernel, dim3(plan.tiles, plan.splits), kInsideThreads, plan.inside_shared, LaunchStream(stream, true), map_x,
                      map_a, args, plan.chunks_each, plan.stages);
  if (err != cudaSuccess) return err;
  const size_t shared = sizeof(OutsideControl) + 1024 + OutsideLayout(args.rank).total();
  return launch_kernel(outside_kernel, dim3(sms), kOutsideThreads, shared, LaunchStream(stream, true), y_rows, y_few, map_b, args,
                       plan.splits);
}

}  // namespace nmoe
