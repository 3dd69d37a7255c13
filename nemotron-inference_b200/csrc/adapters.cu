// Low-rank adapters of many requests beside a projection that they share: with the adapter of a row's request
//   out = y + scale (x A^T) B^T,   A [rank, inner], B [outer, rank]
//
// What bounds it is memory: x and y are read and out is written once, A and B of the adapters in use; a row costs
// 2 rank (inner + outer) operations, some tens to a byte.  Two launches:
//   inside   t = x A^T for a tile of rows of one request, the tensor cores taking A as the operand of 128 rows (the
//            ranks; those behind the rank are whatever lies there and their results are not read) and the rows of x as the
//            one of 16 or 128, so that a single token costs no more than its own bytes.  The contraction is cut
//            into parts where tiles are few; each leaves FP32 sums.
//   outside  out = y + (scale t) B^T for a tile of 128 rows and 128 columns at a time.  t, summed up in a fixed order,
//            is two bf16 terms (within 2^-17 of it; as one it would be off by 2^-9, of the size of what y's own rounding
//            leaves), both multiplied with the same tile of B into one sum; y is added in FP32 and the result rounded
//            once.  Rows without an adapter are copied.
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
constexpr int kInsideThreads = 192, kOutsideThreads = 320;
constexpr int kOutsideStages = 3;
constexpr uint32_t kPanelBytes = kTile * 128;  // 128 rows of 64 bf16

// A tile of rows of one entry.
struct RowsTile {
  int first, rows, adapter;  // adapter -1: none; rows 0: no such tile
};

struct Found {
  int before[32];
  RowsTile tile;
};

// All threads: tile `u` of the entries' tiles of `height` rows.
__device__ RowsTile find_tile(const AdapterArgs& args, int u, int height, Found* f) {
  const int threads = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (args.count + threads - 1) / threads;
  const int begin = min(static_cast<int>(threadIdx.x) * each, args.count), end = min(begin + each, args.count);
  auto tiles_of = [&](int i, int& from) {
    from = args.offsets[i];
    const int to = args.offsets[i + 1];
    return from >= 0 && from <= to && to <= args.rows ? (to - from + height - 1) / height : 0;
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
        const int skip = (u - at) * height, id = args.ids[i];
        f->tile = {from + skip, min(args.offsets[i + 1] - from - skip, height),
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

template <int N>
__global__ void __launch_bounds__(kInsideThreads)
    inside_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const AdapterArgs args,
                  int chunks_each, int stages) {
  extern __shared__ uint8_t raw[];
  InsideControl* c = reinterpret_cast<InsideControl*>(raw);
  uint8_t* ring = raw + sizeof(InsideControl);
  ring += (1024 - (smem_u32(ring) & 1023)) & 1023;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kColumns = N < 32 ? 32 : N;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMostStages; ++i) {
      mbar_init(&c->full[i], 1);
      mbar_init(&c->empty[i], 1);
    }
    mbar_init(&c->done, 1);
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(&c->tmem, kColumns);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  wait_for_predecessor();
  const RowsTile t = find_tile(args, blockIdx.x, N, &c->found);
  release_successor();  // (the columns of TMEM are there)
  tcgen05_fence_after();
  if (blockIdx.x == 0 && blockIdx.y == 0) report_entries(args);
  const uint32_t tmem = c->tmem;
  const int chunks = (args.inner + kChunk - 1) / kChunk, from = blockIdx.y * chunks_each;
  const int count = t.rows > 0 && t.adapter >= 0 ? min(chunks_each, chunks - from) : 0;
  const uint32_t a_bytes = args.rank * 128, stage_bytes = a_bytes + N * 128;
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
    constexpr uint32_t kDesc = make_idesc_bf16(N, false);
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
    tmem_dealloc(tmem, kColumns);
  }
}

struct OutsideControl {
  uint64_t full[kOutsideStages], empty[kOutsideStages], d_full[2], d_empty[2], t_full, drained;
  uint32_t tmem;
  Found found;
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

// blockIdx.y: `tiles_each` tiles of columns.
__global__ void __launch_bounds__(kOutsideThreads, 2)
    outside_kernel(const __grid_constant__ CUtensorMap map_b, const AdapterArgs args, int splits, int tiles_each) {
  extern __shared__ uint8_t raw[];
  OutsideControl* c = reinterpret_cast<OutsideControl*>(raw);
  const int panels = (args.rank + kChunk - 1) / kChunk;
  uint8_t* terms = raw + sizeof(OutsideControl);  // of t: first terms, second terms, `panels` panels each
  terms += (1024 - (smem_u32(terms) & 1023)) & 1023;
  uint8_t* ring = terms + 2 * panels * kPanelBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kOutsideStages; ++i) {
      mbar_init(&c->full[i], 1);
      mbar_init(&c->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c->d_full[i], 1);
      mbar_init(&c->d_empty[i], 8);
    }
    mbar_init(&c->t_full, 8);
    mbar_init(&c->drained, 1);
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(&c->tmem, 2 * kTile);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  wait_for_predecessor();
  const RowsTile t = find_tile(args, blockIdx.x, kTile, &c->found);
  release_successor();  // (the columns of TMEM are there)
  tcgen05_fence_after();
  const uint32_t tmem = c->tmem;
  const int all = (args.outer + kTile - 1) / kTile, from = blockIdx.y * tiles_each;
  const int count = t.rows > 0 ? min(tiles_each, all - from) : 0;
  const bool adapted = t.adapter >= 0;
  const int steps = (args.rank + 15) / 16;
  const uint32_t stage_bytes = panels * kPanelBytes;
  if (warp == 8) {
    bool ok = true;
    int i = 0;
    for (; adapted && i < count && ok; ++i) {
      const int stage = i % kOutsideStages;
      ok = mbar_wait_warp(smem_u32(&c->empty[stage]), ((i / kOutsideStages) & 1) ^ 1);
      if (ok && elect_one()) {
        const uint32_t bar = smem_u32(&c->full[stage]), to = smem_u32(ring) + stage * stage_bytes;
        mbar_arrive_expect_tx_at(bar, stage_bytes);
        for (int p = 0; p < panels; ++p) {
          tma_load_2d_at(to + p * kPanelBytes, &map_b, p * kChunk, t.adapter * args.outer + (from + i) * kTile, bar);
        }
      }
      __syncwarp();
    }
    if (!ok) {  // what is in flight arrives before the block's shared memory is given up
      if (lane == 0) report_cache_error(args.error, kDevWaitTimeout);
      for (int back = max(0, i - 1 - kOutsideStages); back < i - 1; ++back) {
        mbar_wait_warp(smem_u32(&c->full[back % kOutsideStages]), (back / kOutsideStages) & 1);
      }
    }
  } else if (warp == 9) {
    constexpr uint32_t kDesc = make_idesc_bf16(kTile, false);
    bool ok = !adapted || count <= 0 || mbar_wait_warp(smem_u32(&c->t_full), 0);
    for (int i = 0; adapted && i < count && ok; ++i) {
      const int stage = i % kOutsideStages, buffer = i & 1;
      ok = mbar_wait_warp(smem_u32(&c->full[stage]), (i / kOutsideStages) & 1);
      ok = ok && mbar_wait_warp(smem_u32(&c->d_empty[buffer]), ((i >> 1) & 1) ^ 1);
      tcgen05_fence_after();
      if (ok && elect_one()) {
        const uint64_t t_desc = make_smem_desc(smem_u32(terms), 16, 1024, 2);
        const uint64_t b_desc = make_smem_desc(smem_u32(ring) + stage * stage_bytes, 16, 1024, 2);
        for (int term = 0; term < 2; ++term) {
          for (int k = 0; k < steps; ++k) {
            const uint32_t at = k / 4 * kPanelBytes + k % 4 * 32;
            mma_f16_ss(tmem + buffer * kTile, advance_smem_desc(t_desc, term * panels * kPanelBytes + at), advance_smem_desc(b_desc, at),
                       kDesc, term > 0 || k > 0);
          }
        }
        tcgen05_commit(&c->d_full[buffer]);
        tcgen05_commit(&c->empty[stage]);
      }
      __syncwarp();
    }
    if (elect_one()) {
      if (!ok) report_cache_error(args.error, kDevWaitTimeout);
      tcgen05_commit(&c->drained);
    }
    __syncwarp();
    mbar_wait_warp(smem_u32(&c->drained), 0);
  } else if (count > 0) {
    // a thread to a row, and to half of a tile's columns
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;
    const bool valid = row < t.rows;
    const __nv_bfloat16* y = args.y + static_cast<int64_t>(t.first + row) * args.y_stride;
    __nv_bfloat16* out = args.out + static_cast<int64_t>(t.first + row) * args.out_stride;
    if (adapted) {
      if (valid) {
        const float scale = args.scales[t.adapter];
        const float* inside = args.inside + static_cast<size_t>(t.first + row) * args.rank;
        const size_t split = static_cast<size_t>(args.rows) * args.rank;
        for (int chunk = half; chunk < 2 * steps; chunk += 2) {  // of eight ranks
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.0f;
          if (chunk * 8 < args.rank) {
            for (int s = 0; s < splits; ++s) {
              const float4 lo = __ldcg(reinterpret_cast<const float4*>(inside + s * split + chunk * 8));
              const float4 hi = __ldcg(reinterpret_cast<const float4*>(inside + s * split + chunk * 8) + 1);
              v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
              v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
            }
          }
          uint32_t first[4], second[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = v[2 * i] * scale, q = v[2 * i + 1] * scale;
            first[i] = pack_bf16(p, q);
            const float p1 = __uint_as_float(first[i] << 16), q1 = __uint_as_float(first[i] & 0xffff0000u);
            // (nothing is left of what has become infinite)
            second[i] = pack_bf16(fabsf(p1) < INFINITY ? p - p1 : 0.0f, fabsf(q1) < INFINITY ? q - q1 : 0.0f);
          }
          uint8_t* to = terms + (chunk >> 3) * kPanelBytes + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
          *reinterpret_cast<uint4*>(to) = make_uint4(first[0], first[1], first[2], first[3]);
          *reinterpret_cast<uint4*>(to + panels * kPanelBytes) = make_uint4(second[0], second[1], second[2], second[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->t_full);
    }
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21) + half * 64;
    bool ok = true;
    for (int i = 0; i < count && ok; ++i) {
      const int buffer = i & 1, column = (from + i) * kTile + half * 64;
      uint4 had[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (valid && column + k * 8 < args.outer) had[k] = *reinterpret_cast<const uint4*>(y + column + k * 8);
      }
      if (!adapted) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (valid && column + k * 8 < args.outer) *reinterpret_cast<uint4*>(out + column + k * 8) = had[k];
        }
        continue;
      }
      ok = mbar_wait_warp(smem_u32(&c->d_full[buffer]), (i >> 1) & 1);
      tcgen05_fence_after();
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        uint32_t d[16];
        tmem_ld_x16_async(lanes + buffer * kTile + k * 8, d);
        tmem_ld_wait();
        registers_loaded<16>(d);
        if (!valid || !ok) continue;
        if (column + k * 8 < args.outer) *reinterpret_cast<uint4*>(out + column + k * 8) = add_eight(had[k], d);
        if (column + k * 8 + 8 < args.outer) *reinterpret_cast<uint4*>(out + column + k * 8 + 8) = add_eight(had[k + 1], d + 8);
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->d_empty[buffer]);
    }
    if (!ok && lane == 0) report_cache_error(args.error, kDevWaitTimeout);
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 9) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, 2 * kTile);
  }
}

// How a call is cut.
struct Plan {
  int height;       // rows of a tile of the first launch
  int tiles[2];     // of both launches, at most
  int chunks_each, splits, stages;
  size_t inside_shared;

  Plan(int64_t rows, int count, int inner, int rank, int sms) {
    // A tile of 16 rows holds its sums in fewer columns and less shared memory; one of 128 reads A once for more rows.
    height = rows <= 16 * static_cast<int64_t>(count) ? 16 : kTile;
    for (int k = 0; k < 2; ++k) {
      const int h = k ? kTile : height;
      tiles[k] = static_cast<int>(std::min<int64_t>(rows, rows / h + count));
    }
    const int chunks = (inner + kChunk - 1) / kChunk;
    splits = std::clamp(2 * sms / std::max(tiles[0], 1), 1, std::min(kMostSplits, std::max(chunks / 3, 1)));
    chunks_each = (chunks + splits - 1) / splits;
    splits = (chunks + chunks_each - 1) / chunks_each;
    const size_t stage = static_cast<size_t>(rank + height) * 128;
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
  CUtensorMap map_x, map_a, map_b;
  if (!matrix_tensor_map(args.x, args.rows, args.inner, args.x_stride, 8, &map_x) ||
      !matrix_tensor_map(args.a, static_cast<int64_t>(args.adapters) * args.rank, args.inner, args.inner, args.rank, &map_a) ||
      !matrix_tensor_map(args.b, static_cast<int64_t>(args.adapters) * args.outer, args.rank, args.rank, kTile, &map_b)) {
    return cudaErrorInvalidValue;
  }
  static std::atomic<uint64_t> allowed[3];
  cudaError_t err = allow_shared_memory_once(inside_kernel<16>, allowed[0]);
  if (err == cudaSuccess) err = allow_shared_memory_once(inside_kernel<kTile>, allowed[1]);
  if (err == cudaSuccess) err = allow_shared_memory_once(outside_kernel, allowed[2]);
  if (err != cudaSuccess) return err;
  auto* inside = plan.height == 16 ? inside_kernel<16> : inside_kernel<kTile>;
  err = launch_kernel(inside, dim3(plan.tiles[0], plan.splits), kInsideThreads, plan.inside_shared, LaunchStream(stream, true), map_x,
                      map_a, args, plan.chunks_each, plan.stages);
  if (err != cudaSuccess) return err;
  const int all = (args.outer + kTile - 1) / kTile;
  const int groups = std::clamp(4 * sms / plan.tiles[1], 1, all), tiles_each = (all + groups - 1) / groups;
  const int panels = (args.rank + kChunk - 1) / kChunk;
  const size_t shared = sizeof(OutsideControl) + 1024 + (2 + kOutsideStages) * static_cast<size_t>(panels) * kPanelBytes;
  return launch_kernel(outside_kernel, dim3(plan.tiles[1], (all + tiles_each - 1) / tiles_each), kOutsideThreads, shared,
                       LaunchStream(stream, true), map_b, args, plan.splits, tiles_each);
}

}  // namespace nmoe
