// Attention over the 8-bit cache for a batch in groups whose sequences hold the same first pages (continuations of a
// prompt, forked), and how many tokens these are.
//
// A row's softmax over all tokens is joined from that over the shared ones and that over its own: with the reference
// r, the sum of weights l and the weighted sum of values o of each piece,
//   r = max r_i,   o = sum_i 2^(r_i - r) o_i / sum_i 2^(r_i - r) l_i
// The shared tokens are attended by all rows of a group at once: their codes are read once for up to 128 rows of
// queries instead of once for every sequence, and it is the tensor cores' and the exponentials' rate that bounds it
// where groups are large, not the memory's.
//
// What bounds the other pieces is waiting: the sequences' own tokens (64 of 200 tokens, 8 key heads, 18 us) are a chain
// of loads as in attention_cached.cuh, and so is the join, list - RowPart - places - sums, each from L2 (64 rows of 32
// heads in 20 pieces 13 us with its launch; 532 rows 15).
//
// Three launches: the groups' shared tokens, the sequences' own ones (the kernels of attention_cached.cuh, which leave
// sums instead of results), and the join, a warp to a row and head.  The second does not wait for the first, but its blocks
// only find room where one of the first's has left: the call takes about the three's times one after another.
//
// So attention_cached.cu's single launch is faster where little is shared.  Both from a recorded graph, caches in memory, 32
// query heads, 60 tokens of their own, in us (some 6 of each are the graph's): 8 sequences sharing 1024, 8 key heads 22
// by that, 31 by this; 64 sharing 1024 37, 43; 8 sharing 16384 45, 47; 64 sharing 4096 70, 53; 64 sharing 16384 205, 65; 2
// key heads: 64 sharing 4096 41, 51; 64 sharing 16384 82, 60.  They are equal at about 250 MB of codes that are
// not read again.
#include <algorithm>

#include "attention.h"
#include "attention_cached.cuh"
#include "kernels.h"

namespace nmoe {
namespace {

constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;
constexpr int kFindThreads = 512;

struct JoinArgs {
  CachedArgs cached;           // with the group's lists
  const RowPart* of_row[2];    // what sequences share, their own
  const float* sums[2];
  const float* slots[2];
  int slot_rows[2];
  int blocks[2];               // that have slots
};

// The group that entry i belongs to, -1 for none; all lanes of a warp call it with the same i.
__device__ __forceinline__ int group_of(const int* groups, int count, int i, int lane) {
  int found = -1;
  for (int start = 0; start <= count; start += 32) {  // (rising: the last that begins at or before i)
    const int g = start + lane;
    const unsigned begun = __ballot_sync(0xffffffffu, g <= count && groups[g] <= i);
    if (begun == 0) break;
    found = start + 31 - __clz(begun);
  }
  return found < count ? found : -1;
}

// A block to (an entry, some of its rows and heads).
__global__ void __launch_bounds__(kJoinThreads) join_parts_kernel(const JoinArgs args) {
  const CachedArgs& c = args.cached;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.x;
  // (what these read was there before the first of the three launches)
  const BatchEntry e = part_entry<Part::kOwn>(c, i);
  if (e.rows == 0) {  // (nor does this launch end ahead of the others where no entry has rows: they may write zeros)
    wait_for_predecessor();
    return;
  }
  bool valid = true;
  if (e.skip > 0) {
    const int g = group_of(c.groups, c.group_count, i, lane);
    valid = g >= 0;
    if (valid) {
      const BatchEntry group = group_entry(c, g);
      valid = group.valid && group.length == e.skip && e.first >= group.first && e.first + e.rows <= group.first + group.rows;
    }
    if (!valid && threadIdx.x == 0 && blockIdx.y == 0) report_cache_error(c.cache.raised, kCacheBadSequence);
  }
  wait_for_predecessor();
  release_successor();
  const int pairs = e.rows * c.heads;
  const CacheWords words = cache_words(c.cache);
#pragma unroll 1
  for (int p = blockIdx.y * kJoinWarps + warp; p < pairs; p += gridDim.y * kJoinWarps) {
    const size_t at = static_cast<size_t>(e.first) * c.heads + p;
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, top = -INFINITY, sum = 0.0f;
    RowPart part[2];
    part[0].parts_row = 0;
    if (e.skip > 0) part[0] = args.of_row[0][at];
    part[1] = args.of_row[1][at];
    int count[2];
    bool there = valid && words.error == 0;  // (where a wait ran out, there may be nothing, either)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      count[k] = part[k].parts_row > 255 ? part[k].parts_row >> 8 : part[k].parts_row;
      there = there && count[k] >= 0 && (count[k] < 2 || (part[k].lead >= 0 && part[k].lead <= args.blocks[k] - count[k] &&
                                                          (part[k].parts_row & 255) < args.slot_rows[k]));
    }
    if (there) {
      const int all = count[0] + count[1];
#pragma unroll 1
      for (int start = 0; start < all; start += 32) {  // a lane to a piece
        float reference = -INFINITY, weight = 0.0f;
        const float* from = nullptr;
        if (start + lane < all) {
          const int k = start + lane >= count[0], piece = start + lane - (k ? count[0] : 0);
          const RowPart& r = part[k];
          if (r.parts_row == 1) {
            reference = r.reference;
            weight = r.sum;
            from = args.sums[k] + at * kHeadDim;
          } else {
            const int rows = args.slot_rows[k], row = r.parts_row & 255;
            const float* slot = args.slots[k] + slot_floats(rows) * (kSlotsPerBlock * (r.lead + piece) + (piece == 0));
            reference = __ldcg(slot + rows * kHeadDim + row);
            weight = __ldcg(slot + rows * (kHeadDim + 1) + row);
            from = slot + row * kHeadDim;
          }
        }
        float higher = reference;
#pragma unroll
        for (int step = 16; step > 0; step /= 2) higher = fmaxf(higher, __shfl_xor_sync(0xffffffffu, higher, step));
        higher = fmaxf(higher, top);
        const float keep = top > -INFINITY ? exp2_approx(top - higher) : 0.0f;
        const float scale = reference > -INFINITY ? exp2_approx(reference - higher) : 0.0f;
        top = higher;
        sum *= keep;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] *= keep;
        const int some = min(all - start, 32);
#pragma unroll 16
        for (int j = 0; j < some; ++j) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(__shfl_sync(
                                      0xffffffffu, reinterpret_cast<unsigned long long>(from), j))) +
                                  lane);
          const float f = __shfl_sync(0xffffffffu, scale, j), w = __shfl_sync(0xffffffffu, weight, j);
          sum = fmaf(w, f, sum);
          o[0] = fmaf(x.x, f, o[0]);
          o[1] = fmaf(x.y, f, o[1]);
          o[2] = fmaf(x.z, f, o[2]);
          o[3] = fmaf(x.w, f, o[3]);
        }
      }
    }
    const float inverse = there ? 1.0f / sum : 0.0f;
    *reinterpret_cast<uint2*>(c.out + at * kHeadDim + lane * 4) =
        make_uint2(pack_bf16(o[0] * inverse, o[1] * inverse), pack_bf16(o[2] * inverse, o[3] * inverse));
  }
}

// A block to a group (and one for the entries of none): the first page in which a member differs from the first member
// with rows, and the fewest tokens that one holds before its new rows.
__global__ void __launch_bounds__(kFindThreads) find_shared_kernel(PagedCache c, Batch b, const int* groups, int group_count, int* shared) {
  __shared__ int common, fewest, members, leader, wrong;
  wait_for_predecessor();
  release_successor();
  const int g = blockIdx.x;
  const int first = min(max(groups[0], 0), b.count), last = min(max(groups[group_count], first), b.count);
  if (g == group_count) {
    for (int i = threadIdx.x; i < b.count - (last - first); i += kFindThreads) shared[i < first ? i : i + last - first] = 0;
    return;
  }
  // (lists that do not rise: what lies between the ends is written by its blocks or not at all)
  const int from = min(max(groups[g], first), last), to = min(max(groups[g + 1], from), last);
  if (threadIdx.x == 0) {
    common = c.max_pages;
    fewest = INT32_MAX;
    members = wrong = 0;
    leader = INT32_MAX;
    if (groups[g] < 0 || groups[g + 1] < groups[g] || groups[g + 1] > b.count) wrong = 1;
  }
  __syncthreads();
  for (int i = from + threadIdx.x; i < to; i += kFindThreads) {
    const BatchEntry e = batch_entry(c, b, i);
    if (!e.valid) {
      wrong = 1;
    } else if (e.rows > 0) {
      atomicMin(&leader, i);
      atomicAdd(&members, 1);
      atomicMin(&fewest, e.length - e.rows);
    }
  }
  __syncthreads();
  int tokens = 0;
  if (wrong == 0 && members >= 2) {
    const int pages = min(fewest >> c.page_shift, c.max_pages);
    const int* own = c.table + static_cast<size_t>(b.sequences[leader]) * c.max_pages;
    // a warp to a member at a time, its pages side by side
    const int lane = threadIdx.x & 31;
    for (int i = from + (threadIdx.x >> 5); i < to; i += kFindThreads / 32) {
      if (i == leader || b.offsets[i + 1] == b.offsets[i]) continue;
      const int* other = c.table + static_cast<size_t>(b.sequences[i]) * c.max_pages;
      for (int start = 0; start < min(pages, *const_cast<volatile int*>(&common)); start += 128) {
        int differs = INT32_MAX;
#pragma unroll
        for (int k = 3; k >= 0; --k) {
          const int page = start + 32 * k + lane;
          if (page < pages && own[page] != other[page]) differs = page;
        }
        differs = __reduce_min_sync(0xffffffffu, differs);
        if (differs < pages) {
          if (lane == 0) atomicMin(&common, differs);
          break;
        }
      }
    }
    __syncthreads();
    tokens = (min(common, pages) << c.page_shift) / kKeyTile * kKeyTile;
    tokens = min(tokens, fewest / kKeyTile * kKeyTile);
  }
  if (wrong != 0 && threadIdx.x == 0) report_cache_error(c.raised, kCacheBadSequence);
  for (int i = from + threadIdx.x; i < to; i += kFindThreads) shared[i] = tokens;
}

constexpr size_t kAlign = 256;
size_t aligned(size_t bytes) { return (bytes + kAlign - 1) / kAlign * kAlign; }

// Sums and places of both parts, and the pieces of each.
struct Workspace {
  size_t places, sums, queries, slots[2], total;
  Workspace(int64_t rows, int heads) {
    const size_t pairs = static_cast<size_t>(rows) * heads;
    places = aligned(pairs * sizeof(RowPart));
    sums = aligned(pairs * kHeadDim * sizeof(float));
    queries = 2 * places + 2 * sums;
    slots[0] = queries + aligned(shared_pairs_query_bytes(rows, heads));
    slots[1] = slots[0] + aligned(std::max(shared_pairs_slot_bytes(), attention_cached_slot_bytes()));
    total = slots[1] + attention_cached_slot_bytes();
  }
};

}  // namespace

size_t attention_shared_workspace_bytes(int64_t rows, int heads) { return Workspace(rows, heads).total; }

// The second launch begins when all blocks of the first run.  These have waited for what came before, so everything that
// the second reads (it reads nothing of the first's) is there; it ends behind the first, so that the join has both.
cudaError_t launch_attention_shared(const CachedArgs& args, char* workspace, cudaStream_t stream) {
  const Workspace w(args.batch.rows, args.heads);
  const int64_t of_head = args.heads / args.cache.kv_heads;
  JoinArgs join;
  join.cached = args;
  CachedArgs part = args;
  const int64_t entries[2] = {args.group_count, args.batch.count};
  for (int k = 0; k < 2; ++k) {
    part.row_parts = reinterpret_cast<RowPart*>(workspace + k * w.places);
    part.sums = reinterpret_cast<float*>(workspace + 2 * w.places + k * w.sums);
    float* slots = reinterpret_cast<float*>(workspace + w.slots[k]);
    const int64_t rows = (args.batch.rows + entries[k] - 1) / entries[k] * of_head;
    join.of_row[k] = part.row_parts;
    join.sums[k] = part.sums;
    join.slots[k] = slots;
    // (4 groups of 8192 tokens, 8 key heads: 96 rows 79 us with pairs of tiles, 81 without; 144 rows 93, 112; 256 rows 123,
    // 140.  Up to kMaxRows a group's queries fit into the other kernel's one tile, which needs no launch ahead.)
    const bool pairs = k == 0 && rows > kMaxRows && shared_pairs_supported(args.batch.rows, args.heads);
    join.slot_rows[k] = pairs ? shared_pairs_slot_rows() : attention_cached_slot_rows(rows);
    join.blocks[k] = device_sms() * (join.slot_rows[k] <= 16 ? 2 : 1);
    const cudaError_t err = pairs ? launch_shared_pairs(part, slots, workspace + w.queries, stream)
                                  : launch_cached_part(part, k ? Part::kOwn : Part::kShared, rows, slots, stream);
    if (err != cudaSuccess) return err;
  }
  // a pair to a warp
  const int64_t pairs = (args.batch.rows + args.batch.count - 1) / args.batch.count * args.heads;
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((pairs + kJoinWarps - 1) / kJoinWarps, 4096));
  return launch_kernel(join_parts_kernel, dim3(args.batch.count, blocks), kJoinThreads, 0, LaunchStream(stream, true), join);
}

cudaError_t launch_kv_find_shared(const PagedCache& cache, const Batch& batch, const int* groups, int group_count, int* shared,
                                  cudaStream_t stream) {
  return launch_kernel(find_shared_kernel, dim3(group_count + 1), kFindThreads, 0, LaunchStream(stream, true), cache, batch, groups,
                       group_count, shared);
}

}  // namespace nmoe
