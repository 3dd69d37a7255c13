// The paged 8-bit cache of keys and values: new rows are quantised into it, its pages are handed out,
// shared, copied, moved and given back.  Everything is decided on the device: a step launches these
// kernels without reading a length or a free page on the host, and can be recorded once and replayed.
#include <cuda_fp16.h>

#include <algorithm>

#include "attention.h"
#include "common.cuh"
#include "kernels.h"

namespace nmoe {
namespace {

// ---------------------------------------------------------------------------
// New rows
// ---------------------------------------------------------------------------

// The least e with amax <= 448 * 2^e (448 = 1.75 * 2^8).
__device__ __forceinline__ int exponent_for(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int power = static_cast<int>(bits >> 23) - 127;
  const int e = power - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return min(max(e, kMinExponent), kMaxExponent);
}

__device__ __forceinline__ float power_of_two(int e) {
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Two values to two codes; values beyond the range saturate, NaN becomes NaN.
__device__ __forceinline__ uint32_t encode_two(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float2 decode_two(uint32_t codes) {
  const __half2_raw h =
      __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

constexpr int kAppendThreads = 256;
constexpr int kAppendBlocks = 6;  // on an SM

// The largest 16-bit half of all threads' words; `parts` is not in use by another call.
__device__ __forceinline__ uint32_t block_max(uint32_t two, uint32_t* parts) {
  __syncthreads();  // (the parts of the call before are read)
  const uint32_t mine = __reduce_max_sync(0xffffffffu, max(two & 0xffffu, two >> 16));
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = mine;
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < kAppendThreads / 32; ++w) all = max(all, parts[w]);
  return all;
}

// Magnitudes of two bf16, 0 for an infinity or NaN.
__device__ __forceinline__ uint32_t finite_only(uint32_t two) {
  const uint32_t lo = two & 0x7fffu, hi = two & 0x7fff0000u;
  return (lo < 0x7f80u ? lo : 0u) | (hi < 0x7f800000u ? hi : 0u);
}

// A block per page that gets new rows and `per_block` of its heads' keys and values.  A page and head's new
// values stay in registers between the maximum that gives the exponent and their rounding, so they are read
// once; finding the page is a chain of loads, which the heads share where there are blocks enough.
// A page that held tokens may get a larger exponent: its older codes are rounded again then, which
// is exact but for values that fall among the subnormal codes.
// 8190 rows of 23 sequences and 8 heads: 18 us for 49 MB, 0.4 of the copy rate: each block's chain (error word,
// entry, length, page, exponent) is some 5 us and the loads' own latency comes once for each head; the issue slots
// are busy in 40 % of the cycles.  64 rows: 7.4 us, the chain and a launch.
template <int PageTokens>
__global__ void __launch_bounds__(kAppendThreads, PageTokens <= 64 ? kAppendBlocks : 4)
    kv_append_kernel(PagedCache c, Batch b, int layer, const __nv_bfloat16* k, int64_t k_stride,
                     const __nv_bfloat16* v, int64_t v_stride, int per_block) {
  constexpr int kAppendChunks = PageTokens * kHeadDim / 8 / kAppendThreads;  // of 8 values, to a thread
  __shared__ uint32_t warp_max[2][kAppendThreads / 32];
  release_successor();
  wait_for_predecessor();
  const int pending = *c.error;
  const int2 unit = locate_unit(b.count, blockIdx.x, [&](int i) {
    const BatchEntry e = batch_entry(c, b, i);
    if (!e.valid) report_cache_error(c.raised, kCacheBadSequence);
    if (e.rows == 0) return 0;
    return ((e.length - 1) >> c.page_shift) - ((e.length - e.rows) >> c.page_shift) + 1;
  });
  // (after a reservation that failed these rows have no place of their own; no block of an append writes this word,
  // so all of them see the same)
  if (pending != 0 || unit.x < 0) return;
  const BatchEntry e = batch_entry(c, b, unit.x);
  const int place = ((e.length - e.rows) >> c.page_shift) + unit.y;
  const int begin = max(e.length - e.rows, place << c.page_shift);  // positions in the sequence
  const int end = min(e.length, (place + 1) << c.page_shift);
  const int held = begin & (c.page_tokens - 1);
  const int last = min(static_cast<int>(blockIdx.y + 1) * per_block, 2 * c.kv_heads);
  const int chunks = (end - begin) * (kHeadDim / 8), first_row = e.first + begin - (e.length - e.rows);
  auto read = [&](int of, uint4(&raw)[kAppendChunks]) {
    const int64_t stride = of & 1 ? v_stride : k_stride;
    const __nv_bfloat16* from = (of & 1 ? v : k) + (of >> 1) * kHeadDim + first_row * stride;
#pragma unroll
    for (int i = 0; i < kAppendChunks; ++i) {
      const int chunk = i * kAppendThreads + threadIdx.x;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (chunk < chunks) raw[i] = *reinterpret_cast<const uint4*>(from + (chunk / 16) * stride + (chunk % 16) * 8);
    }
  };
  uint4 raw[kAppendChunks];
  read(blockIdx.y * per_block, raw);  // (under way while the page is looked up)
  const int page = page_at(c, e.sequence, place);
  if (page < 0) {
    report_cache_error(c.raised, kCacheBadSequence);
    return;
  }
#pragma unroll 1
  for (int of = blockIdx.y * per_block; of < last; ++of) {
    const size_t block = block_of_page(c, layer, page, of & 1, of >> 1);
    uint8_t* codes = c.codes + block * c.page_tokens * kHeadDim;
    const int before = held > 0 ? c.exponents[block] : 0;
    // magnitudes as whole numbers, two at a time; those of infinities and NaN are beyond all others
    uint32_t two_max = 0;
#pragma unroll
    for (int i = 0; i < kAppendChunks; ++i) {
      const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int w = 0; w < 4; ++w) two_max = __vmaxu2(two_max, words[w] & 0x7fff7fffu);
    }
    uint32_t largest = block_max(two_max, warp_max[0]);
    const bool special = largest >= 0x7f80u;
    if (special) {
      two_max = 0;
#pragma unroll
      for (int i = 0; i < kAppendChunks; ++i) {
        const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int w = 0; w < 4; ++w) two_max = __vmaxu2(two_max, finite_only(words[w]));
      }
      largest = block_max(two_max, warp_max[1]);
    }
    const float amax = __uint_as_float(largest << 16);
    int after = exponent_for(amax);
    if (held > 0) after = max(after, before);
    if (threadIdx.x == 0) c.exponents[block] = static_cast<int8_t>(after);
    if (held > 0 && after > before) {
      const float lower = power_of_two(before - after);
      uint4* older = reinterpret_cast<uint4*>(codes);
      for (int i = threadIdx.x; i < held * (kHeadDim / 16); i += kAppendThreads) {
        uint4 x = older[i];
        uint32_t* words = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 a = decode_two(words[w]), z = decode_two(words[w] >> 16);
          words[w] = encode_two(a.x * lower, a.y * lower) | (encode_two(z.x * lower, z.y * lower) << 16);
        }
        older[i] = x;
      }
    }
    const uint64_t factor2 = pack2(power_of_two(-after), power_of_two(-after));
#pragma unroll
    for (int i = 0; i < kAppendChunks; ++i) {
      const int chunk = i * kAppendThreads + threadIdx.x;
      if (chunk < chunks) {
        const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t two[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float lo, hi;
          unpack2(mul2(pack2(__uint_as_float(words[w] << 16), __uint_as_float(words[w] & 0xffff0000u)), factor2), lo, hi);
          if (special) {  // an infinity is not hidden behind the largest code
            if ((words[w] & 0x7f80u) == 0x7f80u) lo = NAN;
            if ((words[w] & 0x7f800000u) == 0x7f800000u) hi = NAN;
          }
          two[w] = encode_two(lo, hi);
        }
        *reinterpret_cast<uint2*>(codes + held * kHeadDim + chunk * 8) =
            make_uint2(two[0] | (two[1] << 16), two[2] | (two[3] << 16));
      }
    }
    if (of + 1 < last) read(of + 1, raw);
  }
}

// ---------------------------------------------------------------------------
// Pages.  One block keeps the books: lists are short, and every decision (which free page goes to
// whom) follows from a sum over those before.  What they take, some 10 us in a compaction, is their chain of loads.
// ---------------------------------------------------------------------------

constexpr int kBookThreads = 1024;

struct BookShared {
  int warp_sums[kBookThreads / 32];
  int flag;
  int list[kBookThreads];  // pages
};

// Asks for a word that a later step of the books reads: they are chains of loads, some 0.6 us each.
__device__ __forceinline__ void ask_for(const int* p) {
  asm volatile("{\n\t.reg .b32 unused;\n\tld.global.b32 unused, [%0];\n\t}" ::"l"(p));
}

// Whether the books stay as they are.  What follows (an append of rows for which no room was made) does nothing
// either, even if it was an append that found something wrong: so that goes where appends and attention look.
__device__ __forceinline__ bool books_closed(const PagedCache& c, const CacheWords& words) {
  if (words.pending() && threadIdx.x == 0) report_cache_error(c.error, words.raised);
  return words.pending();
}

// For the lists' sequences: their lengths.  (Counts of references and claims are not asked for ahead: they change
// by atomics.)
__device__ __forceinline__ void ask_for_lengths(const PagedCache& c, const int* sequences, int count) {
  if (static_cast<int>(threadIdx.x) >= count) return;
  const int sequence = sequences[threadIdx.x];
  if (static_cast<unsigned>(sequence) < static_cast<unsigned>(c.max_sequences)) ask_for(c.lengths + sequence);
}

// Exclusive sum of `mine` over the block; `total` is the whole sum.
__device__ int block_prefix(int mine, BookShared& s, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = mine;
#pragma unroll
  for (int step = 1; step < 32; step *= 2) {
    const int other = __shfl_up_sync(0xffffffffu, upto, step);
    if (lane >= step) upto += other;
  }
  __syncthreads();  // (the sums of the call before are read)
  if (lane == 31) s.warp_sums[warp] = upto;
  __syncthreads();
  int below = 0;
  total = 0;
  const int other = s.warp_sums[lane];
#pragma unroll
  for (int w = 0; w < kBookThreads / 32; ++w) {
    const int sum = __shfl_sync(0xffffffffu, other, w);
    if (w < warp) below += sum;
    total += sum;
  }
  return below + upto - mine;
}

// The `need` lowest free pages into `list`; false when there are fewer.
__device__ bool list_free_pages(const PagedCache& c, int need, int* list, BookShared& s) {
  int found = 0;
  for (int start = 0; start < c.pages && found < need; start += kBookThreads) {
    const int page = start + threadIdx.x;
    const bool is_free = page < c.pages && c.references[page] == 0;
    int total;
    const int rank = found + block_prefix(is_free, s, total);
    if (is_free && rank < need) list[rank] = page;
    found += total;
  }
  __syncthreads();
  return found >= need;
}

// Marks the sequences of a list as taken; a second mark, or one out of range, raises s.flag.
__device__ void claim(const PagedCache& c, int sequence, BookShared& s) {
  if (static_cast<unsigned>(sequence) >= static_cast<unsigned>(c.max_sequences) ||
      atomicAdd(&c.claims[sequence], 1) != 0) {
    s.flag = kCacheBadSequence;
  }
}

__device__ void unclaim(const PagedCache& c, int sequence) {
  if (static_cast<unsigned>(sequence) < static_cast<unsigned>(c.max_sequences)) {
    c.claims[sequence] = 0;
  }
}

__device__ __forceinline__ int held_tokens(const PagedCache& c, int sequence) {
  const int64_t room = static_cast<int64_t>(c.max_pages) << c.page_shift;
  const int held = c.lengths[sequence];
  return held < 0 ? 0 : held > room ? static_cast<int>(room) : held;
}

// The rows that sequence i of the list is to get; s.flag where the books do not allow it.
__device__ int extension(const PagedCache& c, const Batch& b, int i, int& old_length, BookShared& s) {
  const int rows = b.offsets[i + 1] - b.offsets[i];
  old_length = held_tokens(c, b.sequences[i]);
  if (rows < 0 || b.offsets[i] < 0 || b.offsets[i + 1] > b.rows) {
    s.flag = kCacheBadSequence;
    return 0;
  }
  if (static_cast<int64_t>(old_length) + rows > (static_cast<int64_t>(c.max_pages) << c.page_shift)) {
    s.flag = kCacheNoPages;
    return 0;
  }
  return rows;
}

__global__ void __launch_bounds__(kBookThreads) kv_extend_kernel(PagedCache c, Batch b) {
  __shared__ BookShared s;
  release_successor();
  wait_for_predecessor();
  const CacheWords words = cache_words(c);
  ask_for_lengths(c, b.sequences, b.count);
  if (books_closed(c, words)) return;
  if (threadIdx.x == 0) s.flag = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < b.count; i += kBookThreads) claim(c, b.sequences[i], s);
  __syncthreads();
  int need = 0;
  int* list = nullptr;
  if (s.flag == 0) {
    __syncthreads();
    for (int start = 0; start < b.count; start += kBookThreads) {
      const int i = start + threadIdx.x;
      int mine = 0, held;
      if (i < b.count) {
        const int rows = extension(c, b, i, held, s);
        mine = pages_of(c, held + rows) - pages_of(c, held);
      }
      int total;
      block_prefix(mine, s, total);
      need = min(need + total, c.pages + 1);
    }
    __syncthreads();
    if (s.flag == 0) {
      __syncthreads();
      list = need <= kBookThreads ? s.list : c.move_target;
      if (!list_free_pages(c, need, list, s) && threadIdx.x == 0) s.flag = kCacheNoPages;
    }
  }
  __syncthreads();
  if (s.flag == 0) {
    int before = 0;
    for (int start = 0; start < b.count; start += kBookThreads) {
      const int i = start + threadIdx.x;
      int mine = 0, held = 0, rows = 0;
      if (i < b.count) {
        rows = extension(c, b, i, held, s);
        mine = pages_of(c, held + rows) - pages_of(c, held);
      }
      int total;
      const int at = before + block_prefix(mine, s, total);
      if (i < b.count) {
        const int sequence = b.sequences[i];
        int* row = c.table + static_cast<size_t>(sequence) * c.max_pages + pages_of(c, held);
        for (int j = 0; j < mine; ++j) {
          const int page = list[at + j];
          row[j] = page;
          c.references[page] = 1;
        }
        c.lengths[sequence] = held + rows;
      }
      before += total;
    }
  } else if (threadIdx.x == 0) {
    report_cache_error(c.error, s.flag);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < b.count; i += kBookThreads) unclaim(c, b.sequences[i]);
}

// Adds `change` to the references of the pages that a list's sequences hold; a warp per sequence.
__device__ void count_pages(const PagedCache& c, const int* sequences, int count, int change) {
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < count; i += kBookThreads / 32) {
    const int sequence = sequences[i], held = pages_of(c, held_tokens(c, sequence));
    for (int place = lane; place < held; place += 32) {
      const int page = page_at(c, sequence, place);
      if (page >= 0) atomicAdd(&c.references[page], change);
    }
  }
}

__global__ void __launch_bounds__(kBookThreads)
    kv_free_kernel(PagedCache c, const int* sequences, int count) {
  __shared__ BookShared s;
  release_successor();
  wait_for_predecessor();
  const CacheWords words = cache_words(c);
  ask_for_lengths(c, sequences, count);
  if (books_closed(c, words)) return;
  if (threadIdx.x == 0) s.flag = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kBookThreads) claim(c, sequences[i], s);
  __syncthreads();
  if (s.flag == 0) {
    count_pages(c, sequences, count, -1);
    __syncthreads();
    for (int i = threadIdx.x >> 5; i < count; i += kBookThreads / 32) {
      const int sequence = sequences[i], held = pages_of(c, held_tokens(c, sequence));
      int* row = c.table + static_cast<size_t>(sequence) * c.max_pages;
      for (int place = threadIdx.x & 31; place < held; place += 32) row[place] = 0;
      __syncwarp();
      if ((threadIdx.x & 31) == 0) c.lengths[sequence] = 0;
    }
  } else if (threadIdx.x == 0) {
    report_cache_error(c.error, s.flag);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kBookThreads) unclaim(c, sequences[i]);
}

// The books of a fork.  The children's own pages are given up first, so that they can serve as the
// copies; where the free ones do not suffice all the same, they are taken back.
__global__ void __launch_bounds__(kBookThreads)
    kv_fork_kernel(PagedCache c, const int* parents, const int* children, int count) {
  __shared__ BookShared s;
  release_successor();
  wait_for_predecessor();
  const CacheWords words = cache_words(c);
  ask_for_lengths(c, parents, count);
  ask_for_lengths(c, children, count);
  if (threadIdx.x == 0) {
    s.flag = 0;
    *c.move_count = -1;
  }
  if (books_closed(c, words)) return;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kBookThreads) claim(c, children[i], s);
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kBookThreads) {
    const int parent = parents[i];  // in range, and no child
    if (static_cast<unsigned>(parent) >= static_cast<unsigned>(c.max_sequences) ||
        c.claims[parent] != 0) {
      s.flag = kCacheBadSequence;
    }
  }
  __syncthreads();
  if (s.flag == 0) {
    count_pages(c, children, count, -1);
    int need = 0;
    for (int start = 0; start < count; start += kBookThreads) {
      const int i = start + threadIdx.x;
      const int tokens = i < count ? held_tokens(c, parents[i]) : 0;
      const int mine = (tokens & (c.page_tokens - 1)) != 0;
      const int source = mine ? page_at(c, parents[i], tokens >> c.page_shift) : 0;
      int total;
      const int at = need + block_prefix(mine, s, total);
      if (mine && at < c.pages) c.move_source[at] = source;
      if (source < 0) s.flag = kCacheBadSequence;
      need += total;
    }
    __syncthreads();
    int* list = need <= kBookThreads ? s.list : c.move_target;
    const bool enough = need <= c.pages && list_free_pages(c, need, list, s);
    if (!enough && threadIdx.x == 0) s.flag = kCacheNoPages;
    __syncthreads();
    if (s.flag != 0) {
      count_pages(c, children, count, 1);
    } else {
      // a partly filled last page's copy, then the full pages
      int before = 0;
      for (int start = 0; start < count; start += kBookThreads) {
        const int i = start + threadIdx.x;
        const int tokens = i < count ? held_tokens(c, parents[i]) : 0;
        const int mine = (tokens & (c.page_tokens - 1)) != 0;
        int total;
        const int at = before + block_prefix(mine, s, total);
        if (mine) {
          const int page = list[at];
          c.table[static_cast<size_t>(children[i]) * c.max_pages + (tokens >> c.page_shift)] = page;
          c.references[page] = 1;
          c.move_target[at] = page;
        }
        before += total;
      }
      for (int i = threadIdx.x >> 5; i < count; i += kBookThreads / 32) {
        const int tokens = held_tokens(c, parents[i]), full = tokens >> c.page_shift;
        const bool partial = (tokens & (c.page_tokens - 1)) != 0;
        int* row = c.table + static_cast<size_t>(children[i]) * c.max_pages;
        for (int place = threadIdx.x & 31; place < c.max_pages; place += 32) {
          int page = 0;
          if (place < full) {
            page = c.table[static_cast<size_t>(parents[i]) * c.max_pages + place];
            if (static_cast<unsigned>(page) < static_cast<unsigned>(c.pages)) {
              atomicAdd(&c.references[page], 1);
            } else {  // (copied as it stands: it is no page of the child's, either)
              report_cache_error(c.raised, kCacheBadSequence);
            }
          } else if (place == full && partial) {
            continue;
          }
          row[place] = page;
        }
        if ((threadIdx.x & 31) == 0) c.lengths[children[i]] = tokens;
      }
      if (threadIdx.x == 0) *c.move_count = need;
    }
  }
  __syncthreads();
  if (s.flag != 0 && threadIdx.x == 0) report_cache_error(c.error, s.flag);
  for (int i = threadIdx.x; i < count; i += kBookThreads) unclaim(c, children[i]);
}

// The books of a compaction: with L pages in use, the i-th of them at or above L goes to the i-th free
// one below L.  The block table follows in the copy kernel, which has the threads for it.
__global__ void __launch_bounds__(kBookThreads) kv_compact_kernel(PagedCache c) {
  __shared__ BookShared s;
  release_successor();
  wait_for_predecessor();
  const CacheWords words = cache_words(c);
  if (threadIdx.x == 0) *c.move_count = -1;
  int live = 0;
  for (int page = threadIdx.x; page < c.pages; page += kBookThreads) {
    live += c.references[page] > 0;
    c.remap[page] = page;
  }
  if (books_closed(c, words)) return;
  int total;
  block_prefix(live, s, total);
  live = total;
  int sources = 0, targets = 0;
  for (int start = 0; start < c.pages; start += kBookThreads) {
    const int page = start + threadIdx.x;
    const bool used = page < c.pages && c.references[page] > 0;
    const bool source = used && page >= live, target = page < live && !used;
    const int before = block_prefix(source | (target << 16), s, total);  // (at most 1024 of each)
    if (source) c.move_source[sources + (before & 0xffff)] = page;
    if (target) c.move_target[targets + (before >> 16)] = page;
    sources += total & 0xffff;
    targets += total >> 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < sources; i += kBookThreads) {
    const int from = c.move_source[i], to = c.move_target[i];
    c.remap[from] = to;
    c.references[to] = c.references[from];
    c.references[from] = 0;
  }
  if (threadIdx.x == 0) *c.move_count = sources;
}

// ---------------------------------------------------------------------------
// Contents of pages, all layers
// ---------------------------------------------------------------------------

constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = kCopyThreads * 4;  // of 16 bytes: four loads under way in each thread

// Bound by memory: 781 MB of a compaction in 131 us, 0.91 of the copy rate.  A chunk is a page's part, not a page: 128
// copies in 8 layers, or a few, are spread evenly.  It is launched while the books are kept and waits for them.

__global__ void __launch_bounds__(kCopyThreads)
    kv_copy_kernel(PagedCache c, const int* sources, const int* targets, bool of_books, int count, bool rewrite_table) {
  release_successor();
  wait_for_predecessor();  // (the books)
  if (of_books) {
    count = *c.move_count;
    if (count < 0) return;
  }
  const int heads2 = 2 * c.kv_heads;
  const size_t page_words = static_cast<size_t>(heads2) * c.page_tokens * kHeadDim / 16;
  const int chunks = static_cast<int>((page_words + kCopyChunk - 1) / kCopyChunk);
  const int64_t of_layer = static_cast<int64_t>(count) * chunks;
  for (int64_t u = blockIdx.x; u < of_layer * c.layers; u += gridDim.x) {
    const size_t layer = u / of_layer;
    const int move = static_cast<int>(u % of_layer / chunks), chunk = static_cast<int>(u % chunks);
    const int from = sources[move], to = targets[move];
    if (static_cast<unsigned>(from) >= static_cast<unsigned>(c.pages) ||
        static_cast<unsigned>(to) >= static_cast<unsigned>(c.pages)) {
      report_cache_error(c.raised, kCacheBadSequence);
      continue;
    }
    const size_t read_page = layer * c.pages + from, write_page = layer * c.pages + to;
    const size_t at = static_cast<size_t>(chunk) * kCopyChunk + threadIdx.x;
    const uint4* read = reinterpret_cast<const uint4*>(c.codes) + read_page * page_words + at;
    uint4* write = reinterpret_cast<uint4*>(c.codes) + write_page * page_words + at;
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (at + i * kCopyThreads < page_words) x[i] = __ldcs(read + i * kCopyThreads);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (at + i * kCopyThreads < page_words) __stcs(write + i * kCopyThreads, x[i]);
    }
    if (chunk == 0) {
      for (int i = threadIdx.x; i < heads2; i += kCopyThreads) {
        c.exponents[write_page * heads2 + i] = c.exponents[read_page * heads2 + i];
      }
    }
  }
  if (!rewrite_table) return;
  const int warps = gridDim.x * (kCopyThreads / 32);
  // (from the last block down: of few pages and sequences other blocks do the copies)
  for (int i = warps - 1 - static_cast<int>((blockIdx.x * kCopyThreads + threadIdx.x) >> 5); i < c.max_sequences; i += warps) {
    const int held = pages_of(c, held_tokens(c, i));
    int* row = c.table + static_cast<size_t>(i) * c.max_pages;
    for (int place = threadIdx.x & 31; place < held; place += 32) {
      const int page = page_at(c, i, place);
      if (page >= 0) row[place] = c.remap[page];
    }
  }
}

cudaError_t launch_copy(const PagedCache& cache, const int* sources, const int* targets,
                        bool of_books, int count, bool rewrite_table, cudaStream_t stream) {
  return launch_kernel(kv_copy_kernel, dim3(device_sms() * 8), kCopyThreads, 0,
                       LaunchStream(stream, true), cache, sources, targets, of_books,
                       count, rewrite_table);
}

}  // namespace

cudaError_t launch_kv_append(const PagedCache& cache, const Batch& batch, int layer,
                             const __nv_bfloat16* k, int64_t k_stride, const __nv_bfloat16* v,
                             int64_t v_stride, cudaStream_t stream) {
  // c rows of a sequence touch at most c / page_tokens + 2 pages, and no more than c
  const int64_t units = std::min<int64_t>(
      batch.rows, (batch.rows >> cache.page_shift) + 2 * static_cast<int64_t>(batch.count));
  // as many heads to a block as it takes for all blocks to be resident at once
  const int64_t of = 2 * cache.kv_heads, resident = kAppendBlocks * device_sms();
  const int64_t groups = std::clamp<int64_t>(resident / units, 1, of);
  const int per_block = static_cast<int>((of + groups - 1) / groups);
  const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>((of + per_block - 1) / per_block));
  auto* kernel = cache.page_tokens == 16   ? kv_append_kernel<16>
                 : cache.page_tokens == 32 ? kv_append_kernel<32>
                 : cache.page_tokens == 64 ? kv_append_kernel<64>
                                           : kv_append_kernel<128>;
  return launch_kernel(kernel, grid, kAppendThreads, 0, LaunchStream(stream, true), cache, batch, layer, k,
                       k_stride, v, v_stride, per_block);
}

cudaError_t launch_kv_extend(const PagedCache& cache, const Batch& batch, cudaStream_t stream) {
  return launch_kernel(kv_extend_kernel, dim3(1), kBookThreads, 0, LaunchStream(stream, true), cache, batch);
}

cudaError_t launch_kv_fork(const PagedCache& cache, const int* parents, const int* children, int count,
                           cudaStream_t stream) {
  const cudaError_t err = launch_kernel(kv_fork_kernel, dim3(1), kBookThreads, 0, LaunchStream(stream, true), cache, parents, children, count);
  if (err != cudaSuccess) return err;
  return launch_copy(cache, cache.move_source, cache.move_target, true, 0, false, stream);
}

cudaError_t launch_kv_free(const PagedCache& cache, const int* sequences, int count,
                           cudaStream_t stream) {
  return launch_kernel(kv_free_kernel, dim3(1), kBookThreads, 0, LaunchStream(stream, true), cache, sequences, count);
}

cudaError_t launch_kv_compact(const PagedCache& cache, cudaStream_t stream) {
  const cudaError_t err = launch_kernel(kv_compact_kernel, dim3(1), kBookThreads, 0, LaunchStream(stream, true), cache);
  if (err != cudaSuccess) return err;
  return launch_copy(cache, cache.move_source, cache.move_target, true, 0, true, stream);
}

cudaError_t launch_kv_copy_pages(const PagedCache& cache, const int* sources, const int* targets,
                                 int count, cudaStream_t stream) {
  return launch_copy(cache, sources, targets, false, count, false, stream);
}

}  // namespace nmoe
