// Internal declarations of the attention operators: the paged 8-bit cache as kernels see it, and the
// launchers behind the C ABI of attention_api.cu.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>

#include "kernels.h"

namespace nmoe {

constexpr int kHeadDim = 128;
constexpr int kMinExponent = -32, kMaxExponent = 32;  // of a page and head's scale, 2^exponent

// What a kernel can leave in a cache's words `error` and `raised`, beside kDevWaitTimeout.
enum CacheError : int {
  kCacheNoPages = 16,      // fewer free pages, or places in the block table, than asked for
  kCacheBadSequence = 17,  // a sequence out of range or twice in a list, a page out of range
};

// Codes [layers][pages][2: keys, values][kv_heads][page_tokens][128], exponents without the last two.
struct PagedCache {
  int layers, pages, kv_heads, page_tokens, page_shift, max_sequences, max_pages;
  uint8_t* codes;
  int8_t* exponents;
  int* table;       // [max_sequences][max_pages]
  int* lengths;     // [max_sequences]
  int* references;  // [pages]; 0: free
  // Two words, of which the first code stays.  `error`: the books could not be kept, or a wait ran out; appends and
  // attention read it and do nothing then.  `raised`: an entry or a page that appends, attention or copies of pages
  // found wrong and left out; the books read it, too, and pass it on to `error` when they do nothing.  None of a
  // launch's blocks reads what others of it write, so a wrong entry changes nothing for the rest of its batch.
  int* error;        // the first of four words that are read together: error, move_count, raised, impatient
  int* move_count;   // pages for the copy kernel: the first *move_count of the two lists; -1: the books stay as they are
  int* raised;
  int* move_source;  // [pages]
  int* move_target;  // [pages]
  int* remap;        // [max(pages, max_sequences)]: where a page went, a child's copy
  int* claims;       // [max_sequences], zero between calls
  char* attend_workspace;
};

// Rows of a batch: sequence i has the rows [offsets[i], offsets[i + 1]) of `rows`.
struct Batch {
  const int* sequences;
  const int* offsets;
  int count;
  int rows;
};

struct BatchEntry {
  int sequence, first, rows, length;  // length: tokens in the cache, these rows among them
  int skip;                           // tokens before the first that is attended
  bool valid;
};

#ifdef __CUDACC__

__device__ __forceinline__ void report_cache_error(int* error, int code) {
  if (error != nullptr) atomicCAS(error, 0, code);
}

// The words at c.error, in one load.
struct CacheWords {
  int error, move_count, raised;
  int impatient;  // tests set it: a block leaves a join at once where pieces are missing
  __device__ bool pending() const { return (error | raised) != 0; }  // what the books go by
};
__device__ __forceinline__ CacheWords cache_words(const PagedCache& c) {
  const int4 words = *reinterpret_cast<const int4*>(c.error);
  return {words.x, words.y, words.z, words.w};
}

// Entry i of a batch, brought into range: whatever the arrays hold, its rows lie within the batch's
// and its tokens within the block table.
__device__ __forceinline__ BatchEntry batch_entry(const PagedCache& c, const Batch& b, int i) {
  BatchEntry e;
  e.skip = 0;
  e.sequence = b.sequences[i];
  const int from = b.offsets[i], to = b.offsets[i + 1];
  e.first = min(max(from, 0), b.rows);
  e.rows = min(max(to, e.first), b.rows) - e.first;
  e.valid = static_cast<unsigned>(e.sequence) < static_cast<unsigned>(c.max_sequences) &&
            from == e.first && to == e.first + e.rows;
  e.length = 0;
  if (e.valid) {
    const int held = c.lengths[e.sequence];
    const int64_t room = static_cast<int64_t>(c.max_pages) << c.page_shift;
    e.valid = held >= e.rows && held <= room;
    e.length = e.valid ? held : 0;
  }
  if (!e.valid) e.rows = 0;
  return e;
}

__device__ __forceinline__ int pages_of(const PagedCache& c, int tokens) {
  return (tokens >> c.page_shift) + ((tokens & (c.page_tokens - 1)) != 0);
}

// The page that holds tokens [page_tokens * place, ...) of a sequence, -1 for an entry out of range.
__device__ __forceinline__ int page_at(const PagedCache& c, int sequence, int place) {
  const int page = c.table[static_cast<size_t>(sequence) * c.max_pages + place];
  return static_cast<unsigned>(page) < static_cast<unsigned>(c.pages) ? page : -1;
}

// Index of the (half, head) block of a page; its codes begin at this times page_tokens * 128.
__device__ __forceinline__ size_t block_of_page(const PagedCache& c, int layer, int page, int half,
                                                int head) {
  return ((static_cast<size_t>(layer) * c.pages + page) * 2 + half) * c.kv_heads + head;
}

// Unit `u` of the units that entries 0..n-1 have (units(i) of them, in order): its entry and its place
// in it, entry -1 behind the last.  Called by whole warps with the same u.
template <typename Units>
__device__ __forceinline__ int2 locate_unit(int n, int64_t u, Units units) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int start = 0; start < n; start += 32) {
    const int i = start + lane;
    const int mine = i < n ? units(i) : 0;
    int64_t upto = mine;
#pragma unroll
    for (int step = 1; step < 32; step *= 2) {
      const int64_t other = __shfl_up_sync(0xffffffffu, upto, step);
      if (lane >= step) upto += other;
    }
    const int64_t total = __shfl_sync(0xffffffffu, upto, 31);
    if (u < before + total) {
      const int owner = __ffs(__ballot_sync(0xffffffffu, u < before + upto)) - 1;
      const int place = static_cast<int>(u - (before + upto - mine));
      return make_int2(start + owner, __shfl_sync(0xffffffffu, place, owner));
    }
    before += total;
  }
  return make_int2(-1, 0);
}

#endif  // __CUDACC__

// allow_shared_memory(), once for each device (a bit of `allowed`): it takes a tenth of a short call.
template <typename Kernel>
inline cudaError_t allow_shared_memory_once(Kernel* kernel, std::atomic<uint64_t>& allowed) {
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (allowed.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  err = allow_shared_memory(kernel);
  if (err == cudaSuccess && device < 64) allowed.fetch_or(bit, std::memory_order_release);
  return err;
}

struct PrefillArgs {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t q_stride, k_stride, v_stride;  // elements from one token's row to the next
  int tokens, heads, kv_heads;
  const int* offsets;
  int sequences;
  float scale;
  __nv_bfloat16* out;  // [tokens][heads][128]
  bool out_aligned;    // to 32 bytes
  float* lse;          // [tokens][heads], may be null
  int* error;
};

// Attention over a cache may be taken in parts: what the sequences of a group share, once for all of their rows, and
// what each has of its own.
enum class Part { kAll, kShared, kOwn };

// Where a row's sums of a part are (csrc/attention_shared.cu).
struct alignas(16) RowPart {
  float reference, sum;
  int parts_row;  // 1: beside the other rows'; else 256 times the number of pieces in the workspace, and its row there
  int lead;       // first block that has one
};

struct CachedArgs {
  PagedCache cache;
  Batch batch;
  int layer;
  const __nv_bfloat16* q;
  int64_t q_stride;
  int heads;
  float scale;
  __nv_bfloat16* out;
  // Of a batch in groups: entries [groups[g], groups[g + 1]) share the first shared[i] tokens, whole tiles.
  const int* groups;
  int group_count;
  const int* shared;
  float* sums;        // of this part, [rows][heads][128]
  RowPart* row_parts;  // [rows][heads]
};

// bf16 rows of heads x 128 as [rows][heads * 128], boxes of 64 columns x box_rows, 128-byte swizzle.
bool rows_tensor_map(const void* base, int64_t rows, int64_t heads, int64_t stride, int box_rows,
                     CUtensorMap* map);
// The same of any bf16 matrix [rows][columns]; what lies beside it reads as zeros.
bool matrix_tensor_map(const void* base, int64_t rows, int64_t columns, int64_t stride, int box_rows,
                       CUtensorMap* map);

// A cache's codes as rows of 128 bytes, boxes of a page and head, 128-byte swizzle.
bool pages_tensor_map(const PagedCache& cache, CUtensorMap* map);
// Any rows of 128 codes.
bool codes_tensor_map(const uint8_t* codes, int64_t rows, int box_rows, CUtensorMap* map);

cudaError_t launch_attention_prefill(const PrefillArgs& args, cudaStream_t stream);
// The workspace begins with counters, zero between calls.
constexpr size_t kAttendCounterBytes = 4096;
size_t attention_cached_workspace_bytes();
cudaError_t launch_attention_cached(const CachedArgs& args, cudaStream_t stream);
// The kernels behind it by the rows of queries that an entry, or a group, has on average; `slots` of the workspace for
// pieces, attention_cached_slot_bytes() bytes.
size_t attention_cached_slot_bytes();
int attention_cached_slot_rows(int64_t rows);  // that a piece has room for
cudaError_t launch_cached_part(const CachedArgs& args, Part part, int64_t rows, float* slots, cudaStream_t stream);
// Of shared tokens, for more rows of queries than that (csrc/attention_shared_rows.cu).
size_t shared_pairs_slot_bytes();
int shared_pairs_slot_rows();
size_t shared_pairs_query_bytes(int64_t rows, int heads);  // of `query_space`, 256-byte aligned
bool shared_pairs_supported(int64_t rows, int heads);
cudaError_t launch_shared_pairs(const CachedArgs& args, float* slots, char* query_space, cudaStream_t stream);
// The same results for a batch whose sequences share their first pages; `workspace`:
// attention_shared_workspace_bytes().
size_t attention_shared_workspace_bytes(int64_t rows, int heads);
cudaError_t launch_attention_shared(const CachedArgs& args, char* workspace, cudaStream_t stream);
cudaError_t launch_kv_find_shared(const PagedCache& cache, const Batch& batch, const int* groups, int group_count, int* shared,
                                  cudaStream_t stream);
cudaError_t launch_kv_append(const PagedCache& cache, const Batch& batch, int layer,
                             const __nv_bfloat16* k, int64_t k_stride, const __nv_bfloat16* v,
                             int64_t v_stride, cudaStream_t stream);
cudaError_t launch_kv_extend(const PagedCache& cache, const Batch& batch, cudaStream_t stream);
cudaError_t launch_kv_fork(const PagedCache& cache, const int* parents, const int* children, int count,
                           cudaStream_t stream);
cudaError_t launch_kv_free(const PagedCache& cache, const int* sequences, int count,
                           cudaStream_t stream);
cudaError_t launch_kv_compact(const PagedCache& cache, cudaStream_t stream);
cudaError_t launch_kv_copy_pages(const PagedCache& cache, const int* sources, const int* targets,
                                 int count, cudaStream_t stream);

}  // namespace nmoe
