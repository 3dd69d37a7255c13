// C ABI of the attention operators (include/nmoe.h): checks of arguments, the workspace's layout, and
// the status of what ran on the device.
#include <cmath>

#include "../../include/nmoe.h"
#include "attention.h"
#include "common.cuh"
#include "kernels.h"

namespace {

using nmoe::Batch;
using nmoe::PagedCache;

constexpr size_t kAlign = 256;
size_t aligned(size_t bytes) { return (bytes + kAlign - 1) / kAlign * kAlign; }
bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

bool shape_valid(const nmoe_kv_cache& c) {
  return c.layers > 0 && c.pages > 0 && c.kv_heads > 0 && c.max_sequences > 0 &&
         c.max_pages_per_sequence > 0 &&
         (c.page_tokens == 16 || c.page_tokens == 32 || c.page_tokens == 64 || c.page_tokens == 128) &&
         // tokens of a sequence are counted in 32 bits
         static_cast<int64_t>(c.max_pages_per_sequence) * c.page_tokens <= INT32_MAX - 128;
}

struct Layout {
  size_t move_source, move_target, remap, claims, attend, total;
};

// Header (the words below), the lists of the page kernels, the attention's parts.
enum HeaderWord { kErrorWord, kMoveCountWord, kRaisedWord, kImpatientWord, kHeaderWords };

Layout layout_of(const nmoe_kv_cache& c) {
  const size_t pages = sizeof(int) * static_cast<size_t>(c.pages);
  const size_t sequences = sizeof(int) * static_cast<size_t>(c.max_sequences);
  Layout l;
  l.move_source = kAlign;
  l.move_target = l.move_source + aligned(pages);
  l.remap = l.move_target + aligned(pages);
  l.claims = l.remap + aligned(pages > sequences ? pages : sequences);
  l.attend = l.claims + aligned(sequences);
  l.total = l.attend + nmoe::attention_cached_workspace_bytes();
  return l;
}

// The cache as kernels see it; false where the descriptor is not one.
bool view_of(const nmoe_kv_cache* c, PagedCache& view) {
  if (c == nullptr || !shape_valid(*c) || c->codes == nullptr || c->exponents == nullptr ||
      c->block_table == nullptr || c->lengths == nullptr || c->references == nullptr ||
      c->workspace == nullptr || misaligned(c->codes, 128) || misaligned(c->block_table, 4) ||
      misaligned(c->lengths, 4) || misaligned(c->references, 4) || misaligned(c->workspace, kAlign)) {
    return false;
  }
  const Layout l = layout_of(*c);
  if (c->workspace_bytes < l.total) return false;
  char* w = static_cast<char*>(c->workspace);
  view.layers = c->layers;
  view.pages = c->pages;
  view.kv_heads = c->kv_heads;
  view.page_tokens = c->page_tokens;
  view.page_shift = c->page_tokens == 16 ? 4 : c->page_tokens == 32 ? 5 : c->page_tokens == 64 ? 6 : 7;
  view.max_sequences = c->max_sequences;
  view.max_pages = c->max_pages_per_sequence;
  view.codes = c->codes;
  view.exponents = c->exponents;
  view.table = c->block_table;
  view.lengths = c->lengths;
  view.references = c->references;
  view.error = reinterpret_cast<int*>(w) + kErrorWord;
  view.move_count = reinterpret_cast<int*>(w) + kMoveCountWord;
  view.raised = reinterpret_cast<int*>(w) + kRaisedWord;
  view.move_source = reinterpret_cast<int*>(w + l.move_source);
  view.move_target = reinterpret_cast<int*>(w + l.move_target);
  view.remap = reinterpret_cast<int*>(w + l.remap);
  view.claims = reinterpret_cast<int*>(w + l.claims);
  view.attend_workspace = w + l.attend;
  return true;
}

bool batch_of(const int32_t* sequences, const int32_t* offsets, int32_t count, int64_t rows, Batch& b) {
  if (count < 0 || rows < 0 || rows > INT32_MAX / 2 ||
      (count > 0 && (sequences == nullptr || offsets == nullptr)) || misaligned(sequences, 4) ||
      misaligned(offsets, 4)) {
    return false;
  }
  b = Batch{sequences, offsets, count, static_cast<int>(rows)};
  return true;
}

// Rows of heads x 128 bf16, 16 bytes at a time.
bool rows_valid(const void* p, int64_t stride, int64_t heads) {
  return p != nullptr && !misaligned(p, 16) && stride % 8 == 0 && stride >= heads * nmoe::kHeadDim;
}

nmoe_status status_of(cudaError_t err) {
  if (err == cudaSuccess) return NMOE_OK;
  cudaGetLastError();  // reported here: it must not fail the next launch as well
  return err == cudaErrorInvalidValue ? NMOE_ERR_INVALID_ARGUMENT : NMOE_ERR_CUDA;
}

nmoe_status device_status(int code) {
  switch (code) {
    case nmoe::kDevOk: return NMOE_OK;
    case nmoe::kDevWaitTimeout: return NMOE_ERR_DEVICE_TIMEOUT;
    case nmoe::kCacheNoPages: return NMOE_ERR_CAPACITY;
    default: return NMOE_ERR_INVALID_ARGUMENT;
  }
}

// Waits for the stream, reads an error word and clears it.
nmoe_status sync_error_word(int* word, cudaStream_t stream) {
  int code = 0;
  cudaError_t err = cudaMemcpyAsync(&code, word, sizeof(code), cudaMemcpyDeviceToHost, stream);
  if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
  if (err == cudaSuccess && code != 0) {
    err = cudaMemsetAsync(word, 0, sizeof(code), stream);
    if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
  }
  return err == cudaSuccess ? device_status(code) : status_of(err);
}

// The same for a cache's words, with what a call that gave up may have left.
nmoe_status sync_cache(const PagedCache& cache, cudaStream_t stream) {
  int words[kHeaderWords] = {};
  cudaError_t err = cudaMemcpyAsync(words, cache.error, sizeof(words), cudaMemcpyDeviceToHost, stream);
  if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
  const int code = words[kErrorWord] != 0 ? words[kErrorWord] : words[kRaisedWord];
  if (err == cudaSuccess && code != 0) {
    err = cudaMemsetAsync(cache.error, 0, sizeof(int), stream);
    if (err == cudaSuccess) err = cudaMemsetAsync(cache.raised, 0, sizeof(int), stream);
    if (err == cudaSuccess) err = cudaMemsetAsync(cache.attend_workspace, 0, nmoe::kAttendCounterBytes, stream);
    if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
  }
  return err == cudaSuccess ? device_status(code) : status_of(err);
}

bool scale_valid(float scale) { return std::isfinite(scale) && scale > 0.0f; }

// Entries of a batch in groups.
bool groups_valid(const int32_t* groups, int32_t group_count, int32_t count) {
  return group_count >= 0 && group_count <= count && (group_count == 0 || groups != nullptr) && !misaligned(groups, 4);
}

constexpr int64_t kMostSharedPairs = 1ll << 32;  // rows x heads: 2 TB of sums

}  // namespace

namespace nmoe {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                 CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static const EncodeTiled found = [] {
    void* symbol = nullptr;
    cudaDriverEntryPointQueryResult query;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &symbol, cudaEnableDefault, &query) !=
            cudaSuccess ||
        query != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      symbol = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(symbol);
  }();
  return found;
}

bool rows_tensor_map(const void* base, int64_t rows, int64_t heads, int64_t stride, int box_rows,
                     CUtensorMap* map) {
  return matrix_tensor_map(base, rows, heads * kHeadDim, stride, box_rows, map);
}

bool matrix_tensor_map(const void* base, int64_t rows, int64_t columns, int64_t stride, int box_rows,
                       CUtensorMap* map) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
  const cuuint32_t box[2] = {64u, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t steps[2] = {1u, 1u};
  const EncodeTiled encode = encode_tiled();
  return encode != nullptr &&
         encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box,
                steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool pages_tensor_map(const PagedCache& cache, CUtensorMap* map) {
  return codes_tensor_map(cache.codes, static_cast<int64_t>(cache.layers) * cache.pages * 2 * cache.kv_heads * cache.page_tokens,
                          cache.page_tokens, map);
}

bool codes_tensor_map(const uint8_t* codes, int64_t rows, int box_rows, CUtensorMap* map) {
  if (rows > INT32_MAX) return false;  // a coordinate has 31 bits: 256 GB of codes
  const cuuint64_t dims[2] = {kHeadDim, static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {kHeadDim};
  const cuuint32_t box[2] = {kHeadDim, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t steps[2] = {1u, 1u};
  const EncodeTiled encode = encode_tiled();
  return encode != nullptr &&
         encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, steps,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace nmoe

extern "C" {

size_t nmoe_kv_workspace_bytes(const nmoe_kv_cache* cache) {
  return cache == nullptr || !shape_valid(*cache) ? 0 : layout_of(*cache).total;
}

nmoe_status nmoe_kv_extend(const nmoe_kv_cache* cache, void* stream, const int32_t* sequences,
                           const int32_t* offsets, int32_t count, int64_t rows) {
  PagedCache view;
  Batch batch;
  if (!view_of(cache, view) || !batch_of(sequences, offsets, count, rows, batch)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (count == 0) return NMOE_OK;
  return status_of(nmoe::launch_kv_extend(view, batch, static_cast<cudaStream_t>(stream)));
}

nmoe_status nmoe_kv_append(const nmoe_kv_cache* cache, void* stream, int32_t layer, const void* k,
                           int64_t k_stride, const void* v, int64_t v_stride,
                           const int32_t* sequences, const int32_t* offsets, int32_t count,
                           int64_t rows) {
  PagedCache view;
  Batch batch;
  if (!view_of(cache, view) || !batch_of(sequences, offsets, count, rows, batch) || layer < 0 ||
      layer >= view.layers) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (count == 0 || rows == 0) return NMOE_OK;
  if (!rows_valid(k, k_stride, view.kv_heads) || !rows_valid(v, v_stride, view.kv_heads) ||
      view.kv_heads > 32767) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  return status_of(nmoe::launch_kv_append(
      view, batch, layer, static_cast<const __nv_bfloat16*>(k), k_stride,
      static_cast<const __nv_bfloat16*>(v), v_stride, static_cast<cudaStream_t>(stream)));
}

nmoe_status nmoe_kv_fork(const nmoe_kv_cache* cache, void* stream, const int32_t* parents,
                         const int32_t* children, int32_t count) {
  PagedCache view;
  if (!view_of(cache, view) || count < 0 || count > view.max_sequences ||
      (count > 0 && (parents == nullptr || children == nullptr)) || misaligned(parents, 4) ||
      misaligned(children, 4)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (count == 0) return NMOE_OK;
  return status_of(nmoe::launch_kv_fork(view, parents, children, count,
                                        static_cast<cudaStream_t>(stream)));
}

nmoe_status nmoe_kv_free(const nmoe_kv_cache* cache, void* stream, const int32_t* sequences,
                         int32_t count) {
  PagedCache view;
  if (!view_of(cache, view) || count < 0 || (count > 0 && sequences == nullptr) ||
      misaligned(sequences, 4)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (count == 0) return NMOE_OK;
  return status_of(nmoe::launch_kv_free(view, sequences, count, static_cast<cudaStream_t>(stream)));
}

nmoe_status nmoe_kv_compact(const nmoe_kv_cache* cache, void* stream) {
  PagedCache view;
  if (!view_of(cache, view)) return NMOE_ERR_INVALID_ARGUMENT;
  return status_of(nmoe::launch_kv_compact(view, static_cast<cudaStream_t>(stream)));
}

nmoe_status nmoe_kv_copy_pages(const nmoe_kv_cache* cache, void* stream, const int32_t* sources,
                               const int32_t* targets, int32_t count) {
  PagedCache view;
  if (!view_of(cache, view) || count < 0 || (count > 0 && (sources == nullptr || targets == nullptr)) ||
      misaligned(sources, 4) || misaligned(targets, 4)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (count == 0) return NMOE_OK;
  return status_of(nmoe::launch_kv_copy_pages(view, sources, targets, count,
                                              static_cast<cudaStream_t>(stream)));
}

nmoe_status nmoe_kv_sync_status(const nmoe_kv_cache* cache, void* stream) {
  PagedCache view;
  if (!view_of(cache, view)) return NMOE_ERR_INVALID_ARGUMENT;
  return sync_cache(view, static_cast<cudaStream_t>(stream));
}

nmoe_status nmoe_attention_cached(const nmoe_kv_cache* cache, void* stream, int32_t layer,
                                  const void* q, int64_t q_stride, int32_t heads,
                                  const int32_t* sequences, const int32_t* offsets, int32_t count,
                                  int64_t rows, float scale, void* out) {
  nmoe::CachedArgs args{};
  if (!view_of(cache, args.cache) || !batch_of(sequences, offsets, count, rows, args.batch) ||
      layer < 0 || layer >= args.cache.layers || heads <= 0 || heads % args.cache.kv_heads != 0 ||
      heads > 65535 || !scale_valid(scale)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (count == 0 || rows == 0) return NMOE_OK;
  if (!rows_valid(q, q_stride, heads) || out == nullptr || misaligned(out, 16)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  args.layer = layer;
  args.q = static_cast<const __nv_bfloat16*>(q);
  args.q_stride = q_stride;
  args.heads = heads;
  args.scale = scale;
  args.out = static_cast<__nv_bfloat16*>(out);
  return status_of(nmoe::launch_attention_cached(args, static_cast<cudaStream_t>(stream)));
}

nmoe_status nmoe_kv_find_shared(const nmoe_kv_cache* cache, void* stream, const int32_t* sequences,
                                const int32_t* offsets, int32_t count, int64_t rows,
                                const int32_t* groups, int32_t group_count, int32_t* shared) {
  PagedCache view;
  Batch batch;
  if (!view_of(cache, view) || !batch_of(sequences, offsets, count, rows, batch) ||
      !groups_valid(groups, group_count, count) || misaligned(shared, 4)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (count == 0) return NMOE_OK;
  if (shared == nullptr) return NMOE_ERR_INVALID_ARGUMENT;
  if (group_count == 0) {
    return status_of(cudaMemsetAsync(shared, 0, sizeof(int32_t) * count, static_cast<cudaStream_t>(stream)));
  }
  return status_of(nmoe::launch_kv_find_shared(view, batch, groups, group_count, shared,
                                               static_cast<cudaStream_t>(stream)));
}

size_t nmoe_attention_shared_workspace_bytes(int64_t rows, int32_t heads) {
  if (rows <= 0 || heads <= 0 || heads > 65535 || rows > kMostSharedPairs / heads) return 0;
  return nmoe::attention_shared_workspace_bytes(rows, heads);
}

nmoe_status nmoe_attention_shared(const nmoe_kv_cache* cache, void* stream, int32_t layer,
                                  const void* q, int64_t q_stride, int32_t heads,
                                  const int32_t* sequences, const int32_t* offsets, int32_t count,
                                  int64_t rows, const int32_t* groups, int32_t group_count,
                                  const int32_t* shared, float scale, void* workspace,
                                  size_t workspace_bytes, void* out) {
  if (group_count == 0) {
    return nmoe_attention_cached(cache, stream, layer, q, q_stride, heads, sequences, offsets, count, rows,
                                 scale, out);
  }
  nmoe::CachedArgs args{};
  if (!view_of(cache, args.cache) || !batch_of(sequences, offsets, count, rows, args.batch) ||
      layer < 0 || layer >= args.cache.layers || heads <= 0 || heads % args.cache.kv_heads != 0 ||
      heads > 65535 || !scale_valid(scale) || !groups_valid(groups, group_count, count) ||
      misaligned(shared, 4) || misaligned(workspace, kAlign)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (count == 0 || rows == 0) return NMOE_OK;
  if (!rows_valid(q, q_stride, heads) || out == nullptr || misaligned(out, 16) || shared == nullptr ||
      workspace == nullptr || rows > kMostSharedPairs / heads ||
      workspace_bytes < nmoe::attention_shared_workspace_bytes(rows, heads)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  args.layer = layer;
  args.q = static_cast<const __nv_bfloat16*>(q);
  args.q_stride = q_stride;
  args.heads = heads;
  args.scale = scale;
  args.out = static_cast<__nv_bfloat16*>(out);
  args.groups = groups;
  args.group_count = group_count;
  args.shared = shared;
  return status_of(nmoe::launch_attention_shared(args, static_cast<char*>(workspace),
                                                 static_cast<cudaStream_t>(stream)));
}

nmoe_status nmoe_attention_prefill(void* stream, const void* q, int64_t q_stride, const void* k,
                                   int64_t k_stride, const void* v, int64_t v_stride, int64_t tokens,
                                   int32_t heads, int32_t kv_heads, const int32_t* offsets,
                                   int32_t count, float scale, void* out, float* lse,
                                   int32_t* error) {
  if (tokens < 0 || tokens > INT32_MAX / 2 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 ||
      heads > 65535 || count < 0 || !scale_valid(scale) || misaligned(offsets, 4) ||
      misaligned(lse, 4) || misaligned(error, 4)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (tokens == 0 || count == 0) return NMOE_OK;
  if (!rows_valid(q, q_stride, heads) || !rows_valid(k, k_stride, kv_heads) ||
      !rows_valid(v, v_stride, kv_heads) || offsets == nullptr || out == nullptr ||
      misaligned(out, 16) || error == nullptr) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  nmoe::PrefillArgs args;
  args.q = static_cast<const __nv_bfloat16*>(q);
  args.k = static_cast<const __nv_bfloat16*>(k);
  args.v = static_cast<const __nv_bfloat16*>(v);
  args.q_stride = q_stride;
  args.k_stride = k_stride;
  args.v_stride = v_stride;
  args.tokens = static_cast<int>(tokens);
  args.heads = heads;
  args.kv_heads = kv_heads;
  args.offsets = offsets;
  args.sequences = count;
  args.scale = scale;
  args.out = static_cast<__nv_bfloat16*>(out);
  args.out_aligned = !misaligned(out, 32);
  args.lse = lse;
  args.error = error;
  return status_of(nmoe::launch_attention_prefill(args, static_cast<cudaStream_t>(stream)));
}

nmoe_status nmoe_attention_sync_status(int32_t* error, void* stream) {
  if (error == nullptr || misaligned(error, 4)) return NMOE_ERR_INVALID_ARGUMENT;
  return sync_error_word(error, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
