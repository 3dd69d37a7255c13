// C ABI of the operators of a decode step for many requests (include/nmoe.h): checks of arguments.
#include <cmath>

#include "../../include/nmoe.h"
#include "kernels.h"
#include "serving.h"

namespace {

bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

nmoe_status status_of(cudaError_t err) {
  if (err == cudaSuccess) return NMOE_OK;
  cudaGetLastError();  // reported here: it must not fail the next launch as well
  return err == cudaErrorInvalidValue ? NMOE_ERR_INVALID_ARGUMENT : NMOE_ERR_CUDA;
}

bool pool_valid(const nmoe_adapters* p) {
  return p != nullptr && p->adapters > 0 && p->rank > 0 && p->rank <= nmoe::kMostRank && p->inner > 0 && p->outer > 0 &&
         p->rank % 8 == 0 && p->inner % 8 == 0 && p->outer % 8 == 0 &&
         // rows of A and B are TMA coordinates, up to a tile's behind the last
         static_cast<int64_t>(p->adapters) * p->outer <= INT32_MAX - 256 &&
         static_cast<int64_t>(p->adapters) * p->rank <= INT32_MAX - 256;
}

bool rows_valid(const void* p, int64_t stride, int64_t columns) {
  return p != nullptr && !misaligned(p, 16) && stride % 8 == 0 && stride >= columns;
}

constexpr int64_t kMostAdapterRows = 1 << 24;  // (a launch's tiles)

}  // namespace

extern "C" {

size_t nmoe_adapters_workspace_bytes(const nmoe_adapters* pool, int64_t rows, int32_t count) {
  if (!pool_valid(pool) || rows <= 0 || rows > kMostAdapterRows || count <= 0) return 0;
  return nmoe::adapter_workspace_bytes(rows, count, pool->inner, pool->rank);
}

nmoe_status nmoe_adapters_add(const nmoe_adapters* pool, void* stream, const void* x, int64_t x_stride,
                              const void* y, int64_t y_stride, void* out, int64_t out_stride,
                              int64_t rows, const int32_t* ids, const int32_t* offsets, int32_t count,
                              void* workspace, size_t workspace_bytes, int32_t* error) {
  if (!pool_valid(pool) || rows < 0 || rows > kMostAdapterRows || count < 0 || count > kMostAdapterRows ||
      (count > 0 && (ids == nullptr || offsets == nullptr)) || misaligned(ids, 4) || misaligned(offsets, 4) ||
      misaligned(error, 4)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (rows == 0 || count == 0) return NMOE_OK;
  if (pool->a == nullptr || pool->b == nullptr || pool->scales == nullptr || misaligned(pool->a, 16) ||
      misaligned(pool->b, 16) || misaligned(pool->scales, 4) || !rows_valid(x, x_stride, pool->inner) ||
      !rows_valid(y, y_stride, pool->outer) || !rows_valid(out, out_stride, pool->outer) || error == nullptr ||
      (out == y && out_stride != y_stride && rows > 1) ||  // (over other rows than its own)
      workspace == nullptr || misaligned(workspace, 256) ||
      workspace_bytes < nmoe::adapter_workspace_bytes(rows, count, pool->inner, pool->rank)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  nmoe::AdapterArgs args;
  args.x = static_cast<const __nv_bfloat16*>(x);
  args.x_stride = x_stride;
  args.y = static_cast<const __nv_bfloat16*>(y);
  args.y_stride = y_stride;
  args.out = static_cast<__nv_bfloat16*>(out);
  args.out_stride = out_stride;
  args.rows = static_cast<int>(rows);
  args.inner = pool->inner;
  args.outer = pool->outer;
  args.rank = pool->rank;
  args.adapters = pool->adapters;
  args.a = static_cast<const __nv_bfloat16*>(pool->a);
  args.b = static_cast<const __nv_bfloat16*>(pool->b);
  args.scales = pool->scales;
  args.ids = ids;
  args.offsets = offsets;
  args.count = count;
  args.inside = static_cast<float*>(workspace);
  args.error = error;
  return status_of(nmoe::launch_adapters(args, static_cast<cudaStream_t>(stream)));
}

nmoe_status nmoe_adapters_sync_status(int32_t* error, void* stream) {
  return nmoe_attention_sync_status(error, stream);
}

nmoe_status nmoe_sample(void* stream, const void* logits, nmoe_dtype dtype, int64_t stride, int64_t rows,
                        int32_t vocab, const float* uniform, const float* temperature,
                        float temperature_all, const int32_t* top_k, int32_t top_k_all,
                        const float* top_p, float top_p_all, const float* min_p, float min_p_all,
                        int32_t* tokens, float* logprobs) {
  const bool bf16 = dtype == NMOE_BF16;
  if ((!bf16 && dtype != NMOE_F32) || rows < 0 || rows > INT32_MAX / 8 || vocab <= 0 || stride < vocab ||
      misaligned(temperature, 4) || misaligned(top_k, 4) || misaligned(top_p, 4) || misaligned(min_p, 4) ||
      misaligned(logprobs, 4) || std::isnan(temperature_all) || std::isnan(top_p_all) || std::isnan(min_p_all)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  if (!nmoe::sample_supported(vocab, bf16)) return NMOE_ERR_UNSUPPORTED;
  if (rows == 0) return NMOE_OK;
  if (logits == nullptr || uniform == nullptr || tokens == nullptr || misaligned(logits, bf16 ? 2 : 4) ||
      misaligned(uniform, 4) || misaligned(tokens, 4)) {
    return NMOE_ERR_INVALID_ARGUMENT;
  }
  nmoe::SampleArgs args;
  args.logits = logits;
  args.stride = stride;
  args.rows = static_cast<int>(rows);
  args.vocab = vocab;
  args.uniform = uniform;
  args.temperature = {temperature, temperature_all};
  args.top_k = {top_k, top_k_all};
  args.top_p = {top_p, top_p_all};
  args.min_p = {min_p, min_p_all};
  args.tokens = tokens;
  args.logprobs = logprobs;
  return status_of(nmoe::launch_sample(args, bf16, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
