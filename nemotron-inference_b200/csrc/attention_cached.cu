// Attention of new rows over the paged 8-bit cache.
#include "attention_simple.cuh"
#include "common.cuh"

namespace nmoe {
namespace {

__global__ void __launch_bounds__(kHeadDim) cached_row_kernel(CachedArgs args) {
  const PagedCache& c = args.cache;
  const int row = blockIdx.x, head = blockIdx.y;
  const int2 unit = locate_unit(args.batch.count, row,
                                [&](int i) {
                                  const BatchEntry e = batch_entry(c, args.batch, i);
                                  if (!e.valid) report_cache_error(c.error, kCacheBadSequence);
                                  return e.rows;
                                });
  if (unit.x < 0) return;
  const BatchEntry e = batch_entry(c, args.batch, unit.x);
  const int tokens = e.length - e.rows + unit.y + 1;
  const int kv_head = head / (args.heads / c.kv_heads);
  auto load = [&](int token, int half, int dim, float(&x)[4]) {
    const int page = page_at(c, e.sequence, token >> c.page_shift);
    if (page < 0) {
      report_cache_error(c.error, kCacheBadSequence);
      x[0] = x[1] = x[2] = x[3] = 0.0f;
      return;
    }
    const size_t block = block_of_page(c, args.layer, page, half, kv_head);
    const float scale = exp2f(static_cast<float>(c.exponents[block]));
    const uint8_t* from =
        c.codes + (block * c.page_tokens + (token & (c.page_tokens - 1))) * kHeadDim + dim;
    for (int i = 0; i < 4; ++i) x[i] = decode_e4m3(from[i]) * scale;
  };
  const size_t at = static_cast<size_t>(e.first + unit.y);
  attend_row(args.q + at * args.q_stride + head * kHeadDim, tokens, args.scale, load,
             args.out + (at * args.heads + head) * kHeadDim, nullptr);
}

}  // namespace

size_t attention_cached_workspace_bytes() { return 0; }

cudaError_t launch_attention_cached(const CachedArgs& args, cudaStream_t stream) {
  cached_row_kernel<<<dim3(args.batch.rows, args.heads), kHeadDim, 0, stream>>>(args);
  return cudaGetLastError();
}

}  // namespace nmoe
