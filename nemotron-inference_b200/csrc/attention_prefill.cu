// Causal attention over whole prompts packed one behind the other.
#include "attention_simple.cuh"

namespace nmoe {
namespace {

__global__ void __launch_bounds__(kHeadDim) prefill_row_kernel(PrefillArgs args) {
  const int row = blockIdx.x, head = blockIdx.y;
  int sequence = -1, first = 0;
  for (int i = 0; i < args.sequences; ++i) {
    const int from = max(args.offsets[i], 0), to = min(args.offsets[i + 1], args.tokens);
    if (row >= from && row < to) {
      sequence = i;
      first = from;
    }
  }
  if (sequence < 0) return;
  const int kv_head = head / (args.heads / args.kv_heads);
  auto load = [&](int token, int half, int dim, float(&x)[4]) {
    const __nv_bfloat16* from = (half ? args.v + (first + token) * args.v_stride
                                      : args.k + (first + token) * args.k_stride) +
                                kv_head * kHeadDim + dim;
    for (int i = 0; i < 4; ++i) x[i] = __bfloat162float(from[i]);
  };
  const size_t at = static_cast<size_t>(row) * args.heads + head;
  attend_row(args.q + row * args.q_stride + head * kHeadDim, row - first + 1, args.scale, load,
             args.out + at * kHeadDim, args.lse ? args.lse + at : nullptr);
}

}  // namespace

cudaError_t launch_attention_prefill(const PrefillArgs& args, cudaStream_t stream) {
  prefill_row_kernel<<<dim3(args.tokens, args.heads), kHeadDim, 0, stream>>>(args);
  return cudaGetLastError();
}

}  // namespace nmoe
