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

}  // namespace

extern "C" {

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
