// Internal declarations of the operators of a decode step for many requests: sampling, low-rank adapters.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace nmoe {

// A parameter of each row, or one for all where `rows` is null.
template <typename T>
struct RowParameter {
  const T* rows;
  T all;
  __host__ __device__ T of(int row) const { return rows != nullptr ? rows[row] : all; }
};

struct SampleArgs {
  const void* logits;
  int64_t stride;  // elements from row to row
  int rows, vocab;
  const float* uniform;
  RowParameter<float> temperature;
  RowParameter<int> top_k;
  RowParameter<float> top_p, min_p;
  int* tokens;
  float* logprobs;  // may be null
};

bool sample_supported(int vocab, bool bf16);
cudaError_t launch_sample(const SampleArgs& args, bool bf16, cudaStream_t stream);

}  // namespace nmoe
