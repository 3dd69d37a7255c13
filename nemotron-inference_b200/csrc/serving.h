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

// out = y + scale (x A^T) B^T, rows [offsets[i], offsets[i + 1]) by adapter ids[i].
struct AdapterArgs {
  const __nv_bfloat16* x;  // [rows][inner]
  int64_t x_stride;        // elements from row to row
  const __nv_bfloat16* y;  // [rows][outer]
  int64_t y_stride;
  __nv_bfloat16* out;      // [rows][outer], may be y
  int64_t out_stride;
  int rows, inner, outer, rank, adapters;
  const __nv_bfloat16* a;  // [adapters][rank][inner]
  const __nv_bfloat16* b;  // [adapters][outer][rank]
  const float* scales;     // [adapters]
  const int* ids;          // [count]
  const int* offsets;      // [count + 1]
  int count;
  float* inside;           // [splits][rows][rank]: parts of x A^T
  int* error;
};
constexpr int kMostRank = 128;
size_t adapter_workspace_bytes(int64_t rows, int count, int inner, int rank);
cudaError_t launch_adapters(const AdapterArgs& args, cudaStream_t stream);

bool sample_supported(int vocab, bool bf16);
cudaError_t launch_sample(const SampleArgs& args, bool bf16, cudaStream_t stream);

}  // namespace nmoe
