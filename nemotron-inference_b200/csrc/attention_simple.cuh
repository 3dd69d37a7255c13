// One query row and head per block: scores by warp, an online softmax per warp, joined at the end.
#pragma once
#include "attention.h"

namespace nmoe {

constexpr int kRowWarps = 4;

// Load(token, half, dims of this lane) -> four values of a token's key or value.
template <typename Load>
__device__ __forceinline__ void attend_row(const __nv_bfloat16* q, int tokens, float scale, Load load,
                                           __nv_bfloat16* out, float* lse) {
  __shared__ float part[kRowWarps][kHeadDim + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float qv[4], acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < 4; ++i) qv[i] = __bfloat162float(q[lane * 4 + i]) * scale;
  float top = -INFINITY, sum = 0.0f;
  for (int t = warp; t < tokens; t += kRowWarps) {
    float x[4];
    load(t, 0, lane * 4, x);
    float dot = qv[0] * x[0] + qv[1] * x[1] + qv[2] * x[2] + qv[3] * x[3];
    for (int step = 16; step > 0; step /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, step);
    const float higher = fmaxf(top, dot);
    const float keep = top == -INFINITY ? 0.0f : expf(top - higher);
    const float p = expf(dot - higher);
    top = higher;
    sum = sum * keep + p;
    load(t, 1, lane * 4, x);
    for (int i = 0; i < 4; ++i) acc[i] = acc[i] * keep + p * x[i];
  }
  for (int i = 0; i < 4; ++i) part[warp][lane * 4 + i] = acc[i];
  if (lane == 0) {
    part[warp][kHeadDim] = top;
    part[warp][kHeadDim + 1] = sum;
  }
  __syncthreads();
  float all = -INFINITY;
  for (int w = 0; w < kRowWarps; ++w) all = fmaxf(all, part[w][kHeadDim]);
  float value = 0.0f, total = 0.0f;
  for (int w = 0; w < kRowWarps; ++w) {
    if (part[w][kHeadDim + 1] == 0.0f) continue;  // this warp saw no token
    const float f = expf(part[w][kHeadDim] - all);
    value += f * part[w][threadIdx.x];
    total += f * part[w][kHeadDim + 1];
  }
  out[threadIdx.x] = __float2bfloat16(tokens > 0 ? value / total : 0.0f);
  if (lse != nullptr && threadIdx.x == 0) *lse = all + logf(total);
}

}  // namespace nmoe
