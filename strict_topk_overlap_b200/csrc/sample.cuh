// Arguments of the sampling kernel.
#pragma once

#include "internal.cuh"

namespace stk {

// A parameter of a call: one value for each row, or one for all.
template <typename T>
struct PerRow {
  const T* rows;
  T all;
};

struct SampleArgs {
  const void* logits;  // [R, V], rows `stride` elements apart
  long long stride;
  int R, V;
  const float* uniforms;  // [R] in [0, 1)
  PerRow<float> temperature, top_p, min_p;
  PerRow<int> top_k;
  int* tokens;  // [R]
  int* status;
};

constexpr int kSampleCluster = 8;         // CTAs that share a row at most
constexpr int kSampleBytes = 4 * 49152;   // of its logits that one of them holds in shared memory
constexpr int kSampleMost = kSampleCluster * kSampleBytes / 4;

int launch_sample(const SampleArgs& a, int dtype, int sms, cudaStream_t stream);

}  // namespace stk
