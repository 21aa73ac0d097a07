// What selections by a CTA of 1,024 threads share: order keys of floats, a sort
// of one value to a thread and prefix sums.
#pragma once

#include "common.cuh"

namespace stk {
namespace {

using u64 = unsigned long long;

// Ascending like the floats, zeros of either sign alike (NaN is the caller's).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return x == 0.f ? 0x80000000u : u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// Sorts the first n of the CTA's values, one to a thread, in descending order
// (the others are 0 and stay behind them). Warps without values only meet.
__device__ __forceinline__ u64 sort_descending(u64 x, int n, u64* list) {
  const int tid = threadIdx.x;
  int size = 32;
  while (size < n) size *= 2;
  const bool active = tid < size;
  for (int k = 2; k <= size; k *= 2) {
    int j = k / 2;
    for (; j >= 32; j /= 2) {
      __syncthreads();
      if (active) list[tid] = x;
      __syncthreads();
      if (active) {
        const u64 y = list[tid ^ j];
        const bool keep_large = ((tid & k) == 0) == ((tid & j) == 0);
        x = (x > y) == keep_large ? x : y;
      }
    }
    if (active) {
#pragma unroll 1
      for (; j > 0; j /= 2) {
        const u64 y = __shfl_xor_sync(kFull, x, j);
        const bool keep_large = ((tid & k) == 0) == ((tid & j) == 0);
        x = (x > y) == keep_large ? x : y;
      }
    }
  }
  return x;
}

template <typename T>
__device__ __forceinline__ T scan_add(T v, T* warp_sums, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(kFull, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  T s = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(kFull, s, o);
    if (lane >= o) s += y;
  }
  total = __shfl_sync(kFull, s, 31);
  const T before = __shfl_sync(kFull, s, max(warp - 1, 0));
  return (warp ? before : T{0}) + x - v;
}

}  // namespace
}  // namespace stk
