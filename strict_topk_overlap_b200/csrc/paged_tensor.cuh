// What the two tensor-core attention kernels over a paged cache share: tensor
// maps of the page pool, score arithmetic in powers of two, and the row-wise
// form for rows whose tile met values that are not finite.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "paged_ops.cuh"

namespace stk {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void tma_load(const CUtensorMap* map, void* dst, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// tanh(x) for capped scores. 1 - 2 / (1 + e^2x) keeps an absolute error of a
// few 2^-24, which the cap turns into the error of a score.
__device__ __forceinline__ float cap_tanh(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2(x * (2.f * kLog2e))));
  return fmaf(-2.f, r, 1.f);
}

// A row recomputed from its own keys [lo, hi), one at a time, by one warp:
// the definition, for rows whose tile sums met values of other rows' keys
// that are not finite. On return every lane has m (natural log), l and its
// D / 32 dims of the sum (dims lane * D / 32 + j).
template <typename T, int D>
__device__ void single_row(const PagedAttnArgs& a, int rp, int h, const T* q, int lo, int hi, int pos, float slope,
                           int lane, float& m, float& l, float (&o)[D / 32]) {
  constexpr int N = D / 32;
  float x[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    x[j] = to_f32(q[lane * N + j]);
    o[j] = 0.f;
  }
  m = neg_inf();
  l = 0.f;
  for (int k = lo; k < hi; ++k) {
    const int page = page_of(a, rp, k);
    if (page < 0) continue;
    const long long at = ((static_cast<long long>(page) * a.L.hkv + h) * a.L.page_size + k % a.L.page_size) * D;
    const T* kr = static_cast<const T*>(a.L.k) + at + lane * N;
    const T* vr = static_cast<const T*>(a.L.v) + at + lane * N;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) s = fmaf(x[j], to_f32(kr[j]), s);
    s = warp_sum(s) * a.scale;
    if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
    if (slope != 0.f) s -= slope * fabsf(static_cast<float>(pos - k));
    const float mn = fmaxf(m, s);
    const float base = mn == neg_inf() ? 0.f : mn;
    const float alpha = expf(m - base), w = expf(s - base);
    l = l * alpha + w;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = o[j] * alpha + (w == 0.f ? 0.f : w * to_f32(vr[j]));
    m = mn;
  }
  m = state_max(m, l);
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// A tensor map over a page pool: (64 dims, box_rows tokens) boxes of one KV
// head's page, 128-byte swizzle.
inline int encode_pool_map(CUtensorMap* map, const PagedAttnArgs& a, const void* pool, int kv_dtype, int box_rows) {
  const EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return static_cast<int>(cudaErrorNotSupported);
  const int ps = a.L.page_size;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.d), static_cast<cuuint64_t>(ps),
                              static_cast<cuuint64_t>(a.L.hkv), static_cast<cuuint64_t>(a.pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(a.d) * 2, static_cast<cuuint64_t>(ps) * a.d * 2,
                                 static_cast<cuuint64_t>(a.L.hkv) * ps * a.d * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, kv_dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                        const_cast<void*>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : static_cast<int>(cudaErrorInvalidValue);
}

}  // namespace stk
