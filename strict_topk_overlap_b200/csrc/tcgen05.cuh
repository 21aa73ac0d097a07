// Tensor-core (tcgen05) and tensor-memory primitives, bounded waits of whole
// warps and FP32 arithmetic in pairs, as the kernels on them share them.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace stk {
namespace {

// ---------------------------------------------------------------- tcgen05
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, int columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t at, int columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Issued by one elected lane, as a predicate inside warp-uniform code: with a
// branch around them, their uniform operands are moved lane by lane and the
// issue, not the tensor cores, bounds the kernel (100 instead of 64 clocks
// per 128 x 128 x 16 product).
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.u32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc))
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.u32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc))
      : "memory");
}

// 32 consecutive columns of the warp's 32 lanes: element j of lane i is
// column at + j of TMEM lane 32 (warp % 4) + i.
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// The registers of a load, after its wait: keeps their uses behind it.
template <int N = 32>
__device__ __forceinline__ void tmem_loaded(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                      "+r"(r[i + 6]), "+r"(r[i + 7]));
}
// Whether x holds for any thread of a group of `count` that meets on named
// barrier `id`. What one half's threads know of finished products, and their
// own accesses to tensor memory, are ordered before the other's after it.
__device__ __forceinline__ bool group_any(int id, int count, bool x) {
  uint32_t r;
  fence_before();
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n barrier.cta.red.or.pred p, %2, %3, q;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(x)), "r"(id), "r"(count)
      : "memory");
  fence_after();
  return r != 0;
}
// The value of lane 0, known to the compiler as the warp's.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(kFull, x, 0); }
// A bounded wait of a whole warp, converged again on return.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, unsigned parity, int* status) {
  return __all_sync(kFull, mbar_wait(bar, parity, status));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle (rows of 128 bytes,
// groups of 8 rows 1024 bytes apart); `lead` bytes between the 64-element
// column groups of an operand whose rows run along the contraction (V).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | static_cast<uint64_t>(lead >> 4) << 16 |
         static_cast<uint64_t>(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// Instruction descriptor of kind::f16 with FP32 accumulators.
template <typename T>
constexpr uint32_t mma_desc(int m, int n, bool b_along_n) {
  const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return 1u << 4 | fmt << 7 | fmt << 10 | (b_along_n ? 1u : 0u) << 16 | static_cast<uint32_t>(n >> 3) << 17 |
         static_cast<uint32_t>(m >> 4) << 24;
}

// ---------------------------------------------------------------- pairs of FP32
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 c, a, b, c;\n mov.b64 {%0, %1}, c;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 a, b;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
      " mul.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 a, b;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
      " add.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// 2^x of a pair on the FMA units: x = n + f with |f| <= 1/2 (n by adding and
// subtracting 1.5 * 2^23), 2^f by a quartic that is 1 at 0 (weighted
// least-maximum fit on [-1/2, 1/2], relative error 2.9e-6, far below a 16-bit
// weight's rounding), n added to the exponent. x is clamped to [-127, 128],
// where 1 becomes an exact 0 and infinity: a masked key's -inf has no weight at
// all, whatever its value holds. NaN comes out as NaN (the clamp passes it on;
// the last addition undoes what the exponent did to it). The special function
// unit yields 16 exponentials per SM and clock, as many as the tensor cores
// need weights.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
  asm("{\n .reg .f32 t;\n max.NaN.f32 t, %2, %4;\n min.NaN.f32 %0, t, %5;\n max.NaN.f32 t, %3, %4;\n min.NaN.f32 %1, t, %5;\n}\n"
      : "=f"(x.x), "=f"(x.y)
      : "f"(x.x), "f"(x.y), "f"(-127.f), "f"(128.f));
  const float2 t = add2(x, both(12582912.f));
  const float2 n = add2(t, both(-12582912.f));
  const float2 f = fma2(n, both(-1.f), x);
  float2 p = fma2(f, both(0.009582853f), both(0.055906426f));
  p = fma2(p, f, both(0.24024099f));
  p = fma2(p, f, both(0.6931242f));
  p = fma2(p, f, both(1.f));
  p = make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                  __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
  return fma2(x, both(0.f), p);
}

}  // namespace
}  // namespace stk
