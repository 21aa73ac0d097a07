// Appending new tokens to a paged cache: the keys (and the queries) are
// rotated by their positions on the way, keys and values go to their page
// slots, and the per-block key bounds lo / hi are folded in the same pass.
//
// Rotation of pair p of a head, (x, y) -> (x c - y s, y c + x s), with c, s
// the table's entries of pair p at the token's position on the pair's axis
// (one axis: the token's place; several: time, height, width). Pairs are
// (p, p + pairs) of the head's first 2 * pairs dims, or (2p, 2p + 1)
// (`interleaved`). Products and sums are rounded one by one in FP32 (no
// contraction), so the stored keys do not depend on the variant that computed
// them; the result is rounded once to the cache's type, and the bounds are
// those of the rounded keys.
//
// HBM-bound for prompts: every q, k, v element is read and written once, plus
// 8 bytes of table per (token, pair) and 8 bytes of bounds per (block, KV
// head, dim). One CTA takes the new tokens of one block (request, block), so
// a block's bounds have one writer and need no atomics; it stages the
// cosines and sines of its tokens in shared memory once, and each warp then
// takes whole heads: lanes cover a head's 16-byte vectors, two per lane (the
// two halves of a pair in one lane, no shuffles), and several tokens at once.
// Which (request, block) a CTA has follows from token_offsets on the device:
// request r's blocks start at slot offs[r] / B + 2 r, which leaves room for
// the ceil of its tokens wherever its first block begins.

#include <type_traits>

#include "paged_ops.cuh"

namespace stk {

constexpr int kAppendWarps = 8;

// min / max that propagate NaN like torch.amin / amax.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// VEC consecutive elements: one 16-byte access, or one element.
template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Vec {
  T e[VEC];
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kAppendWarps * 32) append_kernel(AppendArgs a, int tile_tokens) {
  // (cos, sin) of pair it * VEC + e of token tk at tk * stride + e * rot_items + it: consecutive lanes read
  // consecutive entries, and the stride's extra rot_items keep a warp's tokens on different banks.
  extern __shared__ float2 turn[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = a.L.b, D = a.L.d;
  int r, t0, n, f;
  if (a.token_offsets == nullptr) {
    r = blockIdx.x;
    t0 = r;
    n = 1;
    f = 0;
  } else {
    r = request_of_slot(a.token_offsets, a.R, 1, B, 2, blockIdx.x, lane);
    t0 = a.token_offsets[r];
    n = a.token_offsets[r + 1] - t0;
    f = blockIdx.x - t0 / B - 2 * r;
  }
  if (n <= 0) return;
  const int len = a.lengths[r];
  if (len < 0) {
    if (tid == 0) report(a.status, kStatusBadLength);
    return;
  }
  const int j = len / B + f;                                 // block of the request
  const int begin = max(len, j * B), end = static_cast<int>(min(static_cast<long long>(len) + n, (j + 1ll) * B));
  if (begin >= end) return;
  const bool room = j < request_blocks(a.L, r);
  if (!room && tid == 0) report(a.status, kStatusBadLength);
  const int ppb = B / a.L.page_size;
  const int base = a.L.block_offsets ? a.L.block_offsets[r] : 0;
  const int* table = a.L.page_table + (static_cast<long long>(base) + j) * ppb;

  const int rot_items = a.cos ? a.pairs / VEC : 0;
  const int stride = a.pairs + rot_items;
  const int tail0 = a.cos ? 2 * a.pairs : 0;                // first dim that passes through
  const int row_items = rot_items + (D - tail0 + 2 * VEC - 1) / (2 * VEC);
  const int copy_items = (D + 2 * VEC - 1) / (2 * VEC);
  const int heads = (a.q ? a.hq : 0) + 2 * a.L.hkv;
  const int hq = a.q ? a.hq : 0;

  for (int tile = begin; tile < end; tile += tile_tokens) {
    const int nt = min(tile_tokens, end - tile);
    if (a.cos) {
      if (tile != begin) __syncthreads();
      for (int i = tid; i < nt * a.pairs; i += blockDim.x) {
        const int tt = i / a.pairs, p = i - tt * a.pairs;
        int pos = tile + tt;
        if (a.positions) {
          const int ax = a.axis ? a.axis[p] : 0;
          pos = ax < a.axes ? a.positions[static_cast<long long>(ax) * a.T + t0 + (tile + tt - len)] : -1;
        }
        if (pos < 0 || pos >= a.max_position) {
          report(a.status, kStatusBadPosition);
          pos = 0;
        }
        const long long o = static_cast<long long>(pos) * a.pairs + p;
        turn[tt * stride + p % VEC * rot_items + p / VEC] = make_float2(a.cos[o], a.sin[o]);
      }
      __syncthreads();
    }
    for (int hd = blockIdx.y * kAppendWarps + warp; hd < heads; hd += gridDim.y * kAppendWarps) {
      // kind 0: query head, 1: key head, 2: value head.
      const int kind = hd < hq ? 0 : hd < hq + a.L.hkv ? 1 : 2;
      const int h = kind == 0 ? hd : kind == 1 ? hd - hq : hd - hq - a.L.hkv;
      if (kind != 0 && !room) continue;
      const T* src = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                     h * (kind == 0 ? a.q_hs : kind == 1 ? a.k_hs : a.v_hs);
      const long long ts = kind == 0 ? a.q_ts : kind == 1 ? a.k_ts : a.v_ts;
      T* dst = static_cast<T*>(kind == 0 ? a.q_out : const_cast<void*>(kind == 1 ? a.L.k : a.L.v));
      const int items = kind == 2 ? copy_items : row_items;
      const int rots = kind == 2 ? 0 : rot_items;
      const int tail = kind == 2 ? 0 : tail0;
      int width = 1;  // lanes along a head's items; the others take further tokens
      while (width < items && width < 32) width <<= 1;
      const int tlanes = 32 / width, li = lane & (width - 1), lt = lane / width;
      for (int it = li; it - li < items; it += width) {
        const bool active = it < items;
        int o1, o2;
        if (it < rots) {
          o1 = a.interleaved ? 2 * it * VEC : it * VEC;
          o2 = a.interleaved ? o1 + VEC : a.pairs + it * VEC;
        } else {
          o1 = tail + 2 * (it - rots) * VEC;
          o2 = o1 + VEC;
        }
        const bool second = o2 < D;
        float mn[2 * VEC], mx[2 * VEC];
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e) {
          mn[e] = __int_as_float(0x7f800000);
          mx[e] = neg_inf();
        }
        if (active) {
          constexpr int U = 4;  // tokens in flight per lane
          for (int tt = lt; tt < nt; tt += U * tlanes) {
            Vec<T, VEC> x[U], y[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int tk = tt + u * tlanes;
              if (tk < nt) {
                const T* s = src + static_cast<long long>(t0 + (tile + tk - len)) * ts;
                x[u] = *reinterpret_cast<const Vec<T, VEC>*>(s + o1);
                if (second) y[u] = *reinterpret_cast<const Vec<T, VEC>*>(s + o2); else y[u] = x[u];
              }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int tk = tt + u * tlanes;
              if (tk >= nt) continue;
              const int at = tile + tk;  // the token's place in its request
              if (it < rots) {
                const float2* cs = turn + tk * stride + it;
                auto pair = [&](T& first, T& other, int e) {
                  const float p = to_f32(first), w = to_f32(other);
                  const float2 c = cs[e * rot_items];
                  first = from_f32<T>(__fsub_rn(__fmul_rn(p, c.x), __fmul_rn(w, c.y)));
                  other = from_f32<T>(__fadd_rn(__fmul_rn(w, c.x), __fmul_rn(p, c.y)));
                };
                if (a.interleaved) {
                  auto at = [&](int i) -> T& { return i < VEC ? x[u].e[i] : y[u].e[i - VEC]; };
#pragma unroll
                  for (int e = 0; e < VEC; ++e) pair(at(2 * e), at(2 * e + 1), e);
                } else {
#pragma unroll
                  for (int e = 0; e < VEC; ++e) pair(x[u].e[e], y[u].e[e], e);
                }
              }
              T* d;
              if (kind == 0) {
                d = dst + (static_cast<long long>(t0 + (at - len)) * a.hq + h) * D;
              } else {
                const int in = at - j * B, pg = in / a.L.page_size;
                const int page = table[pg];
                if (page < 0 || page >= a.pages) {
                  report(a.status, kStatusBadBlockId);
                  continue;
                }
                d = dst + ((static_cast<long long>(page) * a.L.hkv + h) * a.L.page_size + (in - pg * a.L.page_size)) * D;
              }
              *reinterpret_cast<Vec<T, VEC>*>(d + o1) = x[u];
              if (second) *reinterpret_cast<Vec<T, VEC>*>(d + o2) = y[u];
              if (kind == 1) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                  const float p = to_f32(x[u].e[e]), s = to_f32(y[u].e[e]);
                  mn[e] = min_nan(mn[e], p);
                  mx[e] = max_nan(mx[e], p);
                  mn[VEC + e] = min_nan(mn[VEC + e], s);
                  mx[VEC + e] = max_nan(mx[VEC + e], s);
                }
              }
            }
          }
        }
        if (kind == 1 && a.lo != nullptr) {
#pragma unroll
          for (int e = 0; e < 2 * VEC; ++e) {
            for (int o = width; o < 32; o <<= 1) {
              mn[e] = min_nan(mn[e], __shfl_xor_sync(kFull, mn[e], o));
              mx[e] = max_nan(mx[e], __shfl_xor_sync(kFull, mx[e], o));
            }
          }
          if (active && lt == 0) {
            // The block's first token resets its bounds; later tokens fold
            // into them (this warp alone writes this head's bounds).
            const bool fold = tile > j * B;
            const long long o = (static_cast<long long>(h) * a.total + base + j) * D;
#pragma unroll
            for (int e = 0; e < 2 * VEC; ++e) {
              if (e >= VEC && !second) continue;
              const long long at = o + (e < VEC ? o1 + e : o2 + e - VEC);
              a.lo[at] = fold ? min_nan(a.lo[at], mn[e]) : mn[e];
              a.hi[at] = fold ? max_nan(a.hi[at], mx[e]) : mx[e];
            }
          }
        }
      }
    }
  }
}

template <typename T, int VEC>
static int launch_append_t(const AppendArgs& a, cudaStream_t stream) {
  const int slots = a.token_offsets ? a.T / a.L.b + 2 * a.R : a.R;
  const int heads = (a.q ? a.hq : 0) + 2 * a.L.hkv;
  // 32 tokens of tables per tile up to 128 pairs, fewer for wider heads.
  const int pairs = a.cos ? a.pairs : 0;
  const int tile = pairs <= 128 ? 32 : 8;
  const size_t smem = static_cast<size_t>(tile) * (pairs + pairs / VEC) * sizeof(float2);
  auto kern = append_kernel<T, VEC>;
  if (smem > 48 * 1024)
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  const int y = (heads + kAppendWarps - 1) / kAppendWarps;
  kern<<<dim3(static_cast<unsigned>(slots), static_cast<unsigned>(y)), kAppendWarps * 32, smem, stream>>>(a, tile);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
static int launch_append_v(const AppendArgs& a, cudaStream_t stream) {
  // 16-byte vectors where every row of every tensor starts on one and a
  // pair's two vectors stay inside the rotated dims; single elements else.
  constexpr int VEC = 16 / sizeof(T);
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  bool ok = a.L.d % VEC == 0 && a.k_ts % VEC == 0 && a.k_hs % VEC == 0 && a.v_ts % VEC == 0 && a.v_hs % VEC == 0 &&
            aligned(a.k) && aligned(a.v) && aligned(a.L.k) && aligned(a.L.v);
  if (a.q) ok = ok && a.q_ts % VEC == 0 && a.q_hs % VEC == 0 && aligned(a.q) && aligned(a.q_out);
  if (a.cos) ok = ok && a.pairs % VEC == 0;
  return ok ? launch_append_t<T, VEC>(a, stream) : launch_append_t<T, 1>(a, stream);
}

int launch_append_tokens(const AppendArgs& a, int kv_dtype, cudaStream_t stream) {
  switch (kv_dtype) {
    case kF32: return launch_append_v<float>(a, stream);
    case kF16: return launch_append_v<__half>(a, stream);
    default: return launch_append_v<__nv_bfloat16>(a, stream);
  }
}

}  // namespace stk
