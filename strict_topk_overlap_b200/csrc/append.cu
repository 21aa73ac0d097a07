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
// head, dim). A CTA takes the new tokens of one block (request, block) and
// eight heads at a time, so a block's bounds have one writer and need no atomics. It
// stages the cosines, sines and page slots of its tokens in shared memory
// once; each warp then takes whole heads: lanes cover a head's 16-byte
// vectors, two per lane (the two halves of a pair in one lane, no shuffles),
// and several tokens at once. Bounds of 16-bit keys are kept as packed pairs
// (the stored values themselves), which halves their registers and leaves
// three CTAs per SM.
// CTAs take equal runs of (block, eight heads) items, so that the last wave is
// as full as the others and a block's tables are staged once; with few items
// (a decode step) each is a CTA of its own and latency is all that counts.
//
// Measured (B200, D 128): 8 tokens, 32 / 8 heads bf16: 7 us, a launch and
// three dependent loads. 8 K prompt tokens of five requests (167 MB): 38 us,
// 4.4 TB/s; the same in FP32: 71 us, 4.7 TB/s. 32 K tokens, 16 / 8 heads f16,
// three axes (552 MB): 113 us, 4.9 TB/s, 75 % of a copy's rate; one item per
// CTA took 126 us, and asking L2 for the next heads' rows ahead 125 us (the
// loads are waited for either way, and the requests compete with the stores).
//
// Which (request, block) an item is follows from token_offsets on the device:
// request r's blocks start at slot offs[r] / B + 2 r, which leaves room for
// the ceil of its tokens wherever its first block begins; padding's "blocks"
// come last.

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

// Running minimum and maximum of a lane's 2 VEC stored keys.
template <typename T, int VEC, bool PACKED = (sizeof(T) == 2 && VEC % 2 == 0)>
struct Bounds {
  float lo[2 * VEC], hi[2 * VEC];
  __device__ __forceinline__ Bounds() {
#pragma unroll
    for (int e = 0; e < 2 * VEC; ++e) {
      lo[e] = __int_as_float(0x7f800000);
      hi[e] = neg_inf();
    }
  }
  __device__ __forceinline__ void add(const Vec<T, VEC>& x, int half) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float v = to_f32(x.e[e]);
      lo[half * VEC + e] = min_nan(lo[half * VEC + e], v);
      hi[half * VEC + e] = max_nan(hi[half * VEC + e], v);
    }
  }
  __device__ __forceinline__ void join(int o) {
#pragma unroll
    for (int e = 0; e < 2 * VEC; ++e) {
      lo[e] = min_nan(lo[e], __shfl_xor_sync(kFull, lo[e], o));
      hi[e] = max_nan(hi[e], __shfl_xor_sync(kFull, hi[e], o));
    }
  }
  __device__ __forceinline__ float low(int e) const { return lo[e]; }
  __device__ __forceinline__ float high(int e) const { return hi[e]; }
};

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  using type = __half2;
  static constexpr uint32_t kInf = 0x7c007c00u;
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static constexpr uint32_t kInf = 0x7f807f80u;
};

template <typename T, int VEC>
struct Bounds<T, VEC, true> {
  using P = typename Pair<T>::type;
  uint32_t lo[VEC], hi[VEC];  // element e in half e & 1 of word e / 2
  __device__ __forceinline__ Bounds() {
#pragma unroll
    for (int w = 0; w < VEC; ++w) {
      lo[w] = Pair<T>::kInf;
      hi[w] = Pair<T>::kInf | 0x80008000u;
    }
  }
  static __device__ __forceinline__ uint32_t least(uint32_t a, uint32_t b) {
    const P r = __hmin2_nan(*reinterpret_cast<const P*>(&a), *reinterpret_cast<const P*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) {
    const P r = __hmax2_nan(*reinterpret_cast<const P*>(&a), *reinterpret_cast<const P*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ __forceinline__ void add(const Vec<T, VEC>& x, int half) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      lo[half * VEC / 2 + i] = least(lo[half * VEC / 2 + i], w[i]);
      hi[half * VEC / 2 + i] = most(hi[half * VEC / 2 + i], w[i]);
    }
  }
  __device__ __forceinline__ void join(int o) {
#pragma unroll
    for (int w = 0; w < VEC; ++w) {
      lo[w] = least(lo[w], __shfl_xor_sync(kFull, lo[w], o));
      hi[w] = most(hi[w], __shfl_xor_sync(kFull, hi[w], o));
    }
  }
  static __device__ __forceinline__ float element(uint32_t w, int e) {
    const unsigned short u = static_cast<unsigned short>(e & 1 ? w >> 16 : w & 0xffffu);
    return to_f32(*reinterpret_cast<const T*>(&u));
  }
  __device__ __forceinline__ float low(int e) const { return element(lo[e / 2], e); }
  __device__ __forceinline__ float high(int e) const { return element(hi[e / 2], e); }
};

// What a CTA's warps share about a tile of new tokens.
struct Tile {
  const float* cosine;     // [nt][pairs]
  const float* sine;
  const long long* slot;   // [nt] element of the page slot in its KV head 0, or -1: not stored
  int nt, pairs, rot_items, tail, D;
  bool interleaved;
};

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// (x, y) -> (x c - y s, y c + x s), each product and sum rounded by itself.
__device__ __forceinline__ float2 turned(float x, float y, float c, float s) {
  return make_float2(__fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s)), __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s)));
}

// Rotates a lane's VEC pairs: element e of x with element e of y, or, when
// interleaved, the neighbours in x and then in y. 16-bit vectors are taken
// word by word (two elements), so that nothing is unpacked beyond a pair.
template <typename T, int VEC>
__device__ __forceinline__ void turn_pairs(Vec<T, VEC>& x, Vec<T, VEC>& y, const float* cosine, const float* sine,
                                           bool interleaved) {
  if constexpr (VEC == 1) {
    const float2 z = turned(to_f32(x.e[0]), to_f32(y.e[0]), cosine[0], sine[0]);
    x.e[0] = from_f32<T>(z.x);
    y.e[0] = from_f32<T>(z.y);
  } else if constexpr (sizeof(T) == 4) {
    const float4 c = *reinterpret_cast<const float4*>(cosine), s = *reinterpret_cast<const float4*>(sine);
    if (interleaved) {
      float2 z = turned(x.e[0], x.e[1], c.x, s.x), w = turned(x.e[2], x.e[3], c.y, s.y);
      x = {z.x, z.y, w.x, w.y};
      z = turned(y.e[0], y.e[1], c.z, s.z);
      w = turned(y.e[2], y.e[3], c.w, s.w);
      y = {z.x, z.y, w.x, w.y};
    } else {
      const float2 z0 = turned(x.e[0], y.e[0], c.x, s.x), z1 = turned(x.e[1], y.e[1], c.y, s.y);
      const float2 z2 = turned(x.e[2], y.e[2], c.z, s.z), z3 = turned(x.e[3], y.e[3], c.w, s.w);
      x = {z0.x, z1.x, z2.x, z3.x};
      y = {z0.y, z1.y, z2.y, z3.y};
    }
  } else {
    uint32_t* xw = reinterpret_cast<uint32_t*>(&x);
    uint32_t* yw = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
    for (int q = 0; q < 2; ++q) {  // pairs 4q .. 4q + 3
      const float4 c = *reinterpret_cast<const float4*>(cosine + 4 * q);
      const float4 s = *reinterpret_cast<const float4*>(sine + 4 * q);
      if (interleaved) {
        uint32_t* w = q == 0 ? xw : yw;
        float2 p = unpack_pair<T>(w[0]), z = turned(p.x, p.y, c.x, s.x);
        w[0] = pack_pair<T>(z.x, z.y);
        p = unpack_pair<T>(w[1]), z = turned(p.x, p.y, c.y, s.y);
        w[1] = pack_pair<T>(z.x, z.y);
        p = unpack_pair<T>(w[2]), z = turned(p.x, p.y, c.z, s.z);
        w[2] = pack_pair<T>(z.x, z.y);
        p = unpack_pair<T>(w[3]), z = turned(p.x, p.y, c.w, s.w);
        w[3] = pack_pair<T>(z.x, z.y);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 p = unpack_pair<T>(xw[2 * q + i]), r = unpack_pair<T>(yw[2 * q + i]);
          const float2 z0 = turned(p.x, r.x, i ? c.z : c.x, i ? s.z : s.x);
          const float2 z1 = turned(p.y, r.y, i ? c.w : c.y, i ? s.w : s.y);
          xw[2 * q + i] = pack_pair<T>(z0.x, z1.x);
          yw[2 * q + i] = pack_pair<T>(z0.y, z1.y);
        }
      }
    }
  }
}

// The rows of one head: rotated (ROT), copied to dst + (slot, or tt * dst_ts),
// and their bounds taken (BOUNDS).
template <typename T, int VEC, bool ROT, bool BOUNDS>
__device__ __forceinline__ void head_rows(const Tile& t, const T* src, long long ts, T* dst, const long long* slot,
                                          long long dst_ts, int lane, float* lo, float* hi, bool fold) {
  const int rots = ROT ? t.rot_items : 0, tail = ROT ? t.tail : 0;
  const int items = rots + (t.D - tail + 2 * VEC - 1) / (2 * VEC);
  int width = 1;  // lanes along a head's items; the others take further tokens
  while (width < items && width < 32) width <<= 1;
  const int step = 32 / width, li = lane & (width - 1), lt = lane / width;
  for (int it = li; it - li < items; it += width) {
    const bool active = it < items, turn = ROT && it < rots;
    int o1, o2;
    if (turn) {
      o1 = t.interleaved ? 2 * it * VEC : it * VEC;
      o2 = t.interleaved ? o1 + VEC : t.pairs + it * VEC;
    } else {
      o1 = tail + 2 * (it - rots) * VEC;
      o2 = o1 + VEC;
    }
    const bool second = o2 < t.D;
    Bounds<T, VEC> bounds;
    constexpr int U = BOUNDS ? 2 : 4;  // tokens in flight per lane
    for (int tt = lt; active && tt < t.nt; tt += U * step) {
      Vec<T, VEC> x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const T* s = src + min(tt + u * step, t.nt - 1) * ts;
        x[u] = *reinterpret_cast<const Vec<T, VEC>*>(s + o1);
        y[u] = *reinterpret_cast<const Vec<T, VEC>*>(second ? s + o2 : s + o1);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int tk = tt + u * step;
        if (tk >= t.nt) break;
        if (turn) turn_pairs<T, VEC>(x[u], y[u], t.cosine + tk * t.pairs + it * VEC, t.sine + tk * t.pairs + it * VEC,
                                     t.interleaved);
        const long long to = slot ? slot[tk] : tk * dst_ts;
        if (to < 0) continue;
        *reinterpret_cast<Vec<T, VEC>*>(dst + to + o1) = x[u];
        if (second) *reinterpret_cast<Vec<T, VEC>*>(dst + to + o2) = y[u];
        if constexpr (BOUNDS) {
          bounds.add(x[u], 0);
          bounds.add(y[u], 1);
        }
      }
    }
    if constexpr (BOUNDS) {
      __syncwarp();
      for (int o = width; o < 32; o <<= 1) bounds.join(o);
      if (active && lt == 0) {
        // The block's first token resets its bounds; later tokens fold into
        // them (this warp alone writes this head's bounds).
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e) {
          if (e >= VEC && !second) continue;
          const int at = e < VEC ? o1 + e : o2 + e - VEC;
          lo[at] = fold ? min_nan(lo[at], bounds.low(e)) : bounds.low(e);
          hi[at] = fold ? max_nan(hi[at], bounds.high(e)) : bounds.high(e);
        }
      }
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kAppendWarps * 32, VEC > 1 ? 3 : 2)
append_kernel(AppendArgs a, int tile_tokens, int chunks, int items) {
  extern __shared__ float tables[];  // cosines, then sines, of tile_tokens tokens
  __shared__ long long page_slot[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = a.L.b, D = a.L.d, hkv = a.L.hkv, ps = a.L.page_size;
  Tile t;
  t.pairs = a.cos ? a.pairs : 0;
  t.rot_items = t.pairs / VEC;
  t.tail = 2 * t.pairs;
  t.D = D;
  t.interleaved = a.interleaved != 0;
  float* cosine = tables;
  float* sine = tables + tile_tokens * t.pairs;
  t.cosine = cosine;
  t.sine = sine;
  t.slot = page_slot;
  const int hq = a.q ? a.hq : 0, heads = hq + 2 * hkv;
  // Items (slot, chunk of heads) in order; a run of chunks of one slot shares its tables.
  const int per = (items + gridDim.x - 1) / gridDim.x;
  const int last = min(items, static_cast<int>(blockIdx.x + 1) * per);
  int at = -1, staged = -1;
  int r = 0, t0 = 0, n = 0, len = 0, j = 0, begin = 0, end = 0, base = 0;
  bool room = false, padding = false;
  const int* table = nullptr;
  for (int item = blockIdx.x * per; item < last; ++item) {
    const int slot = item / chunks, chunk = item - slot * chunks;
    if (slot != at) {
      at = slot;
      int f = 0;
      if (a.token_offsets == nullptr) {
        r = t0 = slot;
        n = 1;
      } else {
        r = request_of_slot(a.token_offsets, a.R + 1, 1, B, 2, slot, lane);
        const int2 tn = new_tokens(a.token_offsets, r, a.R, a.T, a.status);
        t0 = tn.x;
        n = tn.y;
        f = slot - t0 / B - 2 * r;
      }
      padding = r >= a.R;  // tokens of no request: stored nowhere, their q turned by position 0
      len = padding ? 0 : a.lengths[r];
      base = a.L.block_offsets[r];
      const int blocks = padding ? 0 : a.L.block_offsets[r + 1] - base;
      begin = end = 0;
      if (n > 0 && len >= 0 && f >= 0) {
        j = len / B + f;  // block of the request
        begin = max(len, j * B);
        end = static_cast<int>(min(static_cast<long long>(len) + n, (j + 1ll) * B));
      }
      room = j < blocks;
      if (tid == 0 && n > 0 && !padding && (len < 0 || (begin < end && !room))) report(a.status, kStatusBadLength);
      table = a.L.page_table + (static_cast<long long>(base) + j) * (B / ps);
    }
    for (int tile = begin; tile < end; tile += tile_tokens) {
      t.nt = min(tile_tokens, end - tile);
      const int token = t0 + (tile - len);  // packed token of the tile's first
      if (staged != slot || end - begin > tile_tokens) {
        staged = slot;
        __syncthreads();
        if (tid < t.nt) {
          const int in = tile + tid - j * B, pg = in / ps;
          const int page = room ? table[pg] : -1;
          if (room && (page < 0 || page >= a.pages)) report(a.status, kStatusBadBlockId);
          page_slot[tid] =
              page < 0 || page >= a.pages ? -1 : (static_cast<long long>(page) * hkv * ps + (in - pg * ps)) * D;
        }
        for (int tt = warp; tt < t.nt; tt += kAppendWarps) {
          for (int p = lane; p < t.pairs; p += 32) {
            int pos = padding ? 0 : tile + tt;
            if (a.positions && !padding) {
              const int ax = a.axis ? a.axis[p] : 0;
              pos = ax < a.axes ? a.positions[static_cast<long long>(ax) * a.T + token + tt] : -1;
            }
            if (pos < 0 || pos >= a.max_position) {
              report(a.status, kStatusBadPosition);
              pos = 0;
            }
            const long long o = static_cast<long long>(pos) * t.pairs + p;
            cosine[tt * t.pairs + p] = a.cos[o];
            sine[tt * t.pairs + p] = a.sin[o];
          }
        }
        __syncthreads();
      }
      const int hd = chunk * kAppendWarps + warp;
      if (hd < hq) {
        const T* src = static_cast<const T*>(a.q) + token * a.q_ts + hd * a.q_hs;
        T* dst = static_cast<T*>(a.q_out) + (static_cast<long long>(token) * a.hq + hd) * D;
        head_rows<T, VEC, true, false>(t, src, a.q_ts, dst, nullptr, static_cast<long long>(a.hq) * D, lane, nullptr,
                                       nullptr, false);
      } else if (hd < hq + hkv) {
        const int h = hd - hq;
        const T* src = static_cast<const T*>(a.k) + token * a.k_ts + h * a.k_hs;
        T* dst = static_cast<T*>(const_cast<void*>(a.L.k)) + static_cast<long long>(h) * ps * D;
        const long long o = (static_cast<long long>(h) * a.total + base + j) * D;
        if (a.lo != nullptr && room)
          head_rows<T, VEC, true, true>(t, src, a.k_ts, dst, page_slot, 0, lane, a.lo + o, a.hi + o, tile > j * B);
        else
          head_rows<T, VEC, true, false>(t, src, a.k_ts, dst, page_slot, 0, lane, nullptr, nullptr, false);
      } else if (hd < heads) {
        const int h = hd - hq - hkv;
        const T* src = static_cast<const T*>(a.v) + token * a.v_ts + h * a.v_hs;
        T* dst = static_cast<T*>(const_cast<void*>(a.L.v)) + static_cast<long long>(h) * ps * D;
        head_rows<T, VEC, false, false>(t, src, a.v_ts, dst, page_slot, 0, lane, nullptr, nullptr, false);
      }
    }
  }
}

template <typename T, int VEC>
static int launch_append_t(const AppendArgs& a, int sms, cudaStream_t stream) {
  const int slots = a.token_offsets ? a.T / a.L.b + 2 * a.R + 1 : a.R;
  const int heads = (a.q ? a.hq : 0) + 2 * a.L.hkv;
  // 32 tokens of tables per tile up to 128 pairs, 8 for wider heads: at most 32 KB.
  const int pairs = a.cos ? a.pairs : 0;
  const int tile = pairs <= 128 ? 32 : 8;
  const size_t smem = static_cast<size_t>(tile) * pairs * sizeof(float2);
  auto kern = append_kernel<T, VEC>;
  // One item (a slot's eight heads, one per warp) per CTA while that leaves
  // SMs free; beyond, equal runs of items for the CTAs that fit.
  const int chunks = (heads + kAppendWarps - 1) / kAppendWarps;
  const long long items = static_cast<long long>(slots) * chunks;
  if (items > 0x3fffffff) return static_cast<int>(cudaErrorInvalidValue);
  const long long fit = 3ll * sms;
  kern<<<static_cast<unsigned>(items < fit ? items : fit), kAppendWarps * 32, smem, stream>>>(a, tile, chunks,
                                                                                              static_cast<int>(items));
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
static int launch_append_v(const AppendArgs& a, int sms, cudaStream_t stream) {
  // 16-byte vectors where every row of every tensor starts on one and a
  // pair's two vectors stay inside the rotated dims; single elements else.
  constexpr int VEC = 16 / sizeof(T);
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  bool ok = a.L.d % VEC == 0 && a.k_ts % VEC == 0 && a.k_hs % VEC == 0 && a.v_ts % VEC == 0 && a.v_hs % VEC == 0 &&
            aligned(a.k) && aligned(a.v) && aligned(a.L.k) && aligned(a.L.v);
  if (a.q) ok = ok && a.q_ts % VEC == 0 && a.q_hs % VEC == 0 && aligned(a.q) && aligned(a.q_out);
  if (a.cos) ok = ok && a.pairs % VEC == 0;
  return ok ? launch_append_t<T, VEC>(a, sms, stream) : launch_append_t<T, 1>(a, sms, stream);
}

int launch_append_tokens(const AppendArgs& a, int kv_dtype, int sms, cudaStream_t stream) {
  switch (kv_dtype) {
    case kF32: return launch_append_v<float>(a, sms, stream);
    case kF16: return launch_append_v<__half>(a, sms, stream);
    default: return launch_append_v<__nv_bfloat16>(a, sms, stream);
  }
}

}  // namespace stk
