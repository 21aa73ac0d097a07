// Dense paged attention of few rows per KV head (at most 16: single tokens,
// a few drafted ones), HBM-bound: every key and value is read once per KV head.
//
// The work of a batch is the list of all (request, KV head, 16 keys) units in
// order; the warps of a persistent grid cut it into equal runs, so that
// requests of any lengths load every SM alike and no warp waits for another.
// Each CTA finds its warps' runs from the requests' key ranges (a prefix sum
// over the batch, taken by every CTA). A warp streams its keys through a ring
// of its own (TMA boxes of 16 keys x 64 dims, swizzled for ldmatrix, page ids
// looked up one unit ahead) across the borders of requests and heads.
// The rows form the 16-row side of mma.sync tiles, which hold up to 16 query
// heads whatever their number and are far from bounding the kernel; the
// online softmax is FP32, P rounded to the type. Where a (request, head) ends
// inside a run, its state goes to one partial; the join kernel adds the
// partials of each row.
//
// Measured (B200, bf16, D 128): 64 requests of 8-32 K tokens, 16 / 8 heads
// (5.1 GB): 800 us with the join, 6.4 TB/s, 97 % of a copy's rate. One request
// of 65,536 tokens, 32 / 8 heads, capped: 57 us, 4.7 TB/s; the other 16 us are
// launches, the first loads and the join. The tcgen05 kernel on the same
// calls, its 128-row tiles mostly empty: 1,317 and 85 us (and 184 against 92
// us for 12 heads a group), so it takes over above 16 rows only. Runs of
// whole CTAs with a join of their four warps took 65 us for the long request
// and 36 % more for many short ones.
//
// Values past the keys that any row sees are zeroed in shared memory. Rows of
// several tokens that see different keys are recomputed one by one where a
// value that is not finite made their sum NaN.

#include "paged_tensor.cuh"

namespace stk {

int set_wait_limit_token(unsigned long long ns) { return set_wait_limit_this_unit(ns); }

namespace {

constexpr int kWarps = 4;
constexpr int kUnit = 16;  // keys of a unit
constexpr int kMostRequests = 16384;

template <int D>
struct TokenPlan {
  static constexpr int kHalves = D / 64;
  static constexpr int kStage = 2 * kUnit * D * 2;              // K and V of a unit
  static constexpr int kStages = D == 128 ? 3 : 6;              // per warp: 96 KB per CTA, two CTAs per SM
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kBytes = kRing + 1024;                    // + alignment of the swizzle atoms
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The new tokens of request r and the keys [kmin, kmax) that any of them sees.
struct Request {
  RowTile t;
  int kmin, kmax;
  int pos;  // of the last of them
};

// (A request with more rows than the call's max_tokens allows keeps its first ones and is reported.)
__device__ __forceinline__ Request request_at(const PagedAttnArgs& a, int r, int most_rows) {
  Request q;
  q.t.r = a.shared ? 0 : r;
  q.t.row0 = 0;
  const int2 tn = a.shared ? make_int2(0, a.T) : new_tokens(a.token_offsets, r, a.R, a.T, a.status);
  q.t.t0 = tn.x;
  q.t.n = tn.y;
  q.t.rows = min(q.t.n * a.G, most_rows);
  if (q.t.n * a.G > most_rows) report(a.status, kStatusShapeOverflow);
  q.t.len = a.shared ? request_blocks(a.L, 0) * a.L.b : q.t.n > 0 ? cached_tokens(a, r, q.t.n) : 0;
  q.kmin = 0x7fffffff;
  q.kmax = q.pos = 0;
  for (int i = 0; i * a.G < q.t.rows; ++i) {
    const RowKeys k = row_keys(a, q.t, i);
    q.pos = k.pos;
    if (k.hi > k.lo) {
      q.kmin = min(q.kmin, k.lo);
      q.kmax = max(q.kmax, k.hi);
    }
  }
  if (q.kmax == 0) q.kmin = 0;
  return q;
}

__device__ __forceinline__ int units_of(const Request& q) { return (q.kmax + kUnit - 1) / kUnit - q.kmin / kUnit; }

// A walk over the run's units in order: (request, head, unit of the request).
struct Walk {
  int r, h, u, units;
  Request q;
  __device__ __forceinline__ void start(const PagedAttnArgs& a, const int* prefix, int requests, int most_rows,
                                        long long at) {
    int lo = 0, hi = requests;  // the request with prefix[r] * hkv <= at < prefix[r + 1] * hkv
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (static_cast<long long>(prefix[mid]) * a.L.hkv <= at) lo = mid; else hi = mid;
    }
    r = lo;
    units = prefix[r + 1] - prefix[r];
    const int in = static_cast<int>(at - static_cast<long long>(prefix[r]) * a.L.hkv);
    h = in / units;
    u = in - h * units;
    q = request_at(a, r, most_rows);
  }
  __device__ __forceinline__ void next(const PagedAttnArgs& a, const int* prefix, int requests, int most_rows) {
    if (++u < units) return;
    u = 0;
    if (++h < a.L.hkv) return;
    h = 0;
    do {
      ++r;
    } while (r < requests && prefix[r + 1] == prefix[r]);
    if (r < requests) {
      units = prefix[r + 1] - prefix[r];
      q = request_at(a, r, most_rows);
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32, 2)
token_attn_kernel(const PagedAttnArgs a, int requests, int most_rows, int* prefix_out,
                  const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using P = TokenPlan<D>;
  constexpr int NT = D / 8;
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t bars[kWarps][P::kStages];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  int* prefix = reinterpret_cast<int*>(base + P::kRing);  // [requests + 1] units before each request
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int i = 0; i < P::kStages; ++i) mbar_init(&bars[w][i], 1);
    fence_barrier_init();
  }
  for (int r = tid; r < requests; r += blockDim.x) prefix[r + 1] = units_of(request_at(a, r, most_rows));
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    for (int r0 = 0; r0 < requests; r0 += 32) {
      int x = r0 + lane < requests ? prefix[r0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(kFull, x, o);
        if (lane >= o) x += y;
      }
      if (r0 + lane < requests) prefix[r0 + lane + 1] = carry + x;
      carry += __shfl_sync(kFull, x, 31);
    }
    if (lane == 0) prefix[0] = 0;
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int r = tid; r <= requests; r += blockDim.x) prefix_out[r] = prefix[r];
  const long long total = static_cast<long long>(prefix[requests]) * a.L.hkv;
  const int stream = blockIdx.x * kWarps + warp, streams = gridDim.x * kWarps;
  const long long per = (total + streams - 1) / streams;
  const long long first = min(total, stream * per), last = min(total, first + per);
  if (first >= last) {
    if (a.chained) pdl_wait();
    return;
  }
  const int jobs = static_cast<int>(last - first);

  // ---- this warp's stream of units, issued kStages ahead
  const int ppb = a.L.b / a.L.page_size;
  unsigned char* ring = base + warp * P::kStages * P::kStage;
  Walk ahead;
  ahead.start(a, prefix, requests, most_rows, first);
  int issued = 0;  // units asked for
  int page = 0, key = 0, head = 0;
  // The place of the next unit to ask for; the page id arrives while others are computed.
  auto find = [&]() {
    const int k = (ahead.q.kmin / kUnit + ahead.u) * kUnit;
    const int rp = ahead.q.t.r;
    // In the table: kmax is at most the request's room.
    page = a.L.page_table[static_cast<long long>(a.L.block_offsets[rp]) * ppb + k / a.L.page_size];
    key = k % a.L.page_size;
    head = ahead.h;
  };
  auto issue = [&]() {
    if (lane == 0) {
      const int slot = issued % P::kStages;
      if (page < 0 || page >= a.pages) {
        report(a.status, kStatusBadBlockId);
        page = a.pages;  // reads as zeros
      }
      unsigned char* dst = ring + slot * P::kStage;
      mbar_arrive_expect_tx(&bars[warp][slot], P::kStage);
#pragma unroll
      for (int half = 0; half < P::kHalves; ++half) {
        tma_load(&kmap, dst + half * 2048, &bars[warp][slot], half * 64, key, head, page);
        tma_load(&vmap, dst + P::kStage / 2 + half * 2048, &bars[warp][slot], half * 64, key, head, page);
      }
    }
    if (++issued < jobs) {
      ahead.next(a, prefix, requests, most_rows);
      find();
    }
  };
  find();
  for (int i = 0; i < P::kStages && issued < jobs; ++i) issue();

  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t sring = smem_u32(ring);
  Walk walk;
  walk.start(a, prefix, requests, most_rows, first);
  int taken = 0;  // chunks consumed
  bool ok = true;
  for (int done = 0; done < jobs;) {
    const Request q = walk.q;
    const int h = walk.h, u0 = walk.u, slot_rh = walk.r * a.L.hkv + walk.h;
    const int u1 = min(walk.units, u0 + (jobs - done));
    if (done + (u1 - u0) >= jobs) pdl_release();  // the join may be launched: it waits for the states
    // ---- rows g and g + 8 of the tile: their queries, keys and slopes
    uint32_t qf[D / 16][4];
    RowKeys rk[2];
    float slope[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = g + 8 * x;
      const bool have = row < q.t.rows;
      const int tok = have ? row / a.G : 0, hd = h * a.G + (have ? row - tok * a.G : 0);
      rk[x] = !have ? RowKeys{0, 0, 0} : q.t.n == 1 ? RowKeys{q.kmin, q.kmax, q.pos} : row_keys(a, q.t, tok);
      slope[x] = a.slopes && have ? a.slopes[hd] * kLog2e : 0.f;
      const T* src = static_cast<const T*>(a.q) + (q.t.t0 + tok) * a.q_ts + hd * a.q_hs + t4 * 2;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[ks][x] = have ? *reinterpret_cast<const uint32_t*>(src + ks * 16) : 0u;
        qf[ks][2 + x] = have ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8) : 0u;
      }
    }
    float o[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {neg_inf(), neg_inf()}, l[2] = {0.f, 0.f};
    const float c = a.softcap > 0.f ? a.scale / a.softcap : a.scale * kLog2e, cap2 = a.softcap * kLog2e;
    for (int u = u0; u < u1; ++u) {
      const int k0 = (q.kmin / kUnit + u) * kUnit;
      const int slot = taken % P::kStages;
      ok = ok && __all_sync(kFull, mbar_wait(&bars[warp][slot], (taken / P::kStages) & 1, a.status));
      ++taken;
      if (!ok) break;
      const uint32_t ks = sring + slot * P::kStage, vs = ks + P::kStage / 2;
      if (k0 < q.kmin || k0 + kUnit > q.kmax) {  // values that no row sees may be anything
        unsigned char* v = ring + slot * P::kStage + P::kStage / 2;
        for (int x = lane; x < kUnit * 8 * P::kHalves; x += 32) {
          const int y = x / (8 * P::kHalves);
          if (k0 + y < q.kmin || k0 + y >= q.kmax)
            *reinterpret_cast<uint4*>(v + x % P::kHalves * 2048 + y * 128 + x / P::kHalves % 8 * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the stage's next copy
        __syncwarp();
      }
      // ---- S = Q K^T: two tiles of 8 keys
      float s[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
        const int row = n * 8 + (lane & 7);
#pragma unroll
        for (int kp = 0; kp < D / 32; ++kp) {
          const int ch = kp * 4 + (lane >> 3);
          uint32_t b[4];
          ldsm4(b, ks + (ch >> 3) * 2048 + row * 128 + (((ch ^ row) & 7) << 4));
          mma<T>(s[n], qf[2 * kp], b[0], b[1]);
          mma<T>(s[n], qf[2 * kp + 1], b[2], b[3]);
        }
      }
      // ---- scores of rows g (e < 2) and g + 8, keys 8 n + 2 t4 + (e & 1)
      float mx[2] = {neg_inf(), neg_inf()};
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = k0 + n * 8 + t4 * 2 + (e & 1), x = e >> 1;
          float v = s[n][e] * c;
          if (a.softcap > 0.f) v = cap2 * cap_tanh(v);
          if (a.slopes) v = fmaf(-slope[x], fabsf(static_cast<float>(rk[x].pos - k)), v);
          v = k >= rk[x].lo && k < rk[x].hi ? v : neg_inf();
          s[n][e] = v;
          mx[x] = fmaxf(mx[x], v);
        }
      }
      float nm[2], alpha[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        mx[x] = fmaxf(mx[x], __shfl_xor_sync(kFull, mx[x], 1));
        mx[x] = fmaxf(mx[x], __shfl_xor_sync(kFull, mx[x], 2));
        mx[x] = fmaxf(m[x], mx[x]);
        nm[x] = mx[x] == neg_inf() ? 0.f : -mx[x];
        alpha[x] = ex2(m[x] + nm[x]);
      }
      if (__any_sync(kFull, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          o[n][0] *= alpha[0];
          o[n][1] *= alpha[0];
          o[n][2] *= alpha[1];
          o[n][3] *= alpha[1];
        }
      }
      uint32_t p[4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float p0 = ex2(s[0][2 * x] + nm[x]), p1 = ex2(s[0][2 * x + 1] + nm[x]);
        const float p2 = ex2(s[1][2 * x] + nm[x]), p3 = ex2(s[1][2 * x + 1] + nm[x]);
        p[x] = pack2<T>(p0, p1);
        p[2 + x] = pack2<T>(p2, p3);
        l[x] = l[x] * alpha[x] + ((p0 + p1) + (p2 + p3));
        m[x] = mx[x];
      }
      // ---- O += P V
#pragma unroll
      for (int np = 0; np < NT / 2; ++np) {
        const int row = lane & 15, ch = 2 * np + (lane >> 4);
        uint32_t b[4];
        ldsm4_t(b, vs + (ch >> 3) * 2048 + row * 128 + (((ch ^ row) & 7) << 4));
        mma<T>(o[2 * np], p, b[0], b[1]);
        mma<T>(o[2 * np + 1], p, b[2], b[3]);
      }
      __syncwarp();  // every lane has read the stage
      if (issued < jobs) issue();
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(kFull, l[x], 1);
      l[x] += __shfl_xor_sync(kFull, l[x], 2);
    }
    if (ok) {
      const long long slot = static_cast<long long>(stream) + slot_rh;
      unsigned redo = 0;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = g + 8 * x;
        if (row < q.t.rows) {
          const long long at = slot * most_rows + row;
          if (t4 == 0) a.part_ml[at] = make_float2(m[x] * kLn2, l[x]);
          bool nan = false;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 v = make_float2(o[n][2 * x], o[n][2 * x + 1]);
            nan = nan || v.x != v.x || v.y != v.y;
            *reinterpret_cast<float2*>(a.part_o + at * D + n * 8 + t4 * 2) = v;
          }
          redo |= nan ? 1u << row : 0u;
        }
      }
      redo = __reduce_or_sync(kFull, redo);
      while (redo) {
        const int row = __ffs(redo) - 1;
        redo &= redo - 1;
        const int tok = row / a.G, hd = h * a.G + row - tok * a.G;
        const RowKeys k = row_keys(a, q.t, tok);
        float xm, xl, xo[D / 32];
        single_row<T, D>(a, q.t.r, h, static_cast<const T*>(a.q) + (q.t.t0 + tok) * a.q_ts + hd * a.q_hs,
                         max(k.lo, (q.kmin / kUnit + u0) * kUnit), min(k.hi, (q.kmin / kUnit + u1) * kUnit), k.pos,
                         a.slopes ? a.slopes[hd] : 0.f, lane, xm, xl, xo);
        const long long at = slot * most_rows + row;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < D / 32; ++j) a.part_o[at * D + lane * (D / 32) + j] = xo[j];
        if (lane == 0) a.part_ml[at] = make_float2(xm, xl);
      }
    }
    done += u1 - u0;
    if (!ok) {  // a wait ran out and was reported: leave after this warp's copies have landed
      for (; taken < issued; ++taken)
        mbar_wait(&bars[warp][taken % P::kStages], (taken / P::kStages) & 1, a.status);
      break;
    }
    walk.u = u1 - 1;
    if (done < jobs) walk.next(a, prefix, requests, most_rows);
  }
  // Behind a first phase: this grid's completion has to imply that one's. The
  // phases read the same inputs and write different states, so that nothing
  // before this point waits for the first.
  if (a.chained) pdl_wait();
}

template <typename T, int D>
int launch_t(const PagedAttnArgs& a, int streams, int most_rows, int* prefix, const CUtensorMap& km, const CUtensorMap& vm,
             cudaStream_t stream) {
  const int requests = a.shared ? 1 : a.R;
  auto kern = token_attn_kernel<T, D>;
  const int smem = TokenPlan<D>::kBytes + (requests + 1) * 4;
  // The limit belongs to the kernel, not to this call: always that of the
  // largest batch, so that no other thread's call lowers it before the launch.
  constexpr int kMost = TokenPlan<D>::kBytes + (kMostRequests + 1) * 4;
  const int rc = static_cast<int>(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
  if (rc) return rc;
  if (a.chained)
    return launch_pdl(kern, dim3(streams / kWarps), dim3(kWarps * 32), smem, stream, 0, a, requests, most_rows, prefix, km,
                      vm);
  kern<<<streams / kWarps, kWarps * 32, smem, stream>>>(a, requests, most_rows, prefix, km, vm);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

bool token_attn_takes(int kv_dtype, int d, int page_size, int R, const void* k, const void* v, const void* q,
                      long long q_ts, long long q_hs) {
  const uintptr_t pool = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
  const uintptr_t rows = reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(q_ts * 2) | static_cast<uintptr_t>(q_hs * 2);
  return kv_dtype != kF32 && (d == 64 || d == 128) && page_size % kUnit == 0 && R <= kMostRequests && pool % 16 == 0 &&
         rows % 4 == 0;
}

int launch_token_attn(const PagedAttnArgs& a, int kv_dtype, int streams, int most_rows, int* prefix, cudaStream_t stream) {
  CUtensorMap km, vm;
  int rc = encode_pool_map(&km, a, a.L.k, kv_dtype, kUnit);
  if (rc == 0) rc = encode_pool_map(&vm, a, a.L.v, kv_dtype, kUnit);
  if (rc) return rc;
  if (kv_dtype == kBF16)
    return a.d == 64 ? launch_t<__nv_bfloat16, 64>(a, streams, most_rows, prefix, km, vm, stream)
                     : launch_t<__nv_bfloat16, 128>(a, streams, most_rows, prefix, km, vm, stream);
  return a.d == 64 ? launch_t<__half, 64>(a, streams, most_rows, prefix, km, vm, stream)
                   : launch_t<__half, 128>(a, streams, most_rows, prefix, km, vm, stream);
}

}  // namespace stk
