// Dense paged attention on the FP32 units: the form that is right for every
// type, head size, page size and number of rows, and the one that FP32 takes.
//
//   s_j = scale q.k_j;  s_j = cap tanh(s_j / cap);  s_j -= slope |pos - j|;
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m) over the row's keys
//   lo <= j < hi, m their maximum; a row without keys gives zeros.
//
// A CTA takes a tile of at most 16 rows of one KV head (rows = new tokens x
// query heads of the group) and one of nsplit parts of the tile's key range.
// Warps hold RW rows each: warp w has row group w % groups and every
// (8 / groups)-th run of TB tokens, so that a run's keys are read from
// memory once and by the other row groups from L1. Lanes own the head's
// dims; a run's TB x RW dot products are finished by one transposed
// butterfly, which leaves one score per lane, and the running maximum and
// sum of a row live in the lanes that hold its scores. K and V go from
// memory to registers directly, TB rows of each in flight per warp.
// Single tokens are HBM-bound (each key and value once per KV head) up to
// four heads a group; each further four read the run again from L1 and take
// as many instructions once more.
//
// Measured (B200, FP32): one token of 4096 keys, 8 / 2 heads: 10 us with the
// join, launch latency. 16 requests of 4-16 K tokens, 32 / 8 heads, D 128:
// 302 us, 4.3 TB/s; 96 / 8 heads: 918 us, 1.4 TB/s, issue-bound. A prompt of
// 2,000 tokens, 32 / 8 heads: FP32, D 128: 2.8 ms (the tensor cores' 16-bit
// form 54 us); bf16, D 96 6.0 ms, D 256 5.3 ms. 16 single tokens, bf16: D 96
// 530 us, D 256 460 us (D 128 on the tensor cores: 92 us). With a branch
// around each token's load the loads came one by one (a fifth of this rate).

#include "block_state.cuh"
#include "paged_ops.cuh"

namespace stk {

constexpr int kRowsWarps = 8;
constexpr int kRowTile = 16;

// Finishes 32 lane-partial sums: lane t ends with the total of v[t].
__device__ __forceinline__ float finish32(float (&v)[32], int lane) {
  transpose_reduce32(v, lane);
  return v[0];
}

template <typename T, int NPL, bool VEC>
__device__ __forceinline__ void load_lane(const T* row, int D, int lane, float (&x)[NPL]) {
  if constexpr (VEC) {
    load_vec<T, NPL>(row + lane * NPL, x);
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int dd = lane + 32 * j;
      x[j] = dd < D ? to_f32(row[dd]) : 0.f;
    }
  }
}

template <typename T, int NPL, int RW, bool VEC>
__global__ void __launch_bounds__(kRowsWarps * 32) rows_attn_kernel(PagedAttnArgs a) {
  constexpr int TB = 32 / RW;  // tokens of a run
  extern __shared__ float rsm[];
  __shared__ RowKeys range[kRowTile];
  __shared__ float wm[kRowsWarps][RW], wl[kRowsWarps][RW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = blockIdx.x % a.nsplit, h = blockIdx.y, D = a.d;
  const RowTile t = row_tile<kRowTile>(a, blockIdx.x / a.nsplit, lane);
  if (t.rows == 0) return;
  if (tid < kRowTile) range[tid] = tid < t.rows ? row_keys(a, t, (t.row0 + tid) / a.G) : RowKeys{0, 0, 0};
  __syncthreads();
  int kmin = 0x7fffffff, kmax = 0;
#pragma unroll
  for (int i = 0; i < kRowTile; ++i) {
    const RowKeys rk = range[i];
    if (rk.hi > rk.lo) {
      kmin = min(kmin, rk.lo);
      kmax = max(kmax, rk.hi);
    }
  }
  if (kmax == 0) kmin = 0;  // no row of the tile sees a key
  // This CTA's part of [kmin, kmax), whole runs of TB tokens.
  const int span = max(0, kmax - kmin);
  const int per = ((span + a.nsplit - 1) / a.nsplit + TB - 1) / TB * TB;
  const int begin = kmin + min(span, split * per), end = kmin + min(span, (split + 1) * per);

  const int groups = (t.rows + RW - 1) / RW;
  // Tiles with more row groups than warps take several passes over the keys.
  for (int g0 = 0; g0 < groups; g0 += kRowsWarps) {
    const int ng = min(groups - g0, kRowsWarps);
    const int slices = kRowsWarps / ng;
    const int grp = g0 + warp % ng, slice = warp / ng;
    const bool idle = slice >= slices;
    float q[RW][NPL], acc[RW][NPL];
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int row = min(grp * RW + i, t.rows - 1);
      const int tok = (t.row0 + row) / a.G, g = (t.row0 + row) - tok * a.G;
      load_lane<T, NPL, VEC>(static_cast<const T*>(a.q) + (t.t0 + tok) * a.q_ts + (h * a.G + g) * a.q_hs, D, lane,
                             q[i]);
#pragma unroll
      for (int j = 0; j < NPL; ++j) acc[i][j] = 0.f;
    }
    // Score lane: token lane / RW of the run, row lane % RW of the group.
    const int my = grp * RW + lane % RW;
    const bool have = my < t.rows;
    const RowKeys rk = range[min(my, kRowTile - 1)];
    const int my_tok = (t.row0 + min(my, t.rows - 1)) / a.G;
    const float slope = a.slopes && have ? a.slopes[h * a.G + (t.row0 + my) - my_tok * a.G] : 0.f;
    const float icap = a.softcap > 0.f ? 1.f / a.softcap : 0.f;
    float m = neg_inf(), l = 0.f;
    const int rp = t.r;
    // Element of key token t0 + lane in its head of the pool, or -1.
    auto place = [&](int t0) -> long long {
      if (lane >= TB || t0 + lane >= end) return -1;
      const int page = page_of(a, rp, t0 + lane);
      if (page < 0) return -1;
      return ((static_cast<long long>(page) * a.L.hkv + h) * a.L.page_size + (t0 + lane) % a.L.page_size) * D;
    };
    long long next = idle ? -1 : place(begin + slice * TB);
    for (int t0 = begin + slice * TB; !idle && t0 < end; t0 += slices * TB) {
      const long long off = next;
      float p[32];
      float vv[NPL <= 8 ? TB : 1][NPL];  // the run's values, requested before its scores are needed
      if constexpr (NPL <= 8) {
        // All of the run's rows at once; a token without a place reads the pool's first row and is not seen.
        float kk[TB][NPL];
#pragma unroll
        for (int k = 0; k < TB; ++k)
          load_lane<T, NPL, VEC>(static_cast<const T*>(a.L.k) + max(__shfl_sync(kFull, off, k), 0ll), D, lane, kk[k]);
#pragma unroll
        for (int k = 0; k < TB; ++k)
          load_lane<T, NPL, VEC>(static_cast<const T*>(a.L.v) + max(__shfl_sync(kFull, off, k), 0ll), D, lane, vv[k]);
        next = place(t0 + slices * TB);
#pragma unroll
        for (int k = 0; k < TB; ++k) {
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            float x = 0.f;
#pragma unroll
            for (int j = 0; j < NPL; ++j) x = fmaf(q[i][j], kk[k][j], x);
            p[k * RW + i] = x;
          }
        }
      } else {
        next = place(t0 + slices * TB);
#pragma unroll
        for (int k = 0; k < TB; ++k) {
          float kk[NPL];
          load_lane<T, NPL, VEC>(static_cast<const T*>(a.L.k) + max(__shfl_sync(kFull, off, k), 0ll), D, lane, kk);
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            float x = 0.f;
#pragma unroll
            for (int j = 0; j < NPL; ++j) x = fmaf(q[i][j], kk[j], x);
            p[k * RW + i] = x;
          }
        }
      }
      float s = finish32(p, lane) * a.scale;
      const int key = t0 + lane / RW;
      if (a.softcap > 0.f) s = a.softcap * tanhf(s * icap);
      if (slope != 0.f) s -= slope * fabsf(static_cast<float>(rk.pos - key));
      const long long my_off = __shfl_sync(kFull, off, lane / RW);  // by every lane, before any condition
      const bool seen = have && my_off >= 0 && key >= rk.lo && key < rk.hi;
      s = seen ? s : neg_inf();
      float mx = s;
#pragma unroll
      for (int o = RW; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
      const float mn = fmaxf(m, mx);
      const float base = mn == neg_inf() ? 0.f : mn;
      const float alpha = expf(m - base);
      float w = seen ? expf(s - base) : 0.f;
      float sum = w;
#pragma unroll
      for (int o = RW; o < 32; o <<= 1) sum += __shfl_xor_sync(kFull, sum, o);
      l = l * alpha + sum;
      m = mn;
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        const float al = __shfl_sync(kFull, alpha, i);
#pragma unroll
        for (int j = 0; j < NPL; ++j) acc[i][j] *= al;
      }
#pragma unroll
      for (int k = 0; k < TB; ++k) {
        float vl[NPL];
        if constexpr (NPL > 8) {
          load_lane<T, NPL, VEC>(static_cast<const T*>(a.L.v) + max(__shfl_sync(kFull, off, k), 0ll), D, lane, vl);
        }
#pragma unroll
        for (int i = 0; i < RW; ++i) {
          // A key that the row does not see has weight zero; its value may be
          // infinite or NaN and must not reach the sum.
          const float wi = __shfl_sync(kFull, w, k * RW + i);
          if (wi != 0.f) {
#pragma unroll
            for (int j = 0; j < NPL; ++j) acc[i][j] = fmaf(wi, NPL <= 8 ? vv[NPL <= 8 ? k : 0][j] : vl[j], acc[i][j]);
          }
        }
      }
    }
    if (g0 + kRowsWarps >= groups) pdl_release();  // the join may be launched: it waits for the states
    // Join the slices of each row group in shared memory, in slice order.
    __syncthreads();
    float* mine = rsm + static_cast<size_t>(warp) * RW * D;
    if (!idle) {
      if (lane < RW) {
        wm[warp][lane] = state_max(m, l);
        wl[warp][lane] = l;
      }
#pragma unroll
      for (int i = 0; i < RW; ++i) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
          const int dd = VEC ? lane * NPL + j : lane + 32 * j;
          if (dd < D) mine[i * D + dd] = acc[i][j];
        }
      }
    }
    __syncthreads();
    for (int x = tid; x < ng * RW * D; x += blockDim.x) {
      const int rr = x / D, dd = x - rr * D;
      const int gi = rr / RW, i = rr - gi * RW;
      const int row = (g0 + gi) * RW + i;
      if (row >= t.rows) continue;
      float M = neg_inf();
      for (int sl = 0; sl < slices; ++sl) M = fmaxf(M, wm[sl * ng + gi][i]);
      float Z = 0.f, O = 0.f;
      for (int sl = 0; sl < slices; ++sl) {
        const int w = sl * ng + gi;
        if (wm[w][i] == neg_inf()) continue;
        const float c = expf(wm[w][i] - M);
        Z += c * wl[w][i];
        O += c * rsm[(static_cast<size_t>(w) * RW + i) * D + dd];
      }
      const int tok = (t.row0 + row) / a.G, g = t.row0 + row - tok * a.G;
      const long long o = static_cast<long long>(t.t0 + tok) * a.hq + h * a.G + g;
      if (a.part_ml) {
        const long long at = split * static_cast<long long>(a.T) * a.hq + o;
        if (dd == 0) a.part_ml[at] = make_float2(M, Z);
        a.part_o[at * D + dd] = O;
      } else {
        const float y = M == neg_inf() ? 0.f : O / Z;
        T* out = static_cast<T*>(a.out) + o * D + dd;
        if constexpr (sizeof(T) == 4) *out = y;
        else if constexpr (std::is_same<T, __half>::value) *out = __float2half_rn(y);
        else *out = __float2bfloat16_rn(y);
        if (dd == 0 && a.lse) a.lse[o] = M == neg_inf() ? neg_inf() : M + logf(Z);
      }
    }
    __syncthreads();
  }
}

template <typename T, int NPL, int RW, bool VEC>
static int launch_rows_t(const PagedAttnArgs& a, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(kRowsWarps) * RW * a.d * sizeof(float);  // at most 32 KB
  auto kern = rows_attn_kernel<T, NPL, RW, VEC>;
  const int slots = row_tile_slots(a.R, a.T, a.G, a.token_offsets != nullptr, a.shared != 0, kRowTile);
  kern<<<dim3(static_cast<unsigned>(slots * a.nsplit), static_cast<unsigned>(a.L.hkv)), kRowsWarps * 32, smem,
         stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
static int launch_rows_d(const PagedAttnArgs& a, cudaStream_t stream) {
  // Lane vectors need whole rows of 32 vectors and vector-aligned tensors;
  // heads wider than 256 dims hold one row per warp.
  const int d = a.d;
  auto aligned = [&](int npl) {
    const uintptr_t bytes = npl * sizeof(T) < 16 ? npl * sizeof(T) : 16;
    const uintptr_t any = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.L.k) |
                          reinterpret_cast<uintptr_t>(a.L.v) | static_cast<uintptr_t>(a.q_ts * sizeof(T)) |
                          static_cast<uintptr_t>(a.q_hs * sizeof(T));
    return d == 32 * npl && any % bytes == 0;
  };
  if (aligned(2)) return launch_rows_t<T, 2, 4, true>(a, stream);
  if (aligned(4)) return launch_rows_t<T, 4, 4, true>(a, stream);
  if (aligned(8)) return launch_rows_t<T, 8, 4, true>(a, stream);
  if (d <= 256) return launch_rows_t<T, 8, 4, false>(a, stream);
  return launch_rows_t<T, 32, 1, false>(a, stream);
}

int launch_rows_attn(const PagedAttnArgs& a, int kv_dtype, cudaStream_t stream) {
  switch (kv_dtype) {
    case kF32: return launch_rows_d<float>(a, stream);
    case kF16: return launch_rows_d<__half>(a, stream);
    default: return launch_rows_d<__nv_bfloat16>(a, stream);
  }
}

// ------------------------------------------------------------------ join
// out = sum_s e^{m_s - M} o_s / sum_s e^{m_s - M} l_s over the parts of a row,
// in one pass with a running maximum; parts without keys have m = -inf. The
// parts' states are FP32 and read once (L2-resident); the kernel is bound by
// its few dependent loads, so eight parts' maxima, sums and dims are asked for
// at once. WPR warps share a row: with one, a CTA joins eight rows; where
// there are too few rows to fill the SMs that way, all eight warps take every
// eighth part of one row and meet in shared memory, in warp order. The rule
// (two rows an SM) measured on both sides: 2,048 rows of about 21 parts, the
// whole call 95 us with one warp a row, 107 us with eight; 32 rows of 148
// parts, 79 us against 60 us. Lanes hold V consecutive dims (d = 32 V) or,
// V = 0, every 32nd.
constexpr int kJoinWarps = 8;

template <typename T, int V, int WPR>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(JoinArgs a) {
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = WPR == 1 ? blockIdx.x * kJoinWarps + warp : blockIdx.x;
  const int first_part = WPR == 1 ? 0 : warp;
  if (a.block_offsets != nullptr && blockIdx.x == 0 && threadIdx.x == 0 &&
      static_cast<long long>(a.block_offsets[1] - a.block_offsets[0]) * a.block < a.prefix)
    report(a.status, kStatusBadLength);
  if (row >= a.rows) return;
  // Part s of source k is state base[k] + s * step[k].
  long long base[2], step[2];
  int parts[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k >= a.nsrc) continue;
    const PartSource& p = a.src[k];
    base[k] = row;
    step[k] = a.rows;
    parts[k] = p.parts;
    if (p.prefix != nullptr) {
      const int token = row / a.hq, head = row - token * a.hq, h = head / a.G, hkv = a.hq / a.G;
      const int r = p.shared ? 0 : request_of_token(a.token_offsets, p.requests, token);
      const int first = p.shared ? 0 : a.token_offsets != nullptr ? max(a.token_offsets[r], 0) : token;
      const int local = (token - first) * a.G + head - h * a.G;  // row of the request's tile
      const long long total = static_cast<long long>(p.prefix[p.requests]) * hkv;
      const long long per = (total + p.streams - 1) / p.streams;
      const int before = p.prefix[r], units = r < p.requests ? p.prefix[r + 1] - before : 0;  // padding has none
      const long long u0 = static_cast<long long>(before) * hkv + static_cast<long long>(h) * units;
      const int c0 = units ? static_cast<int>(u0 / per) : 0;
      const bool written = units > 0 && local >= 0 && local < p.most_rows;
      parts[k] = written ? static_cast<int>((u0 + units - 1) / per) - c0 + 1 : 0;
      base[k] = (static_cast<long long>(c0) + r * hkv + h) * p.most_rows + local;
      step[k] = p.most_rows;
    }
  }
  constexpr int N = V ? V : 4;
  constexpr int kBatch = 8;  // parts in flight
  __shared__ float part_o[WPR == 1 ? 1 : kJoinWarps][32 * N];
  __shared__ float2 part_ml[kJoinWarps];
  for (int d0 = 0; d0 < a.d; d0 += 32 * N) {
    float o[N], M = neg_inf(), Z = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      for (int s0 = first_part; s0 < parts[k]; s0 += WPR * kBatch) {
        float2 ml[kBatch];
        float x[kBatch][N];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {  // the last part again past the end, with no weight
          const int s = s0 + WPR * i;
          const long long at = base[k] + min(s, parts[k] - 1) * step[k];
          ml[i] = a.src[k].ml[at];
          if (s >= parts[k]) ml[i].x = neg_inf();
          const float* p = a.src[k].o + at * a.d + d0;
          if constexpr (V != 0) {
            load_vec<float, N>(p + lane * N, x[i]);
          } else {
#pragma unroll
            for (int j = 0; j < N; ++j) x[i][j] = d0 + lane + 32 * j < a.d ? p[lane + 32 * j] : 0.f;
          }
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) top = fmaxf(top, ml[i].x);
        if (top == neg_inf()) continue;
        const float f = expf(M - top);
        Z *= f;
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] *= f;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (ml[i].x == neg_inf()) continue;  // also a part that was never written
          const float w = expf(ml[i].x - top);
          Z = fmaf(w, ml[i].y, Z);
#pragma unroll
          for (int j = 0; j < N; ++j) o[j] = fmaf(w, x[i][j], o[j]);
        }
        M = top;
      }
    }
    if constexpr (WPR > 1) {
#pragma unroll
      for (int j = 0; j < N; ++j) part_o[warp][lane * N + j] = o[j];
      if (lane == 0) part_ml[warp] = make_float2(M, Z);
      __syncthreads();
      if (warp == 0) {
        M = neg_inf();
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) M = fmaxf(M, part_ml[w].x);
        Z = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = 0.f;
        if (M != neg_inf()) {
#pragma unroll
          for (int w = 0; w < kJoinWarps; ++w) {
            const float f = expf(part_ml[w].x - M);
            Z = fmaf(f, part_ml[w].y, Z);
#pragma unroll
            for (int j = 0; j < N; ++j) o[j] = fmaf(f, part_o[w][lane * N + j], o[j]);
          }
        }
      }
      __syncthreads();
      if (warp != 0) continue;
    }
    const bool empty = M == neg_inf();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int dd = d0 + (V ? lane * N + j : lane + 32 * j);
      if (dd >= a.d) continue;
      const float y = empty ? 0.f : o[j] / Z;
      T* out = static_cast<T*>(a.out) + static_cast<long long>(row) * a.d + dd;
      if constexpr (sizeof(T) == 4) *out = y;
      else if constexpr (std::is_same<T, __half>::value) *out = __float2half_rn(y);
      else *out = __float2bfloat16_rn(y);
    }
    if (d0 == 0 && lane == 0 && a.lse) a.lse[row] = empty ? neg_inf() : M + logf(Z);
  }
}

template <typename T, int V>
static int launch_join_v(const JoinArgs& a, int sms, cudaStream_t stream) {
  if (a.rows >= 2 * sms)
    return launch_pdl(join_kernel<T, V, 1>, dim3(static_cast<unsigned>((a.rows + kJoinWarps - 1) / kJoinWarps)),
                      dim3(kJoinWarps * 32), 0, stream, 0, a);
  return launch_pdl(join_kernel<T, V, kJoinWarps>, dim3(static_cast<unsigned>(a.rows)), dim3(kJoinWarps * 32), 0,
                    stream, 0, a);
}

template <typename T>
static int launch_join_t(const JoinArgs& a, int sms, cudaStream_t stream) {
  return a.d == 128 ? launch_join_v<T, 4>(a, sms, stream)
         : a.d == 64 ? launch_join_v<T, 2>(a, sms, stream) : launch_join_v<T, 0>(a, sms, stream);
}

int launch_join(const JoinArgs& a, int sms, cudaStream_t stream) {
  switch (a.dtype) {
    case kF32: return launch_join_t<float>(a, sms, stream);
    case kF16: return launch_join_t<__half>(a, sms, stream);
    default: return launch_join_t<__nv_bfloat16>(a, sms, stream);
  }
}

}  // namespace stk
