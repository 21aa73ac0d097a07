// Attention weight received by each cached key, on the FP32 units: FP32, head
// sizes and layouts that the tensor-core kernel does not take.
//
// A CTA takes 32 keys of one request's KV head, in shared memory as FP32, one
// to a lane. Its four warps take every fourth group of four rows (new tokens x
// query heads), their queries broadcast from shared memory, so that a key's
// four values are read once for four rows. Runs of 64 rows are added in FP32,
// runs and the four warps' sums in FP64, in order: the result does not depend on
// timing, and its error not on the prompt's length (4,100 tokens of 12 heads that
// weigh alike: 1.2e-4 by one FP32 sum per warp, within 4e-6 so).
//
// HBM-bound for single tokens (K is read once per KV head), bound by shared
// memory reads (two per four FMAs) for many rows.
//
// Few rows (at most 16 of a KV head, heads of 64, 128 or 256 dims) need no K in
// shared memory: a warp's lanes share a key's dims, eight keys are on their way
// at once, and the 8 x 4 sums of eight keys and four rows are transposed into
// one per lane (31 shuffles). 5 requests of 700 to 9,000 tokens, 32 / 8 heads,
// FP32 (82 MB): 36 us, 2.3 TB/s (58 in the form above), of which a CTA's chain of
// loads (offsets, lengths, table, keys) is most: it lives for 256 keys.

#include "weigh.cuh"

namespace stk {

namespace {

constexpr int kKeys = 32, kWarps = 4, kRows = 4;
constexpr int kRun = 16;  // groups of rows that are added in FP32

// Row pitch in floats: whole 16-byte chunks, an odd number of them.
__host__ __device__ inline int pitch(int d) { return (((d + 3) / 4) | 1) * 4; }

inline size_t shared_bytes(int d) { return sizeof(float) * static_cast<size_t>(pitch(d)) * (kKeys + kWarps * kRows); }

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
weigh_rows_kernel(const WeighArgs w, int tiles, int vector) {
  const PagedAttnArgs& a = w.a;
  extern __shared__ __align__(16) float smem[];
  __shared__ long long place[kKeys];
  __shared__ int2 seen[kWarps];
  __shared__ double sums[kWarps][kKeys];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tile = static_cast<int>(blockIdx.x % tiles);
  const int h = static_cast<int>(blockIdx.x / tiles) % a.L.hkv, r = static_cast<int>(blockIdx.x / tiles) / a.L.hkv;
  const int2 tn = new_tokens(a.token_offsets, r, a.R, a.T, a.status);
  const int k0 = tile * kKeys, n = min(tn.y, w.most);
  RowTile t;
  t.r = r;
  t.t0 = tn.x;
  t.n = tn.y;
  t.len = cached_tokens(a, r, tn.y);
  if (tn.y > w.most) report(a.status, kStatusShapeOverflow);
  if (n == 0 || k0 >= t.len) return;

  // ---- keys that any row sees
  int lo = 0, hi = t.len - t.n + n;
  if (a.kv_lo || a.kv_hi) {
    lo = 0x7fffffff;
    hi = 0;
    for (int i = tid; i < n; i += blockDim.x) {
      const RowKeys k = row_keys(a, t, i);
      if (k.hi > k.lo) {
        lo = min(lo, k.lo);
        hi = max(hi, k.hi);
      }
    }
    lo = __reduce_min_sync(kFull, lo);
    hi = __reduce_max_sync(kFull, hi);
    if (lane == 0) seen[warp] = make_int2(lo, hi);
    __syncthreads();
    for (int x = 0; x < kWarps; ++x) {
      lo = min(lo, seen[x].x);
      hi = max(hi, seen[x].y);
    }
  }
  lo = max(lo, k0);
  hi = min(hi, k0 + kKeys);
  if (lo >= hi) return;

  // ---- their K, widened
  const int d = a.d, p = pitch(d);
  float* ks = smem;
  float* qs = smem + (kKeys + warp * kRows) * p;
  if (tid < kKeys) {
    const int key = k0 + tid;
    const int page = key >= lo && key < hi ? page_of(a, r, key) : -1;
    place[tid] = page < 0 ? -1 : ((static_cast<long long>(page) * a.L.hkv + h) * a.L.page_size + key % a.L.page_size) * d;
  }
  __syncthreads();
  const T* k = static_cast<const T*>(a.L.k);
  if (vector) {
    constexpr int N = 16 / sizeof(T);
    const int chunks = d / N;
#pragma unroll 4
    for (int x = tid; x < kKeys * chunks; x += kWarps * 32) {
      const int row = x / chunks, c = x - row * chunks;
      float v[N] = {};
      if (place[row] >= 0) load_vec<T, N>(k + place[row] + c * N, v);
      store_vec<N>(ks + row * p + c * N, v);
    }
  } else {
    for (int row = warp; row < kKeys; row += kWarps)
      for (int c = lane; c < p; c += 32) ks[row * p + c] = c < d && place[row] >= 0 ? to_f32(k[place[row] + c]) : 0.f;
  }
  __syncthreads();

  // ---- rows
  const int key = k0 + lane, rows = n * a.G, d4 = (d + 3) / 4;
  const T* q = static_cast<const T*>(a.q);
  double total = 0.0;
  float sum = 0.f;  // of a run of the warp's rows
  int groups = 0;
  for (int r0 = warp * kRows; r0 < rows; r0 += kWarps * kRows) {
    if (groups++ == kRun) {
      total += sum;
      sum = 0.f;
      groups = 1;
    }
    __syncwarp();
    for (int x = 0; x < kRows; ++x) {
      const int row = min(r0 + x, rows - 1), tok = row / a.G;
      const T* src = q + static_cast<long long>(t.t0 + tok) * a.q_ts + static_cast<long long>(h * a.G + row - tok * a.G) * a.q_hs;
      for (int c = lane; c < 4 * d4; c += 32) qs[x * p + c] = c < d ? to_f32(src[c]) : 0.f;
    }
    __syncwarp();
    float4 dot[kRows] = {};
    for (int c = 0; c < d4; ++c) {
      const float4 y = *reinterpret_cast<const float4*>(ks + lane * p + c * 4);
#pragma unroll
      for (int x = 0; x < kRows; ++x) {
        const float4 z = *reinterpret_cast<const float4*>(qs + x * p + c * 4);
        dot[x].x = fmaf(y.x, z.x, dot[x].x);
        dot[x].y = fmaf(y.y, z.y, dot[x].y);
        dot[x].z = fmaf(y.z, z.z, dot[x].z);
        dot[x].w = fmaf(y.w, z.w, dot[x].w);
      }
    }
#pragma unroll
    for (int x = 0; x < kRows; ++x) {
      const int row = r0 + x;
      if (row >= rows) break;
      const int tok = row / a.G, head = h * a.G + row - tok * a.G;
      const RowKeys rk = row_keys(a, t, tok);
      const float lse = w.lse[static_cast<long long>(t.t0 + tok) * a.hq + head];
      float s = ((dot[x].x + dot[x].y) + (dot[x].z + dot[x].w)) * a.scale;
      if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
      if (a.slopes) s -= a.slopes[head] * fabsf(static_cast<float>(rk.pos - key));
      // A row that saw no key (log-sum-exp -inf) gives nothing; unseen keys may hold anything.
      if (key >= rk.lo && key < rk.hi && lse != neg_inf()) sum += expf(s - lse);
    }
  }
  sums[warp][lane] = total + sum;
  __syncthreads();
  if (warp == 0 && key >= lo && key < hi) {
    float* to = w.weights + h * w.slots + static_cast<long long>(a.L.block_offsets[r]) * a.L.b + key;
    *to += static_cast<float>((sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]));
  }
}

constexpr int kFewWarps = 8, kFewRows = 16, kAtOnce = 8;

template <typename T, int VEC>
__device__ __forceinline__ void load_dims(const T* p, float (&x)[VEC]) {
  if constexpr (VEC * sizeof(T) >= 16 || sizeof(T) == 2) {
    load_vec<T, VEC>(p, x);
  } else {
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x;
    x[1] = v.y;
  }
}

// VEC: dims of a lane.
template <typename T, int VEC>
__global__ void __launch_bounds__(kFewWarps * 32, 2) weigh_few_kernel(const WeighArgs w, int tiles) {
  const PagedAttnArgs& a = w.a;
  constexpr int D = VEC * 32;
  __shared__ __align__(16) float qs[kFewRows][D];
  struct Row {
    int lo, hi;
    float pos, slope, lse;
  };
  __shared__ Row info[kFewRows];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tile = static_cast<int>(blockIdx.x % tiles);
  const int h = static_cast<int>(blockIdx.x / tiles) % a.L.hkv, r = static_cast<int>(blockIdx.x / tiles) / a.L.hkv;
  const int2 tn = new_tokens(a.token_offsets, r, a.R, a.T, a.status);
  const int k0 = tile * kFewWarps * 32, n = min(tn.y, w.most), rows = n * a.G;
  RowTile t;
  t.r = r;
  t.t0 = tn.x;
  t.n = tn.y;
  t.len = cached_tokens(a, r, tn.y);
  if (tn.y > w.most) report(a.status, kStatusShapeOverflow);
  if (n == 0 || k0 >= t.len) return;
  if (tid < kFewRows) {
    Row x{0, 0, 0.f, 0.f, neg_inf()};
    if (tid < rows) {
      const int tok = tid / a.G, head = h * a.G + tid - tok * a.G;
      const RowKeys k = row_keys(a, t, tok);
      x.lse = w.lse[static_cast<long long>(t.t0 + tok) * a.hq + head];
      if (x.lse != neg_inf()) {  // (a row that saw no key gives nothing)
        x.lo = k.lo;
        x.hi = k.hi;
      }
      x.pos = static_cast<float>(k.pos);
      x.slope = a.slopes ? a.slopes[head] : 0.f;
    }
    info[tid] = x;
  }
  const T* q = static_cast<const T*>(a.q);
  for (int i = tid; i < kFewRows * D; i += kFewWarps * 32) {
    const int row = i / D, tok = row / a.G;
    qs[row][i - row * D] = row < rows ? to_f32(q[static_cast<long long>(t.t0 + tok) * a.q_ts +
                                                 static_cast<long long>(h * a.G + row - tok * a.G) * a.q_hs + i - row * D]) : 0.f;
  }
  __syncthreads();
  // Keys that any row sees, and where the lane's one is.
  int lo = 0x7fffffff, hi = 0;
  if (lane < kFewRows && info[lane].lo < info[lane].hi) {
    lo = info[lane].lo;
    hi = info[lane].hi;
  }
  lo = __reduce_min_sync(kFull, lo);
  hi = __reduce_max_sync(kFull, hi);
  const int kw = k0 + warp * 32, mine = kw + lane;
  long long place = -1;
  if (mine >= lo && mine < hi) {
    const int page = page_of(a, r, mine);
    if (page >= 0) place = ((static_cast<long long>(page) * a.L.hkv + h) * a.L.page_size + mine % a.L.page_size) * D;
  }
  if (kw >= hi || kw + 32 <= lo) return;
  const T* kp = static_cast<const T*>(a.L.k) + lane * VEC;
  float* to = w.weights + h * w.slots + static_cast<long long>(a.L.block_offsets[r]) * a.L.b;
#pragma unroll 1
  for (int b = 0; b < 32; b += kAtOnce) {
    if (kw + b >= hi || kw + b + kAtOnce <= lo) continue;
    float k[kAtOnce][VEC];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const long long at = __shfl_sync(kFull, place, b + i);
      if (at >= 0) {
        load_dims<T, VEC>(kp + at, k[i]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) k[i][j] = 0.f;
      }
    }
    const int key = kw + b + lane / 4;
    float sum = 0.f;
    for (int r0 = 0; r0 < rows; r0 += 4) {
      float v[32];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float y[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          const float2 z = *reinterpret_cast<const float2*>(&qs[r0 + x][lane * VEC + j]);
          y[j] = z.x;
          y[j + 1] = z.y;
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          float dot = 0.f;
#pragma unroll
          for (int j = 0; j < VEC; ++j) dot = fmaf(k[i][j], y[j], dot);
          v[i * 4 + x] = dot;
        }
      }
      transpose_reduce32(v, lane);
      const Row z = info[r0 + lane % 4];
      float s = v[0] * a.scale;
      if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
      if (a.slopes) s -= z.slope * fabsf(z.pos - static_cast<float>(key));
      if (key >= z.lo && key < z.hi) sum += expf(s - z.lse);
    }
    sum += __shfl_xor_sync(kFull, sum, 1);
    sum += __shfl_xor_sync(kFull, sum, 2);
    if (lane % 4 == 0 && key >= lo && key < hi && sum != 0.f) atomicAdd(to + key, sum);  // the key's only one of the call
  }
}

template <typename T, int VEC>
int launch_few(const WeighArgs& w, cudaStream_t stream) {
  const int tiles = (w.longest + kFewWarps * 32 - 1) / (kFewWarps * 32);
  const long long ctas = static_cast<long long>(tiles) * w.a.L.hkv * w.a.R;
  if (ctas > 0x7fffffff) return static_cast<int>(cudaErrorInvalidValue);
  weigh_few_kernel<T, VEC><<<static_cast<unsigned>(ctas), kFewWarps * 32, 0, stream>>>(w, tiles);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int launch(const WeighArgs& w, cudaStream_t stream) {
  if (static_cast<long long>(w.most) * w.a.G <= kFewRows && reinterpret_cast<uintptr_t>(w.a.L.k) % 16 == 0) {
    if (w.a.d == 64) return launch_few<T, 2>(w, stream);
    if (w.a.d == 128) return launch_few<T, 4>(w, stream);
    if (w.a.d == 256) return launch_few<T, 8>(w, stream);
  }
  const size_t bytes = shared_bytes(w.a.d);
  auto kern = weigh_rows_kernel<T>;
  const int rc = static_cast<int>(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared_bytes(1024))));
  if (rc) return rc;
  const int tiles = (w.longest + kKeys - 1) / kKeys;
  const long long ctas = static_cast<long long>(tiles) * w.a.L.hkv * w.a.R;
  if (ctas > 0x7fffffff) return static_cast<int>(cudaErrorInvalidValue);
  const int vector = w.a.d * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(w.a.L.k) % 16 == 0;
  kern<<<static_cast<unsigned>(ctas), kWarps * 32, bytes, stream>>>(w, tiles, vector);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

int launch_weigh_rows(const WeighArgs& w, int kv_dtype, cudaStream_t stream) {
  if (kv_dtype == kF32) return launch<float>(w, stream);
  return kv_dtype == kBF16 ? launch<__nv_bfloat16>(w, stream) : launch<__half>(w, stream);
}

}  // namespace stk
