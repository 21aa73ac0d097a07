// The next token of each row of logits, from a given uniform number.
//
// Of a row's tokens in descending order of logits (ties: the lower token
// first) stay the first top_k, of those the ones before which less than top_p
// of their mass lies, of those the ones with at least min_p of the largest
// mass; the token is drawn from what stays, in the vocabulary's order.
//
// The mass of a token is e = exp((x - max) / T). It decides between
// neighbouring tokens, so sums must not depend on the order of additions nor
// lose what lies between two tokens of a large vocabulary: e is computed in FP64
// (2^t by a degree-9 polynomial, relative error 2e-14) and added as a 64-bit
// whole number of 2^-44. Thresholds are then found digit by digit of the
// logits' order keys (11, 11 and 10 bits), by counts for top_k and by masses
// for top_p, exactly and the same on every run.
//
// A row is read once, into the shared memory of a cluster of up to eight CTAs.

#include <cooperative_groups.h>

#include "sample.cuh"

namespace stk {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024, kBins = 2048;
constexpr double kUnit = 17592186044416.0;  // 2^44

using u64 = unsigned long long;

__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return x == 0.f ? 0x80000000u : u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

// 2^t for t <= 0 as a whole number of 2^-44: t = n + f with |f| <= 1/2, 2^f by
// a polynomial fitted for the least relative error.
__device__ __forceinline__ double mass_of(double t) {
  const double m = t + 6755399441055744.0;  // 1.5 * 2^52: n in the low bits
  const double f = t - (m - 6755399441055744.0);
  double p = fma(f, 1.0148587078171632e-07, 1.325834013445892e-06);
  p = fma(p, f, 1.5252988727215495e-05);
  p = fma(p, f, 0.00015403440864986972);
  p = fma(p, f, 0.0013333557627726357);
  p = fma(p, f, 0.0096181291811879843);
  p = fma(p, f, 0.055504108668400408);
  p = fma(p, f, 0.24022650695722783);
  p = fma(p, f, 0.69314718055988556);
  p = fma(p, f, 1.0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(m) << 20), __double2loint(p));
}

struct Row {
  float max;
  double rate;   // log2 e / T
  double least;  // mass below which a token does not stay
  // Tokens above `limit` stay, of those at it the first `take`.
  uint32_t limit;
  int take;
  __device__ __forceinline__ double mass(float x) const {
    if (x == max) return 1.0;
    const double t = (static_cast<double>(x) - static_cast<double>(max)) * rate;
    return t < -60.0 ? 0.0 : mass_of(t);
  }
  // In units; 0 for a token of too little mass.
  __device__ __forceinline__ u64 units(float x) const {
    const double e = mass(x);
    return e >= least ? __double2ull_rn(e * kUnit) : 0ull;
  }
};

struct Shared {
  uint32_t low[2][kBins], high[2][kBins];  // of two digits by turns: counts, or the two halves of masses
  int warp_ints[32];
  u64 warp_sums[32];
  u64 best;   // of the CTA: the largest logit's key, and the lowest token that has it
  int equal;  // tokens at the limit
  u64 sum;    // mass of what stays
  int digit;
  u64 above, inside;
};

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

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const SampleArgs a) {
  extern __shared__ float row[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = static_cast<int>(blockIdx.x) / parts;
  const int slice = ((a.V + parts - 1) / parts + 31) / 32 * 32;
  const int begin = min(a.V, part * slice), n = min(a.V, begin + slice) - begin;

  // ---- the slice, and its largest logit (NaN is never chosen)
  const T* src = static_cast<const T*>(a.logits) + r * a.stride + begin;
  u64 best = 0;
  auto take_in = [&](int i, float x) {
    if (x != x) x = neg_inf();
    row[i] = x;
    const u64 b = static_cast<u64>(order_key(x)) << 32 | static_cast<uint32_t>(~(begin + i));
    best = b > best ? b : best;
  };
  constexpr int kVec = 16 / sizeof(T);
  int done = 0;
  if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
    done = n / kVec * kVec;
#pragma unroll 4
    for (int i = tid * kVec; i < done; i += kThreads * kVec) {
      const uint4 v = *reinterpret_cast<const uint4*>(src + i);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) take_in(i + j, to_f32(e[j]));
    }
  }
  for (int i = done + tid; i < n; i += kThreads) take_in(i, to_f32(src[i]));
  for (int i = tid; i < kBins; i += kThreads) sh.low[0][i] = sh.high[0][i] = 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 y = __shfl_xor_sync(kFull, best, o);
    best = y > best ? y : best;
  }
  if (lane == 0) sh.warp_sums[warp] = best;
  __syncthreads();
  best = sh.warp_sums[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 y = __shfl_xor_sync(kFull, best, o);
    best = y > best ? y : best;
  }
  if (tid == 0) sh.best = best;
  cluster.sync();
  for (int p = 0; p < parts; ++p) {
    const u64 y = *cluster.map_shared_rank(&sh.best, p);
    best = y > best ? y : best;
  }
  const int greedy = static_cast<int>(~static_cast<uint32_t>(best));
  const uint32_t top = static_cast<uint32_t>(best >> 32);
  const float temperature = a.temperature.rows ? a.temperature.rows[r] : a.temperature.all;
  const bool nothing = top <= order_key(neg_inf());
  if (nothing || !(temperature > 0.f)) {
    if (part == 0 && tid == 0) {
      a.tokens[r] = nothing ? -1 : greedy;
      if (nothing) report(a.status, kStatusNoToken);
    }
    cluster.sync();  // siblings may still read this CTA's best
    return;
  }
  Row w;
  w.max = __uint_as_float(top & 0x80000000u ? top ^ 0x80000000u : ~top);
  w.rate = 1.4426950408889634 / static_cast<double>(temperature);
  w.least = 0.0;
  w.limit = 0;
  w.take = 0x7fffffff;
  const int top_k = a.top_k.rows ? a.top_k.rows[r] : a.top_k.all;
  const float top_p = a.top_p.rows ? a.top_p.rows[r] : a.top_p.all;
  const float min_p = a.min_p.rows ? a.min_p.rows[r] : a.min_p.all;

  // ---- thresholds: first by counts (top_k), then by masses (top_p)
  int turn = 0;  // of the histograms
  for (int mode = 0; mode < 2; ++mode) {
    const bool counts = mode == 0;
    if (counts ? top_k <= 0 || top_k >= a.V : !(top_p < 1.f)) continue;
    u64 goal = counts ? static_cast<u64>(top_k) : 0;
    uint32_t limit = 0;
    for (int digit = 0; digit < 3; ++digit, turn ^= 1) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
      uint32_t *low = sh.low[turn], *high = sh.high[turn];
      for (int i = tid; i < n; i += kThreads) {
        const float x = row[i];
        const uint32_t key = order_key(x);
        if (digit > 0 && (key >> (shift + bits)) != (limit >> (shift + bits))) continue;
        const int bin = (key >> shift) & ((1u << bits) - 1);
        if (counts) {
          atomicAdd(&low[bin], 1u);
        } else {
          if (key <= w.limit) continue;  // those at top_k's limit follow below
          const u64 e = w.units(x);
          const uint32_t e_low = static_cast<uint32_t>(e), old = atomicAdd(&low[bin], e_low);
          const uint32_t e_high = static_cast<uint32_t>(e >> 32) + (old + e_low < old ? 1u : 0u);
          if (e_high) atomicAdd(&high[bin], e_high);
        }
      }
      // (All that stay at top_k's limit weigh alike.)
      if (!counts && part == 0 && tid == 0 && w.take != 0x7fffffff &&
          (digit == 0 || (w.limit >> (shift + bits)) == (limit >> (shift + bits)))) {
        const float x = __uint_as_float(w.limit & 0x80000000u ? w.limit ^ 0x80000000u : ~w.limit);
        const u64 e = w.units(x) * static_cast<u64>(w.take);
        const int bin = (w.limit >> shift) & ((1u << bits) - 1);
        const uint32_t e_low = static_cast<uint32_t>(e), old = atomicAdd(&low[bin], e_low);
        const uint32_t e_high = static_cast<uint32_t>(e >> 32) + (old + e_low < old ? 1u : 0u);
        if (e_high) atomicAdd(&high[bin], e_high);
      }
      cluster.sync();
      for (int i = tid; i < kBins; i += kThreads) sh.low[turn ^ 1][i] = sh.high[turn ^ 1][i] = 0;
      const int b0 = kBins - 1 - 2 * tid;  // two bins per thread, the highest first
      u64 c0 = 0, c1 = 0;
      for (int p = 0; p < parts; ++p) {
        const uint32_t *l = cluster.map_shared_rank(low, p), *u = cluster.map_shared_rank(high, p);
        c0 += static_cast<u64>(u[b0]) << 32 | l[b0];
        c1 += static_cast<u64>(u[b0 - 1]) << 32 | l[b0 - 1];
      }
      u64 total;
      const u64 before = scan_add<u64>(c0 + c1, sh.warp_sums, total);
      if (!counts && digit == 0) {
        // The least whole number that is not below top_p of the mass; the first token always stays.
        const double g = ceil(static_cast<double>(top_p > 0.f ? top_p : 0.f) * static_cast<double>(total));
        goal = static_cast<u64>(g);
        goal = goal < 1 ? 1 : goal > total ? total : goal;
      }
      if (before < goal && before + c0 + c1 >= goal) {
        const bool first = before + c0 >= goal;
        sh.digit = first ? b0 : b0 - 1;
        sh.above = first ? before : before + c0;
        sh.inside = first ? c0 : c1;
      }
      __syncthreads();
      limit |= static_cast<uint32_t>(sh.digit) << shift;
      goal -= sh.above;
      __syncthreads();
    }
    // What is left of the goal is taken at the limit, token by token.
    if (counts) {
      w.take = static_cast<int>(goal);
    } else {
      const float x = __uint_as_float(limit & 0x80000000u ? limit ^ 0x80000000u : ~limit);
      const u64 e = w.units(x), some = (goal + e - 1) / e;
      const int available = limit == w.limit && w.take != 0x7fffffff ? w.take : 0x7fffffff;
      w.take = some < static_cast<u64>(available) ? static_cast<int>(some) : available;
    }
    w.limit = limit;
  }
  w.least = min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) : 0.0;

  // ---- what stays, in order: each warp a stretch
  const int stretch = (n + 32 * 32 - 1) / (32 * 32) * 32, w0 = min(n, warp * stretch), w1 = min(n, w0 + stretch);
  int equal = 0;
  const bool ties = w.take != 0x7fffffff;  // only then do tokens at the limit differ
  if (ties) {
    for (int i0 = w0; i0 < w1; i0 += 32)
      equal += __popc(__ballot_sync(kFull, i0 + lane < w1 && order_key(row[i0 + lane]) == w.limit));
    int all_equal;
    equal = scan_add<int>(lane == 0 ? equal : 0, sh.warp_ints, all_equal);
    equal = __shfl_sync(kFull, equal, 0);
    if (tid == 0) sh.equal = all_equal;
    cluster.sync();
    for (int p = 0; p < part; ++p) equal += *cluster.map_shared_rank(&sh.equal, p);
  }
  // Mass of token i of the slice, with `e` tokens at the limit before it.
  auto stays = [&](int i, int e) {
    if (i >= w1) return 0ull;
    const uint32_t key = order_key(row[i]);
    return key > w.limit || (key == w.limit && e < w.take) ? w.units(row[i]) : 0ull;
  };
  auto equal_before = [&](int i, int e, unsigned& at) {
    at = ties ? __ballot_sync(kFull, i < w1 && order_key(row[i]) == w.limit) : 0u;
    return e + __popc(at & ((1u << lane) - 1));
  };
  u64 sum = 0;
  int e = equal;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    unsigned at;
    const int mine = equal_before(i0 + lane, e, at);
    sum += stays(i0 + lane, mine);
    e += __popc(at);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
  u64 total;
  const u64 before = __shfl_sync(kFull, scan_add<u64>(lane == 0 ? sum : 0, sh.warp_sums, total), 0);
  if (tid == 0) sh.sum = total;
  cluster.sync();
  u64 all = 0, mine = before;
  for (int p = 0; p < parts; ++p) {
    const u64 y = *cluster.map_shared_rank(&sh.sum, p);
    all += y;
    if (p < part) mine += y;
  }
  cluster.sync();  // the sums have been read: a sibling may leave
  // The first token whose mass and that of those before it exceed u of all.
  const double u = static_cast<double>(a.uniforms[r]);
  const double g = u > 0.0 ? floor(u * static_cast<double>(all)) : 0.0;
  u64 goal = g >= static_cast<double>(all) ? all - 1 : static_cast<u64>(g);
  goal = goal < all ? goal : all - 1;
  if (mine > goal || mine + sum <= goal) return;
  e = equal;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    unsigned at;
    const int eq = equal_before(i0 + lane, e, at);
    u64 x = stays(i0 + lane, eq);
    e += __popc(at);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(kFull, x, o);
      if (lane >= o) x += y;
    }
    const unsigned passed = __ballot_sync(kFull, mine + x > goal);
    if (passed) {
      if (lane == 0) a.tokens[r] = begin + i0 + __ffs(passed) - 1;
      return;
    }
    mine += __shfl_sync(kFull, x, 31);
  }
}

template <typename T>
int launch(const SampleArgs& a, int sms, cudaStream_t stream) {
  // CTAs of a row: as many as its logits need, more while they find SMs and a few thousand logits each.
  int parts = 1;
  while (parts * kSampleSlice < a.V) parts *= 2;
  while (parts < kSampleCluster && static_cast<long long>(a.R) * parts * 2 <= sms && a.V / parts > 4096) parts *= 2;
  if (static_cast<long long>(a.R) * parts > 0x7fffffff) return static_cast<int>(cudaErrorInvalidValue);
  const int bytes = static_cast<int>(sizeof(float)) * (((a.V + parts - 1) / parts + 31) / 32 * 32);
  auto kern = sample_kernel<T>;
  const int rc = static_cast<int>(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleSlice * 4));
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.R * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, a));
}

}  // namespace

int launch_sample(const SampleArgs& a, int dtype, int sms, cudaStream_t stream) {
  if (dtype == kF32) return launch<float>(a, sms, stream);
  return dtype == kBF16 ? launch<__nv_bfloat16>(a, sms, stream) : launch<__half>(a, sms, stream);
}

}  // namespace stk
