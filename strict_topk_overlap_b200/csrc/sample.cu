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
// whole number of 2^-44. A threshold (by counts for top_k, by masses for top_p)
// is found in a histogram over the distance from the largest logit, 32 bins to a
// unit, whose one bin that holds it is sorted by a CTA, a token to a thread; a
// bin of too many tokens is cut by a second histogram. What even that leaves
// crowded (many equal logits), or lies beyond its range, is found digit by digit
// of the logits' order keys (11, 11 and 10 bits). All of it is exact and the same
// on every run.
//
// A row is read once, into the shared memory of a cluster of up to eight CTAs.

#include <cooperative_groups.h>

#include "sample.cuh"

namespace stk {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024, kBins = 1024;  // bins of a histogram: one to a thread
constexpr float kBinsPerUnit = 32.f;

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
  // In units; 0 for a token of too little mass. (The last bits of e + 256 are e's in units of 2^-44, rounded to nearest.)
  __device__ __forceinline__ u64 units(float x) const {
    const double e = mass(x);
    return e >= least ? static_cast<u64>(__double_as_longlong(e + 256.0) - __double_as_longlong(256.0)) : 0ull;
  }
};

struct Hist {
  uint32_t count[kBins], low[kBins], high[kBins];  // tokens, and the two halves of their mass
};

struct Shared {
  Hist hist;
  u64 list[kThreads];  // tokens of a bin: order key, and the token's complement
  int warp_ints[32];
  u64 warp_sums[32];
  u64 best;    // of the CTA: the largest logit's key, and the lowest token that has it
  int equal;   // tokens at the limit
  u64 sum;     // mass of what stays
  int listed;  // tokens asked into the list
  int bin;
  u64 above;         // of the goal, before the bin
  int upto, crowd;   // tokens up to the bin, and in it
  uint32_t limit;  // the threshold found
  int take;
};

__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

__device__ __forceinline__ void add_mass(Hist& h, int bin, u64 e) {
  const uint32_t e_low = static_cast<uint32_t>(e), old = atomicAdd(&h.low[bin], e_low);
  const uint32_t e_high = static_cast<uint32_t>(e >> 32) + (old + e_low < old ? 1u : 0u);
  if (e_high) atomicAdd(&h.high[bin], e_high);
}

// Sorts the CTA's values in descending order, one to a thread.
__device__ __forceinline__ u64 sort_descending(u64 x, int n, u64* list) {
  const int tid = threadIdx.x;
  for (int k = 2; k < 2 * n; k *= 2) {
    for (int j = k / 2; j > 0; j /= 2) {
      u64 y;
      if (j >= 32) {
        __syncthreads();
        list[tid] = x;
        __syncthreads();
        y = list[tid ^ j];
      } else {
        y = __shfl_xor_sync(kFull, x, j);
      }
      const bool keep_large = ((tid & k) == 0) == ((tid & j) == 0);
      x = (x > y) == keep_large ? x : y;
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

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) unsigned char slice_bytes[];
  T* row = reinterpret_cast<T*>(slice_bytes);
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = static_cast<int>(blockIdx.x) / parts;
  const int slice = ((a.V + parts - 1) / parts + 31) / 32 * 32;
  const int begin = min(a.V, part * slice), n = min(a.V, begin + slice) - begin;
  auto clean = [](float x) { return x == x ? x : neg_inf(); };  // NaN is never chosen
  auto logit = [&](int i) { return clean(to_f32(row[i])); };
  constexpr int kVec = 16 / sizeof(T);
  // f(i, logit) for the slice's tokens from `from` on, in any order, 16 bytes of them to each of `threads` threads.
  auto for_each = [&](int from, int to, int me, int threads, auto f) {
    int i = from + me * kVec;
    for (; i + kVec <= to; i += threads * kVec) {
      const uint4 v = *reinterpret_cast<const uint4*>(row + i);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) f(i + j, clean(to_f32(e[j])));
    }
    for (; i < to; ++i) f(i, logit(i));
  };
  auto all_tokens = [&](auto f) { for_each(0, n, tid, kThreads, f); };

  // ---- the slice, and its largest logit
  const T* src = static_cast<const T*>(a.logits) + r * a.stride + begin;
  u64 best = 0;
  auto look = [&](int i, T v) {
    float x = to_f32(v);
    if (x != x) x = neg_inf();
    const u64 b = static_cast<u64>(order_key(x)) << 32 | static_cast<uint32_t>(~(begin + i));
    best = b > best ? b : best;
  };
  int done = 0;
  if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
    done = n / kVec * kVec;
#pragma unroll 4
    for (int i = tid * kVec; i < done; i += kThreads * kVec) {
      const uint4 v = *reinterpret_cast<const uint4*>(src + i);
      *reinterpret_cast<uint4*>(row + i) = v;
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) look(i + j, e[j]);
    }
  }
#pragma unroll 4
  for (int i = done + tid; i < n; i += kThreads) {
    const T v = src[i];
    row[i] = v;
    look(i, v);
  }
  sh.hist.count[tid] = sh.hist.low[tid] = sh.hist.high[tid] = 0;
  if (tid == 0) sh.listed = 0;
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
  w.max = value_of(top);
  w.rate = 1.4426950408889634 / static_cast<double>(temperature);
  w.least = 0.0;
  w.limit = 0;
  w.take = 0x7fffffff;  // (all above)
  const int top_k = a.top_k.rows ? a.top_k.rows[r] : a.top_k.all;
  const float top_p = a.top_p.rows ? a.top_p.rows[r] : a.top_p.all;
  const float min_p = a.min_p.rows ? a.min_p.rows[r] : a.min_p.all;

  // The mass that the draw has to pass, of all that stays.
  const double uniform = static_cast<double>(a.uniforms[r]);
  auto drawn = [&](u64 all) {
    const double g = uniform > 0.0 ? floor(uniform * static_cast<double>(all)) : 0.0;
    const u64 x = g >= static_cast<double>(all) ? all - 1 : static_cast<u64>(g);
    return x < all ? x : all - 1;
  };
  // The rest, by one CTA, for the first m tokens in descending order (in its list, in any order) among which everything
  // that stays is: the first k of them, of those the ones before which less than `goal` lies (0: of top_p of these).
  auto finish = [&](int m, int k, u64 goal) {
    u64 x = tid < m ? sh.list[tid] : 0;
    x = sort_descending(x, m, sh.list);
    const int token = static_cast<int>(~static_cast<uint32_t>(x));
    const float logit_of = value_of(static_cast<uint32_t>(x >> 32));
    u64 e = tid < min(m, k) ? w.units(logit_of) : 0, total;
    const u64 before = scan_add<u64>(e, sh.warp_sums, total);
    if (goal == 0) {
      const double g = top_p < 1.f ? ceil(static_cast<double>(top_p > 0.f ? top_p : 0.f) * static_cast<double>(total)) : 0.0;
      goal = top_p < 1.f ? static_cast<u64>(g) : total;
      goal = goal < 1 ? 1 : goal;
    }
    if (min_p > 0.f) w.least = fmin(static_cast<double>(min_p), 1.0);
    e = before < goal && e ? w.units(logit_of) : 0;
    // In the vocabulary's order.
    u64* masses = reinterpret_cast<u64*>(&sh.hist);
    __syncthreads();
    masses[tid] = e;
    const int kept = __syncthreads_count(e != 0);  // (the first ones)
    u64 y = e ? ~(static_cast<u64>(token) << 10 | tid) : 0;
    y = ~sort_descending(y, kept, sh.list);
    e = tid < kept ? masses[y & 1023] : 0;
    u64 all;
    const u64 sum = scan_add<u64>(e, sh.warp_sums, all) + e;
    const u64 number = drawn(all);
    if (sum > number && sum - e <= number) a.tokens[r] = static_cast<int>(y >> 10);
  };

  // ---- thresholds: first by counts (top_k), then by masses (top_p)
  // Of the cluster's histograms, the thread's bin (in the order of descending logits).
  auto cluster_bin = [&](int bin, u64& count, u64& mass) {
    count = mass = 0;
    for (int p = 0; p < parts; ++p) {
      const Hist* h = cluster.map_shared_rank(&sh.hist, p);
      count += h->count[bin];
      mass += static_cast<u64>(h->high[bin]) << 32 | h->low[bin];
    }
  };
  auto clear = [&]() {  // once all have read
    cluster.sync();
    sh.hist.count[tid] = sh.hist.low[tid] = sh.hist.high[tid] = 0;
    __syncthreads();
  };
  for (int mode = 0; mode < 2; ++mode) {
    const bool counts = mode == 0;
    if (counts ? top_k <= 0 || top_k >= a.V : !(top_p < 1.f)) continue;
    // What of a token counts towards the goal; tokens at top_k's limit that do not all stay are told apart in the list.
    const bool some_at_limit = !counts && w.take != 0x7fffffff;
    u64 goal = counts ? static_cast<u64>(top_k) : 0, start = 0;  // start: the goal of the whole row
    auto weigh = [&](float x, uint32_t key, int bin) {
      if (!counts) {
        if (key <= w.limit) return;  // (those at it that stay are added below)
        add_mass(sh.hist, bin, w.units(x));
      }
      atomicAdd(&sh.hist.count[bin], 1u);
    };
    // All that stay at top_k's limit weigh alike.
    auto weigh_limit = [&](int bin) {
      if (!some_at_limit || part != 0 || tid != 0) return;
      add_mass(sh.hist, bin, w.units(value_of(w.limit)) * static_cast<u64>(w.take));
      atomicAdd(&sh.hist.count[bin], static_cast<uint32_t>(w.take));
    };
    // The bin that holds the goal: `bin` is the thread's place in descending order.
    auto choose = [&](u64 count, u64 mass, bool whole) {
      const u64 v = counts ? count : mass;
      u64 total;
      const u64 before = scan_add<u64>(v, sh.warp_sums, total);
      int all;
      const int ahead = counts ? 0 : scan_add<int>(static_cast<int>(count), sh.warp_ints, all);
      if (whole && !counts) {
        // The least whole number that is not below top_p of the mass; the first token always stays.
        const double g = ceil(static_cast<double>(top_p > 0.f ? top_p : 0.f) * static_cast<double>(total));
        goal = static_cast<u64>(g);
        goal = goal < 1 ? 1 : goal > total ? total : goal;
      }
      if (whole) start = goal;
      if (before < goal && before + v >= goal) {
        sh.bin = tid;
        sh.above = before;
        sh.crowd = static_cast<int>(count);
        sh.upto = (counts ? static_cast<int>(before) : ahead) + static_cast<int>(count);
      }
      __syncthreads();
      goal -= sh.above;
    };
    bool found = false, lost = false;
    int crowded = 0;  // level 1: the bin of level 0 that is cut
    for (int level = 0; level < 2 && !found && !lost; ++level) {
      // Monotone in the logit, so that equal logits share a bin and a lower one's is never before a higher one's; the
      // last bin has no end. -1: not of the bin that is cut.
      auto bin_of = [&](float x) {
        const float d = x == w.max ? 0.f : w.max - x;
        const int bin = static_cast<int>(fminf(d * kBinsPerUnit, static_cast<float>(kBins - 1)));
        if (level == 0) return bin;
        const float in = (d - static_cast<float>(crowded) / kBinsPerUnit) * (kBinsPerUnit * kBins);
        return bin != crowded ? -1 : static_cast<int>(fminf(fmaxf(in, 0.f), static_cast<float>(kBins - 1)));
      };
      all_tokens([&](int, float x) {
        const int bin = bin_of(x);
        if (bin >= 0) weigh(x, order_key(x), bin);
      });
      if (some_at_limit && bin_of(value_of(w.limit)) >= 0) weigh_limit(bin_of(value_of(w.limit)));
      cluster.sync();
      u64 count, mass;
      cluster_bin(tid, count, mass);
      choose(count, mass, level == 0);
      const int bin = sh.bin, crowd = sh.crowd, upto = sh.upto;
      clear();
      u64* list = cluster.map_shared_rank(sh.list, 0);
      int* listed = cluster.map_shared_rank(&sh.listed, 0);
      auto enlist = [&](int i, uint32_t key) {
        const int at = atomicAdd(listed, 1);
        if (at < kThreads) list[at] = static_cast<u64>(key) << 32 | static_cast<uint32_t>(~(begin + i));
      };
      if (level == 0 && upto <= kThreads && !some_at_limit) {
        // ---- few: all of them go to the first CTA, which does the rest
        all_tokens([&](int i, float x) {
          if (bin_of(x) <= bin) enlist(i, order_key(x));
        });
        cluster.sync();
        if (part != 0) return;
        finish(upto, counts ? top_k : 0x7fffffff, counts ? 0 : start);
        return;
      }
      if (crowd > kThreads) {  // its tokens alone, in finer bins
        lost = bin == kBins - 1 || level == 1;
        crowded = bin;
        continue;
      }
      // ---- its tokens to the first CTA, sorted there
      all_tokens([&](int i, float x) {
        if (bin_of(x) != bin) return;
        const uint32_t key = order_key(x);
        if (counts || key > w.limit || (some_at_limit && key == w.limit)) enlist(i, key);
      });
      cluster.sync();
      if (part == 0) {
        const int m = sh.listed;
        if (m <= kThreads) {  // (more where some at top_k's limit do not stay)
          u64 x = tid < m ? sh.list[tid] : 0;
          x = sort_descending(x, m, sh.list);
          __syncthreads();
          sh.list[tid] = x;
          __syncthreads();
          const uint32_t key = static_cast<uint32_t>(x >> 32);
          // Tokens of the same logit before this one.
          int first = tid;
          if (tid < m) {
            int lo = 0;  // the first place with the key
            while (lo < first) {
              const int mid = (lo + first) >> 1;
              if (static_cast<uint32_t>(sh.list[mid] >> 32) > key) lo = mid + 1; else first = mid;
            }
          }
          const int same = tid - first;
          u64 v = 0;
          if (tid < m && !(some_at_limit && key == w.limit && same >= w.take)) v = counts ? 1ull : w.units(value_of(key));
          u64 total;
          const u64 before = scan_add<u64>(v, sh.warp_sums, total);
          if (before < goal && before + v >= goal) {
            // The last of its logit: all of that logit stay, and need not be told apart.
            const bool whole = !(some_at_limit && key == w.limit) &&
                               (tid + 1 == m || static_cast<uint32_t>(sh.list[tid + 1] >> 32) != key);
            sh.limit = whole ? key - 1 : key;
            sh.take = whole ? 0x7fffffff : same + 1;
          }
        } else if (tid == 0) {
          sh.take = 0;
        }
        __syncthreads();
        if (tid == 0) sh.listed = 0;
      }
      cluster.sync();
      const uint32_t limit = *cluster.map_shared_rank(&sh.limit, 0);
      const int take = *cluster.map_shared_rank(&sh.take, 0);
      if (take == 0) {
        lost = true;
      } else {
        w.limit = limit;
        w.take = take;
        found = true;
      }
      cluster.sync();  // read before the first CTA writes them again
    }
    if (found) continue;
    // ---- digit by digit
    goal = start;
    uint32_t limit = 0;
    constexpr int kBits = 10;
    for (int digit = 0; digit < 4; ++digit) {
      const int shift = digit == 3 ? 0 : 22 - kBits * digit, bits = digit == 3 ? 2 : kBits;
      auto digit_of = [&](uint32_t key) { return static_cast<int>((key >> shift) & ((1u << bits) - 1)); };
      auto within = [&](uint32_t key) { return digit == 0 || (key >> (shift + bits)) == (limit >> (shift + bits)); };
      all_tokens([&](int, float x) {
        const uint32_t key = order_key(x);
        if (within(key)) weigh(x, key, kBins - 1 - digit_of(key));
      });
      if (some_at_limit && within(w.limit)) weigh_limit(kBins - 1 - digit_of(w.limit));
      cluster.sync();
      u64 count, mass;
      cluster_bin(tid, count, mass);
      choose(count, mass, false);
      limit |= static_cast<uint32_t>(kBins - 1 - sh.bin) << shift;
      clear();
    }
    // What is left of the goal is taken at the limit, token by token.
    if (counts) {
      w.take = static_cast<int>(goal);
    } else {
      const u64 e = w.units(value_of(limit)), some = (goal + e - 1) / e;
      const int available = limit == w.limit && some_at_limit ? w.take : 0x7fffffff;
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
      equal += __popc(__ballot_sync(kFull, i0 + lane < w1 && order_key(logit(i0 + lane)) == w.limit));
    int all_equal;
    equal = scan_add<int>(lane == 0 ? equal : 0, sh.warp_ints, all_equal);
    equal = __shfl_sync(kFull, equal, 0);
    if (tid == 0) sh.equal = all_equal;
    cluster.sync();
    for (int p = 0; p < part; ++p) equal += *cluster.map_shared_rank(&sh.equal, p);
  }
  // Mass of a token, with `e` tokens at the limit before it.
  auto stays = [&](float x, int e) {
    const uint32_t key = order_key(x);
    return key > w.limit || (key == w.limit && e < w.take) ? w.units(x) : 0ull;
  };
  u64 sum = 0;
  if (!ties) {
    for_each(w0, w1, lane, 32, [&](int, float x) { sum += order_key(x) > w.limit ? w.units(x) : 0ull; });
  } else {
    int e = equal;
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const bool in = i0 + lane < w1;
      const float x = in ? logit(i0 + lane) : neg_inf();
      const unsigned at = __ballot_sync(kFull, in && order_key(x) == w.limit);
      if (in) sum += stays(x, e + __popc(at & ((1u << lane) - 1)));
      e += __popc(at);
    }
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
  // The first token whose mass and that of those before it exceed the draw: in the stretch of one of the warps.
  const u64 number = drawn(all);
  const bool here = mine <= number && mine + sum > number;
  if (here && lane == 0) {
    sh.above = mine;
    sh.bin = warp;
    sh.equal = equal;
  }
  if (!__syncthreads_or(here)) return;
  const int s0 = min(n, sh.bin * stretch), s1 = min(n, s0 + stretch);
  u64 passed = sh.above;
  int at_limit = sh.equal;
  for (int i0 = s0; i0 < s1; i0 += kThreads) {
    const int i = i0 + tid;
    const float x = i < s1 ? logit(i) : neg_inf();
    int some = 0;
    const int e = ties ? scan_add<int>(i < s1 && order_key(x) == w.limit, sh.warp_ints, some) : 0;
    const u64 v = i < s1 ? stays(x, at_limit + e) : 0;
    u64 step;
    const u64 up_to = passed + scan_add<u64>(v, sh.warp_sums, step) + v;
    if (up_to > number && up_to - v <= number) a.tokens[r] = begin + i;
    passed += step;
    at_limit += some;
  }
}

template <typename T>
int launch(const SampleArgs& a, int sms, cudaStream_t stream) {
  // CTAs of a row: as many as its logits need, more while they find SMs and 16 K logits each (fewer pay less for a
  // pass than they pay for meeting).
  constexpr int kSlice = kSampleBytes / static_cast<int>(sizeof(T));
  int parts = 1;
  while (parts * kSlice < a.V) parts *= 2;
  while (parts < kSampleCluster && static_cast<long long>(a.R) * parts * 2 <= sms && a.V / parts > 16384) parts *= 2;
  if (static_cast<long long>(a.R) * parts > 0x7fffffff) return static_cast<int>(cudaErrorInvalidValue);
  const int bytes = static_cast<int>(sizeof(T)) * (((a.V + parts - 1) / parts + 31) / 32 * 32);
  auto kern = sample_kernel<T>;
  const int rc = static_cast<int>(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleBytes));
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
